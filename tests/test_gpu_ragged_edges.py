"""Edges of serving sequences of different lengths: calls that the documentation allows and a formula decides, at the borders of
types, sizes, masks and states.  Sampling has no tolerance: the token is the one of the 64-bit definition."""
import math

import pytest
import torch

import ragged_check as R
from smlm_hip import kernels as K
from test_gpu_ragged_model import model, prompts

pytestmark = pytest.mark.gpu
DEV = "cuda"
bf16, f32 = torch.bfloat16, torch.float32
NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=bf16):
    return torch.randn(*shape, generator=g).to(dtype)


# ------------------------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("V", [1 << 18, 261_500])
def test_the_last_tokens_of_very_large_flat_rows_are_drawn(V, dtype):
    """Equal logits, masks alone and a temperature that leaves no difference: token n holds the share [n, n + 1) / V of u.  (u has
    24 bits, so u V is exact in 64.)"""
    u = torch.tensor([0.5, 0.998, 0.999, 1 - 2.0 ** -24])
    want = [int(float(a) * V) for a in u]
    for x, T in ((torch.full((4, V), -1.5), 1.0), (torch.full((4, V), -math.inf), 1.0), (torch.randn(4, V, generator=gen(V)), 1e30)):
        assert K.sample_tokens(x.to(DEV, dtype), u.to(DEV), T).tolist() == want
    for outside in (1.0, 7.0, math.inf):              # the last token all the same
        assert K.sample_tokens(x.to(DEV, dtype), torch.full((4,), outside, device=DEV), T).tolist() == [V - 1] * 4


@pytest.mark.parametrize("V", [6000, 50304])
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_masked_logits_weigh_nothing_at_any_temperature(dtype, V):
    """Few and half of the tokens left by each kind of mask, logits as far apart as the type has them, and a row of masks alone
    (each token the same weight), up to an infinite temperature, against the definition over the tokens that are left."""
    g = gen(V)
    x = torch.randn(V, generator=g)
    rows, left = [], []
    for mask in (-math.inf, torch.finfo(dtype).min, NAN):
        for share in (0.0005, 0.5):
            keep = torch.rand(V, generator=g) < share
            keep[77] = True
            rows.append(torch.where(keep, x, torch.full((V,), mask)))
            left.append(keep)
    every = torch.ones(V, dtype=torch.bool)
    rows += [torch.where(torch.rand(V, generator=g) < 0.5, -2e38, 1e38), torch.full((V,), -math.inf)]
    left += [every, every]
    rows = torch.stack(rows).to(dtype)
    for T in (1e36, 1e38, math.inf):
        for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.5), (4000, 0.7, 0.0), (40, 1.0, 0.0), (0, 0.8, 0.3)):
            for at in (0.0, 0.4, 1 - 2.0 ** -24):
                u = torch.full((len(rows),), at)
                got = K.sample_tokens(rows.to(DEV), u.to(DEV), T, k, p, m).tolist()
                ids = [keep.nonzero().flatten() for keep in left]
                want = [int(i[R.sample(r[i].float(), R.f32(at), R.f32(T), k, R.f32(p), R.f32(m))]) for r, i in zip(rows, ids)]
                assert got == want, (T, k, p, m, at)


# ------------------------------------------------------------------------------------------- attention over the pages
@pytest.mark.parametrize("codes", ["as appended", "of anything"])
def test_a_key_that_is_not_finite_gives_nan_over_4_bit_pages(codes):
    """Infinities and NaN among the keys: such a row reads back as NaN, so every query that sees it gets NaN, whatever the signs
    and the rounding of its sums."""
    g = gen(50)
    B, H, D, page, n = 512, 16, 64, 16, 5
    pages = K.kv_pages(B, 1, page, D, "q4", DEV)
    qkv = randn(g, B * n, 3 * D)
    qkv[2::2 * n, D + 5], qkv[2 + n::2 * n, D + 9] = math.inf, NAN
    cos, sin = torch.ones(n, D // 2, device=DEV), torch.zeros(n, D // 2, device=DEV)
    pos = torch.arange(n).repeat(B)
    slots = (torch.arange(B).repeat_interleave(n) * page + pos).to(DEV)
    K.paged_append(qkv.to(DEV), cos, sin, pos.to(DEV), slots, pages, 1)
    if codes == "of anything":
        pages[0][:, 0, 2] = torch.randint(0, 256, (B, D // 2), generator=g, dtype=torch.uint8).to(DEV)
    k, _ = K.paged_gather(pages, slots)
    assert torch.isnan(k[2::n]).all() and torch.isfinite(k[3::n]).all()
    q = randn(g, B, H, D)
    q[..., ::13] *= 30
    table, ones = torch.arange(B, dtype=torch.int32, device=DEV).unsqueeze(1), torch.ones(B, dtype=torch.int32, device=DEV)
    assert torch.isnan(K.paged_attention(q.to(DEV), pages, table, n * ones)).all()
    assert torch.isfinite(K.paged_attention(q.to(DEV), pages, table, 2 * ones)).all()


# --------------------------------------------------------------------------------------------- packed prompt attention
@pytest.mark.parametrize("D", [32, 64, 128])
def test_what_the_neighbours_queries_are_does_not_matter(D):
    """A query whose later scores exceed its first ones by 8.995 in the log2 domain, just short of what moves its softmax's reference
    point (a factor that rounds to 2 of bf16, 2^0.995 does not, beyond 2^8): beside queries that stay, that move theirs and that
    are NaN, in its own group of 16 and in the other, the same bits; and the formula's value."""
    g = gen(60 + D)
    T, S, scale = 32, 160, 8.995 / math.log2(math.e)
    k, v = torch.zeros(S, 1, D), randn(g, S, 1, D)
    k[64:128, 0, 0] = torch.rand(64, generator=g)
    k[100, 0, 0], k[128:, 0, 0] = 1.0, 0.25
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (T, S))
    for at in (0, 21):
        got = []
        for other in (0.5, 2.0, NAN):
            q = torch.zeros(T, 1, D)
            q[:, 0, 0] = other
            q[at, 0, 0] = 1.0
            got.append(K.packed_attention(q.to(DEV, bf16), k.to(DEV, bf16), v.to(DEV), cu_q, cu_k, scale=scale)[at].cpu())
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
        seen = torch.arange(S).unsqueeze(0) <= S - T + at
        want, bound = R.attention(q[at:at + 1].double(), k.to(bf16).double(), v.double(), seen, scale)
        assert ((got[0].double() - want[0]).abs() <= R.bound_of(want, bound)[0]).all()


# --------------------------------------------------------------------------------------------------------- refusals
def test_inputs_that_autograd_records_are_refused():
    """There is no backward pass: a ValueError instead of outputs that are not in the graph.  Tokens have no gradient anyway."""
    kv = K.kv_pages(2, 2, 16, 64, device=DEV)
    z = lambda *s, dtype=bf16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    q, n, i32 = z(3, 2, 64), z(3, dtype=torch.long), torch.int32
    cu, cos, table, ones = torch.tensor([0, 3], dtype=i32, device=DEV), z(9, 32, dtype=f32), z(3, 2, dtype=i32), z(3, dtype=i32) + 1
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda r: K.paged_append(r(z(3, 384)), cos, cos, n, n, kv, 2), lambda r: K.paged_append(z(3, 384), cos, r(cos), n, n, kv, 2),
             lambda r: K.paged_append(z(3, 384), cos, cos, n, n, (kv[0], r(kv[1])), 2), lambda r: K.paged_gather((r(kv[0]), kv[1]), n),
             lambda r: K.packed_attention(r(q), q, q, cu), lambda r: K.packed_attention(q, r(q), q, cu), lambda r: K.packed_attention(q, q, r(q), cu),
             lambda r: K.packed_attention(q, q, q, cu, out=r(q)), lambda r: K.paged_attention(r(q), kv, table, ones),
             lambda r: K.paged_attention(q, (r(kv[0]), kv[1]), table, ones)]
    for call in calls:
        with pytest.raises(ValueError, match="no backward"):
            call(leaf)
        call(lambda t: t)                                   # no input that records
        with torch.no_grad():
            call(leaf)
    assert K.sample_tokens(leaf(z(3, 5)), z(3, dtype=f32)).tolist() == [0, 0, 0]


def test_a_recorded_pass_over_a_paged_cache_is_refused():
    m = model()
    cache = m.paged_cache(2, 100)
    cache.reserve([1, 1])
    cache.plan = cache.plan_step()
    tok = torch.zeros(2, 1, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError, match="no backward"):
        m(tok, kv_caches=cache.layers)
    with torch.no_grad():
        m(tok, kv_caches=cache.layers)
    m.requires_grad_(False)
    m(tok, kv_caches=cache.layers)


# ------------------------------------------------------------------------------------------------------ odd strides
def test_append_of_rows_on_top_of_each_other():
    """One row expanded over several tokens, and rows that overlap in memory, are what they are as copies."""
    cos, sin = torch.rand(8, 16, generator=gen(1)).to(DEV), torch.rand(8, 16, generator=gen(2)).to(DEV)
    row = randn(gen(3), 1, 96).to(DEV)
    for qkv in (row.expand(5, 96), row.view(96).repeat(2).unfold(0, 96, 16)[:5], row.view(1, 1, 96).expand(5, 1, 96)):
        n, got = torch.arange(5, device=DEV), []
        for x in (qkv, qkv.contiguous()):
            pages = K.kv_pages(1, 1, 16, 32, device=DEV)
            got.append((*K.paged_append(x, cos, sin, n, n, pages, 1, keys=True), *pages))
        assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][0].any()


def test_sampled_tokens_of_expanded_rows():
    g = gen(5)
    for V in (1, 9):
        row, u = torch.randn(1, V, generator=g).to(DEV), torch.rand(6, generator=g).to(DEV)
        for x in (row.expand(6, V), row.t().expand(V, 6).t()):
            assert torch.equal(K.sample_tokens(x, u), K.sample_tokens(x.clone(memory_format=torch.contiguous_format), u))


def test_packed_attention_into_views():
    """`out` with padded rows, heads first, one row or one head is written as it lies; rows or heads on top of each other are refused."""
    q = randn(gen(2), 5, 2, 64).to(DEV)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    want = K.packed_attention(q, q, q, cu)
    room = lambda: torch.zeros(4000, dtype=bf16, device=DEV)  # noqa: E731
    for strides in ((128, 64, 1), (64, 320, 1), (68, 400, 1), (256, 68, 1)):
        out = room().as_strided(q.shape, strides)
        assert torch.equal(K.packed_attention(q, q, q, cu, out=out), want) and torch.equal(out, want)
    one = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    assert torch.equal(K.packed_attention(q[:1], q[:1], q[:1], one, out=room().as_strided((1, 2, 64), (0, 64, 1))), q[:1])
    assert torch.equal(K.packed_attention(q[:, :1], q[:, :1], q[:, :1], cu, out=room().as_strided((5, 1, 64), (64, 0, 1))), want[:, :1])
    for strides in ((64, 64, 1), (0, 64, 1), (128, 0, 1), (60, 320, 1), (64, 316, 1), (124, 64, 1), (128, 60, 1)):
        with pytest.raises(ValueError, match="twice"):
            K.packed_attention(q, q, q, cu, out=room().as_strided(q.shape, strides))


# ------------------------------------------------------------------------------------------------ the model and its cache
def test_a_cache_of_another_models_shape_is_refused():
    """Fewer positions than the cache is long (its later tokens would have no rotation), other heads or dims; nothing changes."""
    cache, seqs = model().paged_cache(1, 300), prompts([150])
    for other in (model(max_seq_len=299), model(n_heads=4), model(d_model=64), model(n_layers=3)):
        for call in (lambda: other.prefill(cache, seqs), lambda: other.generate_ragged(seqs, 3, cache)):
            with pytest.raises(ValueError, match="cache of"):
                call()
    assert cache.seq_lens == [0] and len(cache._free) == cache.num_pages
    model(max_seq_len=300).prefill(cache, seqs)


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("at", [0, 2])
@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_step_that_fails_leaves_the_prompts_in_the_cache(at, use_graph):
    """An error in a step (before the capture, in it, or among eager ones): lengths and block table are those of the prompts, and the
    next call, of this model or of the one whose graph the cache held, gives what it gives on a fresh cache."""
    m, n = model(), model(seed=9)
    seqs = prompts([5, 20])
    cache = m.paged_cache(2, 100)
    want = [who.generate_ragged(seqs, 4) for who in (m, n)]
    assert torch.equal(m.generate_ragged(seqs, 4, cache), want[0])
    cache.clear()
    calls, step = [], n._ragged_step

    def failing(*args):
        calls.append(0)
        if len(calls) > at:
            raise RuntimeError("a step that fails")
        step(*args)

    n._ragged_step = failing
    with pytest.raises(RuntimeError, match="that fails"):
        n.generate_ragged(seqs, 4, cache, use_graph=use_graph)
    assert cache.seq_lens == [5, 20] == cache.lengths.tolist() and cache.plan is None
    pages = [p + [-1] * (cache.block_table.shape[1] - len(p)) for p in cache._pages]
    assert cache.block_table.tolist() == pages and pages[1][0] >= 0
    del n._ragged_step
    for who, tokens in ((m, want[0]), (n, want[1])):
        cache.clear()
        assert torch.equal(who.generate_ragged(seqs, 4, cache), tokens)


@pytest.mark.parametrize("inside", [True, False])
def test_inference_mode_and_out_of_it(inside):
    """A cache made, or first used, in inference mode serves calls outside of it, and the other way round."""
    m = model()
    seqs = prompts([5, 20])
    want = m.generate_ragged(seqs, 4)
    with torch.inference_mode(inside):
        cache = m.paged_cache(2, 100)
    for mode in (True, False, True):
        with torch.inference_mode(mode):
            cache.clear()
            assert torch.equal(m.generate_ragged(seqs, 4, cache), want)


def test_prefill_of_nothing_is_of_the_type_of_any_other():
    m = model(f32)
    cache = m.paged_cache(2, 100)
    with torch.autocast("cuda", dtype=bf16):
        none = m.prefill(cache, [[], []])
        some = m.prefill(cache, [[3], []])
    assert none.dtype == some.dtype == bf16 and none.shape == some.shape and torch.isnan(none).all()
    assert torch.isnan(some[1]).all() and torch.isfinite(some[0]).all()


# ------------------------------------------------------------------------------------------- how exact the attention is
def close_to_64_bits(q, k, v, scale, key_scale=None, value_scale=None):
    """One query row q (H, D) over keys and values (n, Hk, D), all double: the result, what two bf16 terms a probability and fp32
    scores and sums may be off by, and the result with one bf16 term a probability.  The scales (n, Hk, 2) of 4-bit rows are their steps
    and lowest values: there a probability times its row's step is rounded, which acts on a value's distance from its row's middle."""
    (H, D), n = q.shape, k.shape[0]
    of = torch.arange(H) // (H // k.shape[1])
    k, v = k[:, of], v[:, of]
    s = (k * q).sum(-1) * scale                                           # (n, H)
    p = ((s - s.max(0).values) / math.log(2) - 8).exp2()                  # as the kernel's first reference point has it
    w = (p / p.sum(0)).unsqueeze(-1)
    y = (w * v).sum(0)
    size = q.abs().sum(-1)
    if key_scale is None:
        middle, spread, terms = torch.zeros_like(v), torch.ones_like(v), (k * q).abs().sum(-1)
        added = v.abs()
    else:
        step, low = key_scale[:, of, :1], key_scale[:, of, 1:]
        spread = value_scale[:, of, :1]
        middle = value_scale[:, of, 1:] + 7.5 * spread
        # scores are formed as step (sum (n + code) q - n sum q) + low sum q, n at most 256, q in fp16 to 2^-25 of the largest;
        # values as sums of (128 + code) steps beside the rows' middles
        terms = step[..., 0] * (271 * size + 8 * D * q.abs().amax(-1)) + low[..., 0].abs() * size
        added = 2 * (143 * spread + middle.abs())
    one = ((p.unsqueeze(-1) * spread).to(bf16).double() * ((v - middle) / spread) + p.unsqueeze(-1) * middle).sum(0) / p.sum(0).unsqueeze(-1)
    # a score's D products and sums in fp32 move its weight by as much, and the others' sum; an exponential's argument, up to 16,
    # and the exponential by 2^-18
    weights = 2 * D * 2.0 ** -24 * scale * terms.amax(0) + 2.0 ** -18
    bound = (R.HALF * y.abs() + 2.0 ** -16 * (w * (v - middle).abs()).sum(0) + weights.unsqueeze(-1) * (w * v.abs()).sum(0)
             + (n + 8) * 2.0 ** -24 * (w * added).sum(0))
    return y, bound, one


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 32), (9, 3, 64), (16, 2, 128)])
def test_probabilities_are_two_bf16_terms_over_pages(kind, H, Hk, D):
    """Few tokens, weights of nearly the same size, so that results near zero have small roundings of their own: within what two
    terms allow.  One term a probability is beyond it, by the same formula, on these inputs."""
    g = gen(D + H)
    page, scale = 16, 0.1 / D
    lengths = list(range(2, 34)) + [70, 400]
    total = sum(-(-n // page) for n in lengths)
    table = torch.zeros(len(lengths), 25, dtype=torch.int32)
    ids, at = torch.randperm(total, generator=g), 0
    for b, n in enumerate(lengths):
        need = -(-n // page)
        table[b, :need] = ids[at:at + need]
        at += need
    k, v = randn(g, total, Hk, page, D), randn(g, total, Hk, page, D)
    rows = lambda t: t.transpose(1, 2).flatten(0, 1).double()  # noqa: E731
    if kind == "bf16":
        pages, k, v, scales = (k, v), rows(k), rows(v), ()
    else:
        (ck, sk), (cv, sv) = R.quantized(k), R.quantized(v)
        pages, k, v = (ck, cv, sk, sv), rows(R.values(ck, sk)), rows(R.values(cv, sv))
        scales = rows(sk), rows(sv)
    q = randn(g, len(lengths), H, D)
    got = K.paged_attention(q.to(DEV), [p.to(DEV) for p in pages], table.to(DEV),
                            torch.tensor(lengths, dtype=torch.int32, device=DEV), scale).double().cpu()
    beyond = 0
    for b, n in enumerate(lengths):
        slots = table[b, torch.arange(n) // page].long() * page + torch.arange(n) % page
        y, bound, one = close_to_64_bits(q[b].double(), k[slots], v[slots], scale, *(t[slots] for t in scales))
        assert ((got[b] - y).abs() <= bound).all(), (n, ((got[b] - y).abs() / bound).max())
        beyond += ((one - y).abs() > bound).sum().item()
    assert beyond > 50


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@torch.no_grad()
def test_a_models_attention_over_what_its_cache_holds(kind):
    """A layer's attention, of a second piece of the prompts and of a step, against the formula over the rows that its pages hold
    afterwards (4-bit ones as the values they stand for): no allowance for what the cache itself rounds."""
    m = model(mem=False)
    H, D = m.cfg.n_heads, m.cfg.d_model // m.cfg.n_heads
    attn, lengths, more = m.layers[1].attn, [1, 7, 64, 130, 33], [5, 0, 70, 1, 20]
    cache = m.paged_cache(len(lengths), 300, kind, 32)
    m.prefill(cache, prompts(lengths))
    layer, g = cache.layers[1], gen(8)
    rows = lambda t, at: t.transpose(1, 2).flatten(0, 1)[at.to(DEV)].double().cpu()  # noqa: E731

    def projected(n):
        qkv = randn(g, n, 3 * H * D).to(DEV)
        copies = [t.clone() for t in layer.pages]
        q, _ = K.paged_append(qkv, attn.rope.cos, attn.rope.sin, cache.plan.positions, cache.plan.slots, copies, H)
        return qkv, q.double().cpu()

    cache.reserve(more)
    cache.plan = cache.plan_prompts(more)
    qkv, q = projected(sum(more))
    y = attn._paged(qkv, layer).double().cpu()
    first = 0
    for b, (n, new) in enumerate(zip(lengths, more)):
        k, v = (t.double().cpu() for t in K.paged_gather(layer.pages, cache._slots(b, 0, n + new).to(DEV)))
        want, bound = R.attention(q[first:first + new], k, v, R.causal(new, n + new), D ** -0.5)
        assert ((y[first:first + new] - want).abs() <= R.bound_of(want, bound)).all(), b
        first += new
    cache.advance(more)
    cache.reserve([1] * len(lengths))
    cache.plan = cache.plan_step()
    qkv, q = projected(len(lengths))
    y = attn._paged(qkv, layer).double().cpu()
    for b, n in enumerate(cache.seq_lens):
        at = cache._slots(b, 0, n + 1)
        if kind == "bf16":
            k, v, scales = rows(layer.pages[0], at), rows(layer.pages[1], at), ()
        else:
            k, v = (rows(R.values(c, s), at) for c, s in zip(layer.pages[:2], layer.pages[2:]))
            scales = rows(layer.pages[2], at), rows(layer.pages[3], at)
        want, bound, _ = close_to_64_bits(q[b], k, v, D ** -0.5, *scales)
        assert ((y[b] - want).abs() <= bound).all(), b


@pytest.mark.parametrize("of", ["normal", "far from zero", "small", "tiny", "huge"])
def test_what_4_bit_rows_stand_for(of):
    """Half a step, 2^-8 of the row's lowest value and 2^-8 of its range, and the gather's own rounding; rows of offsets large against
    their range too."""
    g = gen(70)
    N, D = 64, 64
    x = {"normal": 1.0, "far from zero": 0.1, "small": 1e-3, "tiny": 1e-30, "huge": 1e30}[of] * torch.randn(N, 3 * D, generator=g)
    x = (x + 100 if of == "far from zero" else x).to(bf16)
    a = torch.outer(torch.arange(N).double(), 10000.0 ** (-torch.arange(0, D, 2).double() / D))
    cos, sin = a.cos().float(), a.sin().float()
    if of == "far from zero":                              # keys as they are, too
        cos, sin = torch.full_like(cos, 1.003), torch.zeros_like(sin)
    pages, n = K.kv_pages(4, 1, 16, D, "q4", DEV), torch.arange(N, device=DEV)
    K.paged_append(x.to(DEV), cos.to(DEV), sin.to(DEV), n, n, pages, 1)
    rows = x.double().view(N, 3, D)
    keys = R.rotate(rows[:, 1:2], cos.double(), sin.double(), False)[:, 0]
    for got, want in zip(K.paged_gather(pages, n), (keys, rows[:, 2])):
        low, high = want.amin(-1, keepdim=True), want.amax(-1, keepdim=True)
        # (rounded, a step is up to 2^-8 longer; 4 roundings of fp32 in the rotation and the codes)
        bound = ((high - low) / 30 * (1 + R.HALF) + R.HALF * low.abs() + R.HALF * (high - low) + R.HALF * want.abs()
                 + 4 * 2.0 ** -24 * (low.abs() + high.abs()))
        assert ((got[:, 0].double().cpu() - want).abs() <= bound).all()


def test_4_bit_rows_of_a_range_beyond_fp32_are_nan():
    pages, n = K.kv_pages(1, 1, 16, 32, "q4", DEV), torch.arange(2, device=DEV)
    qkv = torch.ones(2, 3, 32)
    qkv[1, 1:, ::3], qkv[1, 1:, 1::3] = 3e38, -3e38
    one, zero = torch.ones(2, 16, device=DEV), torch.zeros(2, 16, device=DEV)
    K.paged_append(qkv.view(2, 96).to(DEV, bf16), one, zero, n, n, pages, 1)
    for got in K.paged_gather(pages, n):
        assert (got[0] == 1).all() and torch.isnan(got[1]).all()
    q, table = torch.ones(1, 1, 32, dtype=bf16, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    at = lambda m: K.paged_attention(q, pages, table, torch.tensor([m], dtype=torch.int32, device=DEV))  # noqa: E731
    assert (at(1) == 1).all() and torch.isnan(at(2)).all()
