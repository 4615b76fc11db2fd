"""Transformer.prefill and generate_ragged: prompts of different lengths in one pass, decoding over a paged cache in bf16 and 4
bits, greedy and sampled, against the model's own passes over single sequences in fp32.

Tolerance of logits, relative in the 2-norm: a block rounds its stream, norms, projections, attention and activation to bf16, some
12 roundings of at most 2^-8 a block; as independent errors 24 of them are 5 * 2^-8 = 2 % for two blocks, doubled for what later
layers amplify.  A row of 64 normal values spans 4.8 of their deviations, so a 4-bit step is 4.8 / 15 = 0.32 and its rounding,
uniform over a step, 0.32 / sqrt(12) = 0.092 of a row's norm: of the values, which a query that sees one token takes as they are,
and as much of the keys, 0.13 of an attention's output together; from two blocks, whose errors are independent, 0.18 of a stream
that were all attention.  That comes on top."""
import copy

import pytest
import torch

from smlm_hip import kernels as K
from smlm_hip.model import ModelConfig, Transformer

pytestmark = pytest.mark.gpu
DEV = "cuda"
NEAR = {"bf16": 0.04, "q4": 0.04 + 0.18}


def model(dtype=torch.bfloat16, mem=True, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = ModelConfig(**{**dict(vocab_size=512, d_model=128, n_layers=2, n_heads=2, ffn_hidden=256, max_seq_len=400, init_std=0.08,
                                mem_layers=[1] if mem else [], mem_n_keys=16, mem_heads=2, mem_knn=4, mem_k_dim=32), **kw})
    return Transformer(cfg).to(DEV).to(dtype).eval()


def prompts(lengths, seed=1, vocab=512):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in lengths]


def near(got, want, tol):
    off = (got.float() - want.float()).norm(dim=-1) / want.float().norm(dim=-1)
    assert torch.isfinite(got).all() and off.max().item() <= tol, off


def whole(m, seq):
    """Logits of a whole sequence from the fp32 copy of a model."""
    return m(seq.to(DEV).unsqueeze(0))[0]


LENGTHS = [1, 7, 64, 130, 33]


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("page", [16, 64])
@torch.no_grad()
def test_prefill_in_pieces_and_steps(kind, page):
    """Prompts in two passes, the second behind the cached first, with an empty piece; then steps of given tokens."""
    m = model()
    ref = copy.deepcopy(m).float()
    cache = m.paged_cache(len(LENGTHS), 200, kind, page)
    seqs = prompts(LENGTHS)
    first = [p[:len(p) // 2 + len(p) % 2] for p in seqs]
    second = [p[len(p) // 2 + len(p) % 2:] for p in seqs]
    near(m.prefill(cache, first), torch.stack([whole(ref, p)[-1] for p in first]), NEAR["bf16"])     # the pass reads no 4-bit keys
    got = m.prefill(cache, second)
    assert torch.isnan(got[0]).all()                    # sequence 0 got nothing new
    near(got[1:], torch.stack([whole(ref, p)[-1] for p in seqs[1:]]), NEAR[kind])
    assert cache.seq_lens == LENGTHS and cache.lengths.tolist() == LENGTHS
    more = prompts([3] * len(LENGTHS), seed=5)
    for i in range(3):
        cache.reserve([1] * len(LENGTHS))
        cache.plan = cache.plan_step()
        got = m(torch.stack([p[i] for p in more]).to(DEV).unsqueeze(1), kv_caches=cache.layers)[:, 0]
        cache.plan = None
        cache.advance([1] * len(LENGTHS))
        near(got, torch.stack([whole(ref, torch.cat([p, x[:i + 1]]))[-1] for p, x in zip(seqs, more)]), NEAR[kind])


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("mem", [False, True])
def test_generate_is_the_same_with_and_without_a_graph_and_on_a_second_call(kind, mem):
    m = model(mem=mem)
    seqs = prompts(LENGTHS)
    for settings in (dict(), dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)):
        runs = []
        cache = m.paged_cache(len(LENGTHS), 200, kind)
        for use_graph in (False, True, True):
            cache.clear()
            g = torch.Generator(DEV).manual_seed(3)
            runs.append(m.generate_ragged(seqs, 20, cache, generator=g, use_graph=use_graph, **settings))
            assert runs[-1].shape == (len(LENGTHS), 21) and cache.seq_lens == [n + 20 for n in LENGTHS]
            assert cache.lengths.tolist() == cache.seq_lens
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    other = m.generate_ragged(seqs, 20, generator=torch.Generator(DEV).manual_seed(4), **settings)
    assert not torch.equal(other, runs[0])


@torch.no_grad()
def test_greedy_tokens_are_the_largest_logits():
    """Every token is the largest logit of the pass before it, computed again over the whole sequence in fp32, or as near to it as
    the logits' tolerance."""
    m = model()
    ref = copy.deepcopy(m).float()
    seqs = prompts([5, 100, 40])
    out = m.generate_ragged(seqs, 12).cpu()
    for p, tokens in zip(seqs, out):
        logits = whole(ref, torch.cat([p, tokens[:-1]]))[len(p) - 1:].cpu()
        took = logits.gather(1, tokens.unsqueeze(1)).squeeze(1)
        slack = 2 * NEAR["bf16"] * logits.norm(dim=1) / logits.shape[1] ** 0.5 * 4
        assert (logits.max(1).values - took <= slack).all()


def test_sampled_tokens_follow_the_settings_of_their_sequence():
    m = model()
    seqs = prompts([9, 9, 9, 9])
    seqs = [seqs[0]] * 4
    T = torch.tensor([0.0, 5.0, 5.0, 5.0])
    k = torch.tensor([0, 1, 0, 3], dtype=torch.int32)
    out = m.generate_ragged(seqs, 30, temperature=T, top_k=k, generator=torch.Generator(DEV).manual_seed(0))
    assert torch.equal(out[0], out[1])                 # greedy, and the largest of one
    assert not torch.equal(out[0], out[2]) and not torch.equal(out[2], out[3])


def test_a_cache_goes_on_and_frees_its_pages():
    """A second call behind the first's tokens; a pool smaller than all sequences at full length; clearing one sequence."""
    m = model()
    cache = m.paged_cache(3, 300, "bf16", 16, num_pages=20)
    a = prompts([20, 33, 5])
    out = m.generate_ragged(a, 10, cache)
    used = sum(-(-(len(p) + 10) // 16) for p in a)
    assert len(cache._free) == 20 - used
    with pytest.raises(ValueError, match="are free"):
        m.generate_ragged(prompts([100, 100, 100]), 10, cache)
    assert cache.seq_lens == [len(p) + 10 for p in a]
    cache.clear(1)
    assert cache.seq_lens[1] == 0 and len(cache._free) == 20 - used + 3
    b = prompts([4, 40, 3], seed=7)
    b[0] = torch.cat([out[0, -1:].cpu(), b[0]])
    again = m.generate_ragged(b, 5, cache)
    fresh = m.paged_cache(3, 300, "bf16", 16)
    all_ = [torch.cat([a[0], out[0, :-1].cpu(), b[0]]), b[1], torch.cat([a[2], out[2, :-1].cpu(), b[2]])]
    want = m.prefill(fresh, all_)
    cache2 = m.paged_cache(3, 300, "bf16", 16)
    m.prefill(cache2, [x[:len(x) - len(y)] for x, y in zip(all_, b)])
    near(m.prefill(cache2, b), want, NEAR["bf16"])
    assert again.shape == (3, 6)


def test_graphs_follow_the_model():
    """A changed weight, another memory table and another model give what a run without graphs gives."""
    m, n = model(), model(seed=9)
    seqs = prompts([5, 17])
    cache = m.paged_cache(2, 100)

    def same(who):
        cache.clear()
        got = who.generate_ragged(seqs, 8, cache)
        cache.clear()
        assert torch.equal(got, who.generate_ragged(seqs, 8, cache, use_graph=False))

    same(m)
    with torch.no_grad():
        m.lm_head.weight.mul_(-1.0)
    same(m)
    m.set_memory_inference_table("int8")
    same(m)
    same(n)
    same(m)


def test_another_models_steps_in_between_leave_the_graph_its_weights():
    """A run of another model over the same cache without a graph, then the first one's graph again."""
    m, n = model(), model(seed=9)
    seqs = prompts([5, 17])
    cache = m.paged_cache(2, 100)
    want = m.generate_ragged(seqs, 8, cache)
    cache.clear()
    n.generate_ragged(seqs, 8, cache, use_graph=False)
    torch.empty(1 << 20, device=DEV).fill_(float("nan"))
    cache.clear()
    assert torch.equal(m.generate_ragged(seqs, 8, cache), want)


def test_a_model_that_the_fused_step_does_not_cover():
    """A width above the fused step's; the tokens are the same with and without a graph, and the largest logits."""
    m = model(mem=False, d_model=512, n_heads=8)
    ref = copy.deepcopy(m).float()
    seqs = prompts([5, 40])
    out = m.generate_ragged(seqs, 6)
    assert torch.equal(out, m.generate_ragged(seqs, 6, use_graph=False))
    with torch.no_grad():
        for p, tokens in zip(seqs, out.cpu()):
            logits = whole(ref, torch.cat([p, tokens[:-1]]))[len(p) - 1:].cpu()
            took = logits.gather(1, tokens.unsqueeze(1)).squeeze(1)
            slack = 2 * NEAR["bf16"] * logits.norm(dim=1) / logits.shape[1] ** 0.5 * 4
            assert (logits.max(1).values - took <= slack).all()


def test_autocast():
    m = model(torch.float32)
    seqs = prompts([30, 3])
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a = m.generate_ragged(seqs, 6)
        b = m.generate_ragged(seqs, 6, use_graph=False)
    assert torch.equal(a, b)
    with pytest.raises(ValueError, match="bf16"):
        m.generate_ragged(seqs, 6)


def test_prompts_of_any_shape():
    """Lists and (1, tokens) tensors are the sequences that they hold."""
    m = model()
    seqs = prompts([70, 17])
    want = m.generate_ragged(seqs, 5)
    assert torch.equal(want, m.generate_ragged([p.unsqueeze(0) for p in seqs], 5))
    assert torch.equal(want, m.generate_ragged([p.tolist() for p in seqs], 5))


def test_refusals():
    m = model()
    seqs = prompts([5, 17])
    for call in (lambda: m.paged_cache(2, 401), lambda: m.paged_cache(0), lambda: m.paged_cache(2, kind="int8"),
                 lambda: m.generate_ragged(seqs, 390), lambda: m.generate_ragged([seqs[0], seqs[0][:0]], 3),
                 lambda: m.generate_ragged(seqs, 3, m.paged_cache(3)), lambda: m.generate_ragged(seqs, -1),
                 lambda: m.prefill(m.paged_cache(2, 10), seqs), lambda: m.prefill(m.paged_cache(3), seqs),
                 lambda: model(n_heads=4, d_model=64, ffn_hidden=64).paged_cache(2)):
        with pytest.raises(ValueError):
            call()


def test_wrappers_refuse_what_the_kernels_do_not_take():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    kv, q4 = K.kv_pages(2, 2, 16, 64, device=DEV), K.kv_pages(2, 2, 16, 64, "q4", DEV)
    n, i32, f32 = z(3, dtype=torch.long), torch.int32, torch.float32
    cos = z(9, 32, dtype=f32)
    cu = torch.tensor([0, 3], dtype=i32, device=DEV)
    for call in (lambda: K.paged_append(z(3, 384), cos, cos, n, n, kv, 4), lambda: K.paged_append(z(3, 384, dtype=f32), cos, cos, n, n, kv, 2),
                 lambda: K.paged_append(z(3, 384), cos, cos, n[:2], n, kv, 2), lambda: K.paged_append(z(3, 384), cos, cos, n.int(), n, kv, 2),
                 lambda: K.paged_append(z(3, 384), z(9, 12, dtype=f32), z(9, 12, dtype=f32), n, n, kv, 2),
                 lambda: K.paged_append(z(3, 384), z(9, 40, dtype=f32), z(9, 40, dtype=f32), n, n, kv, 2),
                 lambda: K.paged_append(z(3, 384), cos, cos.double(), n, n, kv, 2), lambda: K.paged_append(z(3, 384), cos, cos, n, n, kv[:1], 2),
                 lambda: K.paged_append(z(3, 384), cos, cos, n, n, q4[:2], 2), lambda: K.paged_append(z(3, 384), cos, cos, n, n, (kv[0], kv[1][:1]), 2),
                 lambda: K.paged_append(z(3, 384), cos, cos, n, n, (kv[0].transpose(1, 2), kv[1].transpose(1, 2)), 2),
                 lambda: K.paged_gather(kv, n.int()), lambda: K.paged_gather((q4[0], q4[1], q4[2].float(), q4[3]), n),
                 lambda: K.packed_attention(z(3, 2, 48), z(3, 2, 48), z(3, 2, 48), cu), lambda: K.packed_attention(z(3, 3, 64), z(3, 2, 64), z(3, 2, 64), cu),
                 lambda: K.packed_attention(z(3, 2, 64), z(4, 2, 64), z(4, 2, 64), cu), lambda: K.packed_attention(z(3, 2, 64), z(3, 2, 64), z(3, 1, 64), cu),
                 lambda: K.packed_attention(z(3, 2, 64), z(3, 2, 64), z(3, 2, 64), cu.long()),
                 lambda: K.packed_attention(z(3, 2, 64), z(3, 2, 64), z(3, 2, 64), cu, scale=0.0),
                 lambda: K.packed_attention(z(3, 2, 64), z(3, 2, 64), z(3, 2, 64), cu, out=z(3, 2, 64, dtype=f32)),
                 lambda: K.packed_attention(z(3, 2, 64), z(3, 2, 64), z(3, 2, 64).cpu(), cu),
                 lambda: K.paged_attention(z(3, 2, 32), kv, z(3, 2, dtype=i32), z(3, dtype=i32)),
                 lambda: K.paged_attention(z(3, 3, 64), kv, z(3, 2, dtype=i32), z(3, dtype=i32)),
                 lambda: K.paged_attention(z(3, 2, 64), kv, z(2, 2, dtype=i32), z(3, dtype=i32)),
                 lambda: K.paged_attention(z(3, 2, 64), kv, z(3, 2, dtype=i32), z(3, dtype=torch.long)),
                 lambda: K.sample_tokens(z(3, 5), z(2, dtype=f32)), lambda: K.sample_tokens(z(3, 5), z(3)), lambda: K.sample_tokens(z(5), z(5, dtype=f32)),
                 lambda: K.sample_tokens(z(3, 5, dtype=torch.float16), z(3, dtype=f32)), lambda: K.sample_tokens(z(1, (1 << 18) + 1), z(1, dtype=f32)),
                 lambda: K.sample_tokens(z(3, 5), z(3, dtype=f32), z(2, dtype=f32)), lambda: K.sample_tokens(z(3, 5), z(3, dtype=f32), 1.0, z(3, dtype=f32)),
                 lambda: K.sample_tokens(z(3, 5), z(3, dtype=f32), float("nan"))):
        with pytest.raises(ValueError):
            call()
