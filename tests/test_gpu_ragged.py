"""The operators of serving sequences of different lengths against plain 64-bit forms: appending to a paged cache and reading
back, packed prompt attention, single-token attention over the pages in bf16 and 4 bits, sampling.

Tolerances: an output in bf16 is off by half a step, 2^-8 of it; attention adds what rounding each probability to bf16 (2^-8 of
it) moves the weighted sum of |v| by, once in the sum and once in the probabilities' own sum (ragged_check.bound_of).  Rotation
in fp32 adds three roundings of 2^-24.  Sampling has none: the token is the one of the 64-bit definition."""
import math

import pytest
import torch

import ragged_check as R
from smlm_hip import kernels as K
from smlm_hip.capture import capture

pytestmark = pytest.mark.gpu
DEV = "cuda"
bf16 = torch.bfloat16
NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=bf16):
    return torch.randn(*shape, generator=g).to(dtype)


def tables(n, rot, dtype=torch.float32):
    a = torch.outer(torch.arange(n).double(), 10000.0 ** (-torch.arange(0, rot, 2).double() / rot))
    return a.cos().to(dtype), a.sin().to(dtype)


def close(got, want, tol, what=""):
    got, off = got.double().cpu(), None
    assert got.shape == want.shape
    off = (got - want).abs() - tol
    assert not torch.isnan(got).any(), what
    worst = off.max().item() if off.numel() else -1
    assert worst <= 0, f"{what}: over the bound by {worst}, at {off.argmax().item()}"


def filled(g, kind, pages, Hk, page, D):
    """Pages with values of earlier tokens in every slot, on the GPU."""
    k, v = randn(g, pages, Hk, page, D), randn(g, pages, Hk, page, D)
    if kind == "bf16":
        return (k.to(DEV), v.to(DEV))
    (ck, sk), (cv, sv) = R.quantized(k), R.quantized(v)
    return (ck.to(DEV), cv.to(DEV), sk.to(DEV), sv.to(DEV))


def rows_of(pages):
    """k, v (slots, Hk, D) double: what the pages stand for."""
    if len(pages) == 2:
        out = [p.double() for p in pages]
    else:
        out = [R.values(p, s) for p, s in zip(pages[:2], pages[2:])]
    return [x.transpose(1, 2).flatten(0, 1).cpu() for x in out]


# ------------------------------------------------------------------------------------------------ append and gather
@pytest.mark.parametrize("N,H,Hk,D,rot,interleaved,page,kind,rope", [
    (1, 1, 1, 32, 32, False, 16, "bf16", torch.float32), (1, 6, 6, 64, 64, False, 64, "q4", torch.float32),
    (7, 6, 6, 64, 64, False, 16, "bf16", torch.float32), (33, 8, 2, 128, 128, False, 32, "q4", torch.float32),
    (33, 8, 2, 128, 64, False, 32, "bf16", bf16), (19, 3, 1, 64, 32, True, 128, "q4", bf16),
    (50, 5, 5, 32, 16, False, 16, "q4", torch.float32), (50, 5, 1, 32, 32, True, 16, "bf16", torch.float32),
    (64, 4, 4, 128, 48, False, 4096, "bf16", torch.float32), (257, 9, 3, 64, 64, False, 256, "q4", torch.float32)])
@pytest.mark.parametrize("strided", [False, True])
def test_append_and_gather(N, H, Hk, D, rot, interleaved, page, kind, rope, strided):
    g = gen(N + D)
    total = max(3, 2 * N // page + 2)
    pages = filled(g, kind, total, Hk, page, D)
    before = [p.clone() for p in pages]
    C, longest = (H + 2 * Hk) * D, 3000
    wide = randn(g, N, C + (24 if strided else 0))
    qkv = wide.to(DEV)[:, 8:8 + C] if strided else wide.to(DEV)
    cos, sin = tables(longest, rot, rope)
    pos = torch.randint(0, longest, (N,), generator=g)
    slots = torch.randperm(total * page, generator=g)[:N]
    if N > 6:
        slots[1], slots[2], pos[3], pos[4] = -1, total * page, longest, -5
    q, k = K.paged_append(qkv, cos.to(DEV), sin.to(DEV), pos.to(DEV), slots.to(DEV), pages, H, interleaved, keys=True)
    x = qkv.cpu().double().view(N, H + 2 * Hk, D)
    known = (pos >= 0) & (pos < longest)
    at = pos.clamp(0, longest - 1)
    turned = R.rotate(x[:, :H + Hk], cos.double()[at], sin.double()[at], interleaved)
    size = x[:, :H + Hk].abs().amax(-1, keepdim=True)
    tol = R.HALF * turned.abs() + 4 * 2.0 ** -24 * size
    close(q[known.to(DEV)], turned[known, :H], tol[known, :H], "q")
    close(k[known.to(DEV)], turned[known, H:], tol[known, H:], "k")
    assert torch.isnan(q[~known.to(DEV)][..., :rot]).all() and torch.isnan(k[~known.to(DEV)][..., :rot]).all()
    written = known & (slots >= 0) & (slots < total * page)
    got_k, got_v = rows_of(pages)
    new_k, new_v = turned[:, H:], x[:, H + Hk:]
    if kind == "bf16":
        close(got_k[slots[written]], new_k[written], tol[written, H:], "cached k")
        assert torch.equal(got_v[slots[written]], new_v[written])
    else:
        for got, new, scale in ((got_k, new_k[written], pages[2]), (got_v, new_v[written], pages[3])):
            scale = scale.transpose(1, 2).flatten(0, 1).cpu().double()[slots[written]]
            step, lo = scale[..., :1], scale[..., 1:]
            low, high = new.amin(-1, keepdim=True), new.amax(-1, keepdim=True)
            eps = 4 * 2.0 ** -24 * (low.abs() + high.abs())
            assert ((lo - low).abs() <= R.HALF * low.abs() + eps).all()
            assert ((step - (high - lo) / 15).abs() <= R.HALF * 1.01 * (high - lo) / 15 + eps).all()
            # half a step, and at the ends what rounding the lowest value and 15 steps leaves out
            close(got[slots[written]], new, step / 2 * 1.001 + R.HALF * 1.01 * (low.abs() + (high - lo)) + eps, "cached in 4 bits")
    for now, old in zip(pages, before):            # every other slot as it was
        now, old = now.transpose(1, 2).flatten(0, 1).cpu(), old.transpose(1, 2).flatten(0, 1).cpu()
        rest = torch.ones(total * page, dtype=torch.bool)
        rest[slots[written]] = False
        assert torch.equal(now[rest], old[rest])
    ask = torch.cat([slots, torch.tensor([0, total * page - 1, -7])])
    gk, gv = K.paged_gather(pages, ask.to(DEV))
    inside = (ask >= 0) & (ask < total * page)
    for got, want in ((gk, got_k), (gv, got_v)):
        close(got[inside.to(DEV)], want[ask[inside]], R.HALF * want[ask[inside]].abs(), "gathered")
        assert not got[~inside.to(DEV)].any()


def test_append_of_rows_without_spread_or_not_finite_in_4_bits():
    pages = K.kv_pages(2, 1, 16, 32, "q4", DEV)
    x = torch.zeros(6, 3, 32)
    x[0, 2] = 1.5
    x[1, 2] = -7.0
    x[2, 2] = torch.arange(32.0)
    x[2, 2, 5] = NAN
    x[3, 2], x[3, 2, 0] = 1.0, math.inf
    x[4, 2], x[4, 2, 31] = 1.0, -math.inf
    x[5, 2] = torch.arange(32.0) * 1e-38
    cos, sin = tables(8, 32)
    K.paged_append(x.view(6, 96).to(DEV, bf16), cos.to(DEV), sin.to(DEV), torch.arange(6, device=DEV), torch.arange(6, device=DEV),
                   pages, 1)
    k, v = K.paged_gather(pages, torch.arange(6, device=DEV))
    v = v[:, 0].float().cpu()
    assert not k.any()
    assert (v[0] == 1.5).all() and (v[1] == -7.0).all()
    assert torch.isnan(v[2]).all() and torch.isnan(v[3]).all() and torch.isnan(v[4]).all()
    assert torch.isfinite(v[5]).all()


@pytest.mark.parametrize("B", [1, 300])
def test_where_the_next_tokens_go(B):
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, 90, (B,), generator=g, dtype=torch.int32)
    lengths[0], lengths[-1] = 0, 79
    table = torch.randint(0, 1 << 30, (B, 7), generator=g, dtype=torch.int32)[:, :5]
    table[::3, 2] = -1
    before = lengths.clone()
    got = K.paged_step(table.to(DEV), lengths.to(DEV), 16, 75)
    pos = lengths.long()
    page = table.long().gather(1, (pos // 16).clamp(max=4).unsqueeze(1)).squeeze(1)
    want = torch.where((page >= 0) & (pos < 75), page * 16 + pos % 16, -1)
    for a, b in zip(got, (pos, want, before + 1)):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
    edge = torch.tensor([-1, 2 ** 31 - 1], dtype=torch.int32, device=DEV)       # no tokens there are: no slot
    assert K.paged_step(torch.zeros(2, 4, dtype=torch.int32, device=DEV), edge, 16, 2 ** 40)[1].tolist() == [-1, -1]


# --------------------------------------------------------------------------------------------- packed prompt attention
def packed(g, Tq, Sk, H, Hk, D, tail=0, head=0):
    """Packed inputs on the CPU, `head` and `tail` rows of no sequence around them."""
    cu_q, cu_k = [head], [0]
    for t, s in zip(Tq, Sk):
        cu_q.append(cu_q[-1] + t)
        cu_k.append(cu_k[-1] + s)
    N, S = cu_q[-1] + tail, cu_k[-1] + tail
    return (randn(g, N, H, D), randn(g, S, Hk, D), randn(g, S, Hk, D), torch.tensor(cu_q, dtype=torch.int32),
            torch.tensor(cu_k, dtype=torch.int32))


def packed_reference(q, k, v, cu_q, cu_k, scale):
    y, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        rows, keys = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        T, S = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        y[rows], bound[rows] = R.attention(q[rows].double(), k[keys].double(), v[keys].double(), R.causal(T, S), scale)
    return y, bound


LENGTHS = [([1], None), ([5], None), ([64], None), ([65, 63], None), ([0, 3, 0, 1, 0], None), ([127, 1, 129], None),
           ([1] * 40, None), ([30, 170, 2], None), ([5, 1, 40], [9, 100, 40]), ([7, 3], [4, 3]), ([6, 130], [0, 200]),
           ([2, 0, 2], [70, 5, 131])]


@pytest.mark.parametrize("Tq,Sk", LENGTHS, ids=lambda v: "x".join(map(str, v[:6])) if v else "same")
@pytest.mark.parametrize("H,Hk,D", [(1, 1, 32), (2, 2, 64), (6, 2, 64), (4, 1, 128)])
def test_packed_attention(Tq, Sk, H, Hk, D):
    g = gen(len(Tq) + sum(Tq) + D)
    q, k, v, cu_q, cu_k = packed(g, Tq, Tq if Sk is None else Sk, H, Hk, D)
    y = K.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu_q.to(DEV), None if Sk is None else cu_k.to(DEV))
    want, bound = packed_reference(q, k, v, cu_q, cu_k, D ** -0.5)
    close(y, want, R.bound_of(want, bound))


@pytest.mark.parametrize("H,Hk,D", [(8, 2, 64), (16, 16, 32), (8, 1, 128)])
def test_packed_attention_of_very_many_sequences(H, Hk, D):
    """More sequences than their beginnings are kept for beside the tiles, and heads that are spread over the chip's parts."""
    g = gen(H + D)
    Tq = torch.randint(0, 4, (700,), generator=g).tolist() + [150, 1]
    Sk = [n + more for n, more in zip(Tq, torch.randint(0, 3, (702,), generator=g).tolist())]
    q, k, v, cu_q, cu_k = packed(g, Tq, Sk, H, Hk, D)
    y = K.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu_q.to(DEV), cu_k.to(DEV))
    want, bound = packed_reference(q, k, v, cu_q, cu_k, D ** -0.5)
    close(y, want, R.bound_of(want, bound))


def test_packed_attention_of_rows_far_apart():
    """Rows 2^22 elements apart, the last 2^31 and more from the first."""
    g = gen(77)
    D, stride = 64, 1 << 22
    q, k, v, cu_q, cu_k = packed(g, [300, 220], [300, 220], 2, 1, D)
    room = torch.empty(len(q) * stride, dtype=bf16, device=DEV)
    far = []
    for at, t in ((0, q), (256, k), (512, v)):
        view = room.as_strided((len(t), t.shape[1], D), (stride, D, 1), at)
        far.append(view.copy_(t))
    y = room.as_strided(q.shape, (stride, D, 1), 1024).zero_()
    assert K.packed_attention(*far, cu_q.to(DEV), out=y).data_ptr() == y.data_ptr()
    assert torch.equal(y, K.packed_attention(*[t.to(DEV) for t in (q, k, v, cu_q)], out=torch.zeros_like(q, device=DEV)))


def test_packed_attention_of_projection_rows_scaled_with_rows_of_no_sequence():
    """Values as a view of the projection's rows, keys with padded rows, a scale of its own, rows around the sequences."""
    g = gen(5)
    H, Hk, D, Tq = 4, 2, 64, [33, 1, 90]
    q, k, v, cu_q, cu_k = packed(g, Tq, [40, 1, 150], H, Hk, D, tail=9, head=3)
    S = k.shape[0]
    wide = randn(g, S, (H + 2 * Hk) * D + 8)
    wide[:, (H + Hk) * D:(H + 2 * Hk) * D] = v.flatten(1)
    vd = wide.to(DEV)[:, (H + Hk) * D:(H + 2 * Hk) * D].view(S, Hk, D)
    kd = torch.zeros(S, Hk, D + 8, dtype=bf16, device=DEV)[..., :D]
    kd.copy_(k)
    want, bound = packed_reference(q, k, v, cu_q, cu_k, 0.3)
    args = (q.to(DEV), kd, vd, cu_q.to(DEV), cu_k.to(DEV))
    close(K.packed_attention(*args, scale=0.3), want, R.bound_of(want, bound))       # zeros around
    out = torch.full((q.shape[0], H + 1, D), 7.0, dtype=bf16, device=DEV)[:, 1:]
    got = K.packed_attention(*args, scale=0.3, out=out)
    assert got.data_ptr() == out.data_ptr()
    rows = slice(cu_q[0], cu_q[-1])
    close(out[rows], want[rows], R.bound_of(want, bound)[rows])
    assert (out[:3] == 7).all() and (out[cu_q[-1]:] == 7).all()


@pytest.mark.parametrize("D", [32, 64, 128])
def test_masked_keys_and_values_count_for_nothing(D):
    """NaN and infinities in later tokens and in the neighbours' leave every other query's result as it is, bit for bit."""
    g = gen(D)
    q, k, v, cu_q, cu_k = packed(g, [70, 50, 90], [70, 50, 90], 2, 1, D)
    args = [t.to(DEV) for t in (q, k, v, cu_q)]
    want = K.packed_attention(*args)
    for bad in (NAN, math.inf, -math.inf):
        for row in (0, 40, 69, 70, 119, 125, 209):
            kb, vb = args[1].clone(), args[2].clone()
            kb[row, :, 3] = bad
            vb[row, :, 1] = bad
            b = int(torch.searchsorted(cu_q[1:], row, right=True))
            clean = torch.ones(q.shape[0], dtype=torch.bool)
            clean[row:cu_q[b + 1]] = False
            got = K.packed_attention(args[0], kb, vb, args[3])
            assert torch.equal(got[clean.to(DEV)], want[clean.to(DEV)]), (bad, row)
            assert torch.isnan(got[row, :]).any() or not math.isnan(bad)
            got = K.packed_attention(args[0], args[1], vb, args[3])        # the values alone: seen ones give what they are
            assert torch.equal(got[clean.to(DEV)], want[clean.to(DEV)]), (bad, row)
            seen = got[row:cu_q[b + 1], :, 1].float()
            assert (torch.isnan(seen) if math.isnan(bad) else seen == bad).all()
            assert torch.equal(got[~clean.to(DEV)][..., 2:], want[~clean.to(DEV)][..., 2:])


def test_packed_attention_of_huge_scores():
    """One key outweighs all others; scores of thousands stay finite."""
    g = gen(1)
    q, k, v, cu_q, cu_k = packed(g, [100, 30], [100, 30], 2, 2, 64)
    q, k = q * 40, k * 40
    want, bound = packed_reference(q, k, v, cu_q, cu_k, 64 ** -0.5)
    y = K.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu_q.to(DEV))
    # scores up to 64 * 1,600 * 16 / 8 = 2 * 10^5 in fp32: off by 64 roundings of 2^-24 of their terms' sum, 0.3 at most in the
    # exponent where two keys nearly tie, so the weights are compared through the bound of a tie
    off = (y.double().cpu() - want).abs()
    assert torch.isfinite(y).all() and (off <= R.bound_of(want, bound) + 0.35 * bound).all()


def test_packed_attention_of_nothing():
    e = lambda *s: torch.empty(*s, dtype=bf16, device=DEV)  # noqa: E731
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert K.packed_attention(e(0, 2, 64), e(0, 1, 64), e(0, 1, 64), z).shape == (0, 2, 64)
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    got = K.packed_attention(torch.ones(5, 2, 64, dtype=bf16, device=DEV), e(0, 1, 64), e(0, 1, 64), two + torch.tensor(
        [0, 5], device=DEV, dtype=torch.int32), two)
    assert got.shape == (5, 2, 64) and not got.any()
    got = K.packed_attention(torch.ones(5, 2, 64, dtype=bf16, device=DEV), e(5, 1, 64) * 0, e(5, 1, 64) * 0, z)
    assert not got.any()


def test_offsets_that_do_not_fit_the_buffers_stay_inside_them():
    g = gen(2)
    q, k, v, _, _ = packed(g, [130], [130], 2, 1, 64)
    for cu in ([0, 1000], [-50, 60, 400], [90, 20, 130], [0, 0, 0]):
        y = K.packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert torch.isfinite(y).all()


# ------------------------------------------------------------------------------------------- attention over the pages
def paged_case(g, kind, lengths, H, Hk, D, page, extra=1):
    need = [-(-n // page) for n in lengths]
    total, widest = sum(need) + 2, max(need) + extra
    ids = torch.randperm(total, generator=g)
    table, at = torch.full((len(lengths), widest), 10 ** 9, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    pages = filled(g, kind, total, Hk, page, D)
    used = torch.zeros(total * page, dtype=torch.bool)
    slots = [table[b, torch.arange(n) // page].long() * page + torch.arange(n) % page for b, n in enumerate(lengths)]
    for s in slots:
        used[s] = True
    for p in pages:                       # what no sequence holds is anything at all
        rows = p.transpose(1, 2).flatten(0, 1).clone()
        rows[~used.to(DEV)] = NAN if p.dtype == bf16 else 255
        p.copy_(rows.view(total, page, *rows.shape[1:]).transpose(1, 2))
    return randn(g, len(lengths), H, D), pages, table, slots


def paged_reference(q, pages, slots, scale):
    k, v = rows_of(pages)
    y, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, s in enumerate(slots):
        seen = torch.ones(1, len(s), dtype=torch.bool)
        if len(pages) == 2:
            y[b:b + 1], bound[b:b + 1] = R.attention(q[b:b + 1].double(), k[s], v[s], seen, scale)
            continue
        scales = pages[3].transpose(1, 2).flatten(0, 1).cpu().double()[s]
        y[b:b + 1], _ = R.attention(q[b:b + 1].double(), k[s], v[s], seen, scale)
        # probability times step is rounded, which acts on a value's distance from its row's middle, and fp32 sums of (128 +
        # code) steps beside the middles: 2^-24 of each partial sum, of which a wavefront adds one per 32 tokens
        middle = scales[..., 1:] + 7.5 * scales[..., :1]
        parts = R.HALF * (v[s] - middle).abs() + (2.0 ** -20) * (143 * scales[..., :1] + middle.abs())
        _, bound[b:b + 1] = R.attention(q[b:b + 1].double(), k[s], parts / R.HALF, seen, scale)
    return y, bound


MANY = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 129, 300]


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("H,Hk,D,page", [(1, 1, 32, 16), (6, 6, 64, 64), (9, 3, 64, 16), (8, 1, 128, 32), (16, 1, 64, 128),
                                         (20, 1, 32, 64), (6, 2, 128, 256), (40, 2, 128, 16)])
def test_paged_attention(kind, H, Hk, D, page):
    g = gen(H + D + page)
    q, pages, table, slots = paged_case(g, kind, MANY, H, Hk, D, page)
    y = K.paged_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(MANY, dtype=torch.int32, device=DEV))
    want, bound = paged_reference(q, pages, slots, D ** -0.5)
    close(y, want, R.bound_of(want, bound))
    assert not y[0].any()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("lengths,H,Hk,D,page", [([5000], 2, 1, 64, 16), ([4097, 0, 31], 4, 2, 128, 64), ([9000, 1], 1, 1, 32, 16),
                                                 ([2500] * 3, 3, 3, 64, 4096)])
def test_paged_attention_of_long_sequences(kind, lengths, H, Hk, D, page):
    """Walks that are split and joined."""
    g = gen(sum(lengths))
    q, pages, table, slots = paged_case(g, kind, lengths, H, Hk, D, page)
    y = K.paged_attention(q.to(DEV), pages, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=0.2)
    want, bound = paged_reference(q, pages, slots, 0.2)
    close(y, want, R.bound_of(want, bound))


@pytest.mark.parametrize("kind,total", [("bf16", 4200), ("q4", 33800)])
def test_pages_far_into_a_large_pool(kind, total):
    """Tokens in the last pages of a pool whose values are 2^31 elements from its first, and those of a small pool."""
    g = gen(total)
    D, page, N = 128, 4096, 5000
    cos, sin = (t.to(DEV) for t in tables(N, D))
    qkv = randn(g, N, 4 * D).to(DEV)
    pos = torch.arange(N, device=DEV)
    got = []
    for pool, ids in ((K.kv_pages(total, 1, page, D, kind, DEV), [total - 1, total - 2]), (K.kv_pages(2, 1, page, D, kind, DEV), [1, 0])):
        table = torch.tensor([ids], dtype=torch.int32, device=DEV)
        slots = table[0].long().repeat_interleave(page)[:N] * page + pos % page
        q, _ = K.paged_append(qkv, cos, sin, pos, slots, pool, 2)
        y = K.paged_attention(q[-1:], pool, table, torch.tensor([N], dtype=torch.int32, device=DEV))
        got.append((q, y, *K.paged_gather(pool, slots)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert got[0][2].any() and got[0][1].any()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_paged_attention_of_odd_arguments(kind):
    """Queries and tables as views, lengths beyond the table and below zero, ids outside the pages, an empty table."""
    g = gen(9)
    lengths, H, Hk, D, page = [40, 70, 33, 20], 4, 2, 64, 16
    q, pages, table, slots = paged_case(g, kind, lengths, H, Hk, D, page, extra=0)
    wide = torch.zeros(4, 3 * H * D + 8, dtype=bf16, device=DEV)
    view = wide[:, H * D:2 * H * D].view(4, H, D)
    view.copy_(q)
    big = torch.full((4, table.shape[1] + 3), -3, dtype=torch.int32, device=DEV)
    big[:, 2:2 + table.shape[1]] = table.to(DEV)
    tab = big[:, 2:2 + table.shape[1]]
    tab[2, 1] = -1                        # tokens 16 .. 31 of sequence 2 are nowhere
    slots[2] = torch.cat([slots[2][:16], slots[2][32:]])
    tab[3, :] = 10 ** 6
    slots[3] = slots[3][:0]
    want, bound = paged_reference(q, pages, slots, D ** -0.5)
    y = K.paged_attention(view, pages, tab, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    close(y, want, R.bound_of(want, bound))
    full = table[1].long().repeat_interleave(page) * page + torch.arange(table.shape[1] * page) % page
    assert (table[1] < 10 ** 9).all()
    far = torch.tensor([-4, 10 ** 9, 0, 5], dtype=torch.int32, device=DEV)
    for p in pages:                        # the longest one's last page in full
        rows = p.transpose(1, 2).flatten(0, 1).clone()
        rows[full.to(DEV)] = rows[slots[0][0]].clone() if p.dtype == bf16 else rows[full.to(DEV)]
        p.copy_(rows.view(p.shape[0], page, *rows.shape[1:]).transpose(1, 2))
    y = K.paged_attention(view, pages, tab, far)
    want, bound = paged_reference(q[1:2], pages, [full], D ** -0.5)
    close(y[1:2], want, R.bound_of(want, bound))
    assert not y[0].any() and not y[2:].any()
    none = K.paged_attention(view, pages, torch.empty(4, 0, dtype=torch.int32, device=DEV), far)
    assert none.shape == (4, H, D) and not none.any()
    assert K.paged_attention(view[:0], pages, tab[:0], far[:0]).shape == (0, H, D)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_a_value_that_is_not_finite_reaches_its_own_sequence_alone(kind):
    g = gen(4)
    lengths, H, Hk, D, page = [40, 41, 39], 2, 1, 64, 16
    q, pages, table, slots = paged_case(g, kind, lengths, H, Hk, D, page)
    len_ = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = K.paged_attention(q.to(DEV), pages, table.to(DEV), len_)
    at = int(slots[1][7])
    row = pages[1] if kind == "bf16" else pages[3]
    row[at // page, :, at % page, 0] = NAN
    got = K.paged_attention(q.to(DEV), pages, table.to(DEV), len_)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.isnan(got[1]).any()


# ------------------------------------------------------------------------------------------------------------ sampling
def scores(g, B, V, dtype):
    rank = torch.arange(1, V + 1).float().log() * -1.1
    return (torch.randn(B, V, generator=g) + rank[torch.randperm(V, generator=g)] + 5).to(dtype)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.3, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05), (1.0, 1000, 0.5, 0.01), (0.0, 5, 0.5, 0.5),
            (1.0, 1, 1.0, 0.0), (2.0, 0, 0.999, 0.0), (1.0, 0, 0.0, 0.0), (1e-4, 0, 0.9, 0.0), (1.0, 7, 0.3, 1.0), (50.0, 700, 0.99, 0.0)]


@pytest.mark.parametrize("V", [1, 2, 7, 100, 1023, 8192, 32003, 50304])
@pytest.mark.parametrize("dtype", [bf16, torch.float32])
def test_sampled_tokens(V, dtype):
    g = gen(V)
    for n, (T, k, p, m) in enumerate(SETTINGS):
        B = 5
        x, u = scores(g, B, V, dtype), torch.rand(B, generator=g)
        u[0], u[1] = 0.0, 1 - 2.0 ** -24
        got = K.sample_tokens(x.to(DEV), u.to(DEV), T, k, p, m).tolist()
        want = [R.sample(x[b], float(u[b]), R.f32(T), k, R.f32(p), R.f32(m)) for b in range(B)]
        assert got == want, (T, k, p, m)


@pytest.mark.parametrize("V,dtype", [(100003, bf16), (131072, torch.float32), (1 << 18, bf16)])
def test_sampled_tokens_of_large_vocabularies(V, dtype):
    """Rows that LDS does not hold."""
    g = gen(V)
    x, u = scores(g, 3, V, dtype), torch.rand(3, generator=g)
    for T, k, p, m in SETTINGS[:5]:
        got = K.sample_tokens(x.to(DEV), u.to(DEV), T, k, p, m).tolist()
        assert got == [R.sample(x[b], float(u[b]), R.f32(T), k, R.f32(p), R.f32(m)) for b in range(3)], (T, k, p, m)


def test_sampled_tokens_with_settings_of_their_own_and_rows_as_views():
    g = gen(3)
    B, V = 40, 5001
    wide = scores(g, B, V + 10, bf16).to(DEV)
    x = wide[:, 3:3 + V]                   # neither aligned nor dense
    u = torch.rand(B, generator=g)
    T = torch.rand(B, generator=g) * 1.5
    T[::7] = 0
    k = torch.randint(-1, 300, (B,), generator=g, dtype=torch.int32)
    k[::5] = 0
    p, m = 1.05 - torch.rand(B, generator=g) * 0.6, torch.rand(B, generator=g) * 0.1
    got = K.sample_tokens(x, u.to(DEV), T.to(DEV), k.to(DEV), p.to(DEV), m.to(DEV)).tolist()
    rows = x.cpu()
    assert got == [R.sample(rows[b], float(u[b]), float(T[b]), int(k[b]), float(p[b]), float(m[b])) for b in range(B)]


def test_equal_masked_and_odd_logits():
    """Ties by the lowest index, in numbers that no list holds; masks by -inf and by the type's lowest value; NaN; infinities;
    rows that a mask leaves empty."""
    V = 6000
    g = gen(8)
    for dtype in (bf16, torch.float32):
        flat = torch.full((V,), -2.5)
        two = torch.where(torch.rand(V, generator=g) < 0.5, 1.0, 0.0)
        zeros = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
        hidden, lowest = torch.full((V,), -math.inf), torch.full((V,), torch.finfo(dtype).min)
        hidden[[5, 900, 4000]], lowest[[5, 900, 4000]] = torch.tensor([1.0, 3.0, 2.0]), torch.tensor([1.0, 3.0, 2.0])
        odd = torch.randn(V, generator=g)
        odd[::3] = NAN
        top = torch.randn(V, generator=g)
        top[[17, 18, 4444]] = math.inf
        rows = torch.stack([flat, two, zeros, hidden, lowest, odd, top, torch.full((V,), -math.inf), torch.full((V,), NAN)]).to(dtype)
        for T, k, p, m in [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (0.9, 3001, 1.0, 0.0), (1.0, 2000, 0.25, 0.0), (1.0, 2, 0.9, 0.0),
                           (0.0, 0, 1.0, 0.0), (1.0, 0, 0.75, 0.5)]:
            for at in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
                u = torch.full((len(rows),), at)
                got = K.sample_tokens(rows.to(DEV), u.to(DEV), T, k, p, m).tolist()
                want = []
                for x in rows:
                    y = x.float().clone()
                    if dtype == torch.float32:
                        y = torch.where(y == math.inf, torch.full_like(y, 3.3895313892515355e38), y)
                    else:
                        y = torch.where(y == math.inf, torch.full_like(y, torch.finfo(bf16).max), y)
                    want.append(R.sample(y, R.f32(at), R.f32(T), k, R.f32(p), R.f32(m)))
                assert got == want, (dtype, T, k, p, m, at)


def test_cuts_near_zero_among_equal_tokens_and_on_either_side():
    """Cuts among tokens that are zero or some 30 binades below the largest, among few and very many equal ones, in rows of one
    sign, and of tokens whose weights vanish."""
    V = 9000
    g = gen(31)
    x = torch.randn(V, generator=g)
    relu = x.clamp(min=0) * 0.4                                            # half of them zeros, at the cut
    tiny = torch.where(torch.rand(V, generator=g) < 0.999, x * 2.0 ** -30, x)   # cuts among magnitudes of 2^-30
    steps = (x * 4).round() / 4                                            # hundreds of each value
    signed = torch.where(torch.rand(V, generator=g) < 0.5, x * 1e-38, x * 3)    # subnormal magnitudes of both signs
    rows = torch.stack([relu, tiny, steps, signed, -x.abs() - 50, x.abs() + 1e4, x * 300, x * 1e-20]).to(bf16)
    for T, k, p, m in [(1.0, 0, 0.9, 0.0), (0.7, 0, 0.6, 1e-4), (2.0, 6000, 1.0, 0.0), (1.0, 3000, 0.8, 1e-3), (5.0, 0, 0.999, 0.0),
                       (1.0, 400, 0.9, 0.0), (1e30, 0, 0.3, 0.0), (1e-30, 0, 0.3, 0.0)]:
        for at in (0.0, 0.41, 0.93, 1 - 2.0 ** -24):
            u = torch.full((len(rows),), at)
            got = K.sample_tokens(rows.to(DEV), u.to(DEV), T, k, p, m).tolist()
            assert got == [R.sample(row, R.f32(at), R.f32(T), k, R.f32(p), R.f32(m)) for row in rows], (T, k, p, m, at)


def test_random_numbers_outside_their_range_give_a_token_all_the_same():
    x = torch.randn(4, 1000, generator=gen(0)).to(DEV)
    got = K.sample_tokens(x, torch.tensor([1.0, 5.0, -1.0, NAN], device=DEV), 1.0, 10)
    kept = x.topk(10).indices.sort(1).values
    assert got.tolist() == [kept[0, -1].item(), kept[1, -1].item(), kept[2, 0].item(), kept[3, 0].item()]
    assert K.sample_tokens(x[:0], torch.empty(0, device=DEV)).shape == (0,)


# --------------------------------------------------------------------------------------------------- graphs and streams
@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_captured_and_replayed(kind):
    """A step of append, attention and sampling as two graphs on inputs that change, between eager work."""
    g = gen(12)
    B, H, Hk, D, page, V = 3, 4, 2, 64, 16, 3001
    lengths = [70, 300, 9]
    _, pages, table, _ = paged_case(g, kind, [n + 16 for n in lengths], H, Hk, D, page)
    pages = [torch.nan_to_num(p) if p.dtype == bf16 else p for p in pages]
    cos, sin = (t.to(DEV) for t in tables(400, D))
    w = (torch.randn(H * D, V, generator=g) * 0.1).to(DEV)
    qkv = randn(g, B, (H + 2 * Hk) * D).to(DEV)
    table = table.to(DEV)
    len_, u = torch.tensor(lengths, dtype=torch.int32, device=DEV), torch.rand(B, generator=g).to(DEV)

    def step(own):
        pos = len_.long()
        slots = table.gather(1, (pos // page).unsqueeze(1)).squeeze(1).long() * page + pos % page
        q, _ = K.paged_append(qkv, cos, sin, pos, slots, own, H)
        y = K.paged_attention(q, own, table, len_ + 1)
        return y, K.sample_tokens(y.flatten(1).float() @ w, u, 0.8, 40, 0.9)

    mine = [[p.clone() for p in pages] for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for own in mine:
            step(own)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for own in mine[:2]:
        graph = torch.cuda.CUDAGraph()
        with capture(graph):
            out = step(own)
        graphs.append(graph)
        outs.append(out)
    for n in range(4):
        qkv.copy_(randn(g, *qkv.shape))
        u.copy_(torch.rand(B, generator=g))
        len_.copy_(torch.tensor([x + n for x in lengths], dtype=torch.int32))
        graphs[0].replay()
        graphs[1].replay()
        y, token = step(mine[2])
        torch.cuda.synchronize()
        for got in outs:
            assert torch.equal(got[0], y) and torch.equal(got[1], token)
        for own in mine[:2]:
            assert all(torch.equal(a, b) for a, b in zip(own, mine[2]))


def test_same_bits_on_every_call():
    g = gen(21)
    q, k, v, cu_q, _ = packed(g, [200, 3, 77], [200, 3, 77], 4, 2, 64)
    args = [t.to(DEV) for t in (q, k, v, cu_q)]
    assert torch.equal(K.packed_attention(*args), K.packed_attention(*args))
    for kind in ("bf16", "q4"):
        q, pages, table, _ = paged_case(g, kind, [3000, 10], 4, 1, 128, 16)
        args = (q.to(DEV), pages, table.to(DEV), torch.tensor([3000, 10], dtype=torch.int32, device=DEV))
        assert torch.equal(K.paged_attention(*args), K.paged_attention(*args))


def test_nothing_is_read_out_of_order_on_another_stream():
    g = gen(22)
    q, pages, table, slots = paged_case(g, "bf16", [500, 20], 2, 1, 64, 16)
    len_ = torch.tensor([500, 20], dtype=torch.int32, device=DEV)
    want = K.paged_attention(q.to(DEV), pages, table.to(DEV), len_)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        late = torch.zeros(2, 2, 64, dtype=bf16, device=DEV)
        torch.cuda._sleep(2_000_000)
        late.copy_(q.to(DEV))
        got = K.paged_attention(late, pages, table.to(DEV), len_)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)
