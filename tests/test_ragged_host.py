"""The operators of serving sequences of different lengths without a GPU: argument checks of the library and the wrappers,
before anything is launched, and the plain forms that the GPU tests compare with."""
import ctypes

import pytest
import torch

import ragged_check as R
from smlm_hip import _lib, kernels

FAKE = 256                    # a 16-byte aligned address that is never read: the checks fail first
BIG = 1 << 60
bf16 = torch.bfloat16


def pages(**kw):
    ok = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, num_pages=10, kind=_lib.BF16, page_size=16, kv_heads=2, head_dim=64)
    return ctypes.byref(_lib.KVPages(**dict(ok, **kw)))


def refuses_pages(call):
    """What every entry point that takes pages checks of them."""
    assert call(pages=None) == call(pages=pages(k=None)) == call(pages=pages(v=None)) == _lib.EINVAL
    assert call(pages=pages(kind=_lib.F32)) == call(pages=pages(kind=_lib.Q4)) == _lib.EINVAL
    assert call(pages=pages(kind=_lib.Q4, k_scale=FAKE, v_scale=FAKE + 8)) == _lib.EINVAL and "aligned" in _lib.last_error()
    assert call(pages=pages(k=FAKE + 8)) == call(pages=pages(num_pages=0)) == call(pages=pages(kv_heads=0)) == _lib.EINVAL
    assert call(pages=pages(head_dim=48)) == call(pages=pages(head_dim=256)) == _lib.EUNSUPPORTED and "head_dim" in _lib.last_error()
    for size in (8, 24, 0, -16, 8192):
        assert call(pages=pages(page_size=size)) == _lib.EUNSUPPORTED and "page size" in _lib.last_error()


def append_call(**kw):
    ok = dict(qkv=FAKE, stride=512, cos=FAKE, sin=FAKE, dtype=_lib.F32, len=100, rot=64, inter=0, pos=FAKE, slots=FAKE, pages=pages(),
              N=5, H=4, q=FAKE, k=None)
    return _lib.lib().smlm_paged_append(*dict(ok, **kw).values(), None)


def test_paged_append_refusals():
    refuses_pages(append_call)
    for name in ("qkv", "cos", "sin", "pos", "slots", "q"):
        assert append_call(**{name: None}) == _lib.EINVAL and "null" in _lib.last_error(), name
    for name in ("qkv", "cos", "sin", "q", "k"):
        assert append_call(**{name: FAKE + 8}) == _lib.EINVAL and "aligned" in _lib.last_error(), name
    assert append_call(pos=FAKE + 4) == append_call(slots=FAKE + 4) == append_call(dtype=_lib.F16) == _lib.EINVAL
    assert append_call(stride=504) == append_call(stride=516) == append_call(N=-1) == append_call(H=0) == append_call(len=-1) == _lib.EINVAL
    assert append_call(rot=8) == append_call(rot=24) == append_call(rot=80) == append_call(rot=0) == _lib.EUNSUPPORTED
    assert append_call(N=1 << 26) == _lib.EUNSUPPORTED and "2^31" in _lib.last_error()
    assert append_call(N=0) == _lib.OK


def test_paged_gather_refusals():
    def call(**kw):
        return _lib.lib().smlm_paged_gather(*dict(dict(pages=pages(), slots=FAKE, N=5, k=FAKE, v=FAKE), **kw).values(), None)

    refuses_pages(call)
    for name in ("slots", "k", "v"):
        assert call(**{name: None}) == call(**{name: FAKE + 4}) == _lib.EINVAL, name
    assert call(N=-1) == _lib.EINVAL and call(N=1 << 28) == _lib.EUNSUPPORTED and call(N=0) == _lib.OK


def test_paged_step_refusals():
    def call(**kw):
        return _lib.lib().smlm_paged_step(*dict(dict(table=FAKE, stride=7, M=5, lengths=FAKE, B=3, page=16, max_len=75, pos=FAKE,
                                                     slots=FAKE, next=FAKE), **kw).values(), None)

    for name in ("table", "lengths", "pos", "slots", "next"):
        assert call(**{name: None}) == call(**{name: FAKE + 2}) == _lib.EINVAL, name
    assert call(page=8) == call(page=24) == call(page=8192) == _lib.EUNSUPPORTED
    assert call(stride=4) == call(M=0) == call(B=-1) == call(max_len=-1) == call(B=1 << 31) == _lib.EINVAL and call(B=0) == _lib.OK
    with pytest.raises(ValueError, match="must be on a HIP"):
        kernels.paged_step(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 16, 32)


def two(a, b):
    return (ctypes.c_int64 * 2)(a, b)


def test_packed_attention_refusals():
    ok = dict(q=FAKE, qs=two(256, 64), k=FAKE, ks=two(128, 64), v=FAKE, vs=two(128, 64), cu_q=FAKE, cu_k=FAKE, B=2, N=10, S=12, H=4,
              kv=2, hd=64, scale=0.1, y=FAKE, ys=two(256, 64), zero=1)

    def call(**kw):
        return _lib.lib().smlm_packed_attention(*dict(ok, **kw).values(), None)

    for name in ("q", "k", "v", "y", "qs", "ks", "vs", "ys", "cu_q", "cu_k"):
        assert call(**{name: None}) == _lib.EINVAL and "null" in _lib.last_error(), name
    for name in ("q", "k", "v"):
        assert call(**{name: FAKE + 8}) == _lib.EINVAL and "aligned" in _lib.last_error(), name
    assert call(y=FAKE + 4) == call(cu_q=FAKE + 2) == _lib.EINVAL
    assert call(B=-1) == call(N=-1) == call(S=-1) == call(H=0) == call(H=5) == call(kv=0) == _lib.EINVAL
    assert call(hd=48) == call(hd=256) == call(N=(1 << 30) + 1) == call(S=(1 << 30) + 1) == _lib.EUNSUPPORTED
    for name in ("qs", "ks", "vs"):
        for bad in (two(-8, 64), two(256, 60), two((1 << 22) + 8, 64)):
            assert call(**{name: bad}) == _lib.EINVAL and "strides" in _lib.last_error(), name
    assert call(ys=two(258, 64)) == _lib.EINVAL
    assert call(scale=0.0) == call(scale=-1.0) == call(scale=float("nan")) == call(scale=float("inf")) == _lib.EINVAL
    assert call(N=0) == call(B=0, zero=0) == _lib.OK


def test_paged_attention_refusals():
    ok = dict(q=FAKE, stride=256, pages=pages(), table=FAKE, ts=8, max_pages=8, lengths=FAKE, B=2, H=4, scale=0.1, y=FAKE, ws=FAKE,
              bytes=BIG)

    def call(**kw):
        return _lib.lib().smlm_paged_attention(*dict(ok, **kw).values(), None)

    refuses_pages(call)
    for name in ("q", "table", "lengths", "y"):
        assert call(**{name: None}) == _lib.EINVAL and "null" in _lib.last_error(), name
    for name in ("q", "y"):
        assert call(**{name: FAKE + 8}) == _lib.EINVAL and "aligned" in _lib.last_error(), name
    assert call(stride=248) == call(stride=260) == call(table=FAKE + 2) == call(lengths=FAKE + 1) == _lib.EINVAL
    assert call(B=-1) == call(H=0) == call(H=3) == call(max_pages=-1) == call(ts=7) == _lib.EINVAL
    assert call(scale=0.0) == call(scale=float("nan")) == _lib.EINVAL
    assert call(max_pages=1 << 27, ts=1 << 27) == _lib.EUNSUPPORTED and "2^31" in _lib.last_error()
    assert call(B=1 << 31) == _lib.EINVAL and call(B=1 << 30) == _lib.EUNSUPPORTED
    far = dict(max_pages=10000, ts=10000)                       # a long table: the walk is split
    need = _lib.lib().smlm_paged_attention_workspace(2, 4, 2, 64, 16, 10000)
    assert need > 0
    assert call(**far, ws=None) == call(**far, bytes=need - 1) == call(**far, ws=FAKE + 8) == _lib.EINVAL
    assert "workspace" in _lib.last_error()
    assert call(B=0) == _lib.OK


@pytest.mark.parametrize("B,H,Hk,D,page,most", [(1, 1, 1, 32, 16, 1), (1, 32, 8, 128, 16, 8192), (512, 6, 6, 64, 64, 16),
                                                (3, 40, 2, 64, 4096, 100), (1, 1, 1, 128, 4096, 524287)])
def test_workspaces_are_bounded(B, H, Hk, D, page, most):
    """At most 256 splits of every head, and none where the batch fills the GPU."""
    need = _lib.lib().smlm_paged_attention_workspace(B, H, Hk, D, page, most)
    assert 0 <= need <= B * H * 256 * (D + 2) * 4
    assert B * Hk < 4096 or need == 0


def test_sample_refusals():
    ok = dict(x=FAKE, dtype=_lib.BF16, stride=100, u=FAKE, t=None, ta=1.0, k=None, ka=0, p=None, pa=1.0, m=None, ma=0.0, B=2, V=100,
              token=FAKE)

    def call(**kw):
        return _lib.lib().smlm_sample(*dict(ok, **kw).values(), None)

    for name in ("x", "u", "token"):
        assert call(**{name: None}) == _lib.EINVAL and "null" in _lib.last_error(), name
    for name, off in (("x", 1), ("u", 2), ("t", 2), ("k", 2), ("p", 1), ("m", 2), ("token", 4)):
        assert call(**{name: FAKE + off}) == _lib.EINVAL and "aligned" in _lib.last_error(), name
    assert call(dtype=_lib.F16) == call(B=-1) == call(V=0) == call(stride=99) == _lib.EINVAL
    assert call(V=(1 << 18) + 1, stride=1 << 20) == call(B=1 << 31) == _lib.EUNSUPPORTED
    assert call(B=0) == _lib.OK


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu():
    z = lambda *s, dtype=bf16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    kv = (z(2, 1, 16, 32), z(2, 1, 16, 32))
    n = z(3, dtype=torch.int64)
    for call in (lambda: kernels.paged_append(z(3, 96), z(4, 16), z(4, 16), n, n, kv, 1), lambda: kernels.paged_gather(kv, n),
                 lambda: kernels.packed_attention(z(3, 1, 32), z(3, 1, 32), z(3, 1, 32), z(2, dtype=torch.int32)),
                 lambda: kernels.paged_attention(z(1, 1, 32), kv, z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32)),
                 lambda: kernels.sample_tokens(z(1, 5), z(1, dtype=torch.float32))):
        with pytest.raises(ValueError, match="must be on a HIP"):
            call()


def test_kv_pages():
    k, v = kernels.kv_pages(3, 2, 16, 64, device="cpu")
    assert k.shape == v.shape == (3, 2, 16, 64) and k.dtype == bf16
    k, v, ks, vs = kernels.kv_pages(3, 2, 32, 128, "q4", "cpu")
    assert k.shape == v.shape == (3, 2, 32, 64) and k.dtype == torch.uint8 and ks.shape == vs.shape == (3, 2, 32, 2)
    for bad in (dict(kind="int8"), dict(head_dim=48), dict(page_size=24), dict(page_size=8), dict(num_pages=0)):
        with pytest.raises(ValueError, match="kv_pages"):
            kernels.kv_pages(**dict(dict(num_pages=3, n_kv_heads=2, page_size=16, head_dim=64, device="cpu"), **bad))


# ---- the plain forms themselves ------------------------------------------------------------------------------------------
def test_the_plain_attention_is_softmax_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 16, generator=g, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    y, _ = R.attention(q, k, v, R.causal(5, 9), 0.25)
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1), v.repeat_interleave(2, 1).transpose(0, 1),
        attn_mask=R.causal(5, 9), scale=0.25).transpose(0, 1)
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)


def test_the_plain_rotation_is_the_models():
    from smlm_hip.model import RotaryEmbedding
    rope = RotaryEmbedding(32, 50, 10000.0)
    x = torch.randn(7, 3, 32, dtype=torch.float64)
    want = rope.double()(x.transpose(0, 1), 20).transpose(0, 1)
    assert torch.allclose(R.rotate(x, rope.cos[20:27], rope.sin[20:27], False), want)


def test_the_plain_sampling_counts_out_the_distribution():
    """Over an even grid of u each token comes as often as its share."""
    x = torch.tensor([0.0, 2.0, 1.0, 2.0, -1.0])
    n = 4000
    for T, k, p, m, keep in ((1.0, 0, 1.0, 0.0, [0, 1, 2, 3, 4]), (0.5, 3, 1.0, 0.0, [1, 2, 3]), (1.0, 0, 0.6, 0.0, [1, 3]),
                             (1.0, 0, 0.2, 0.0, [1]), (1.0, 0, 1.0, 0.3, [1, 2, 3])):
        got = torch.tensor([R.sample(x, (i + 0.5) / n, T, k, p, m) for i in range(n)]).bincount(minlength=5) / n
        w = torch.zeros(5)
        w[keep] = (x[keep] / T).exp()
        assert torch.allclose(got.double(), (w / w.sum()).double(), atol=1.5 / n), (T, k, p, m)


# ---- the cache's bookkeeping ---------------------------------------------------------------------------------------------
def cache(n=3, max_len=40, page=16, **kw):
    from smlm_hip.paged import PagedKVCache
    return PagedKVCache(2, n, max_len, 1, 32, page, device="cpu", **kw)


def slots_of(c, b, n):
    """Where the first n tokens of sequence b lie, from the block table."""
    t = torch.arange(n)
    return c.block_table[b, t // c.page_size].long() * c.page_size + t % c.page_size


def test_a_cache_plans_prompts_and_steps():
    c = cache()
    new = [17, 0, 1]
    c.reserve(new)
    plan = c.plan_prompts(new)
    assert plan.positions.tolist() == list(range(17)) + [0] and plan.cu_q.tolist() == [0, 17, 17, 18] and plan.cu_k is None
    assert torch.equal(plan.slots, torch.cat([slots_of(c, 0, 17), slots_of(c, 2, 1)]))
    assert len(set(plan.slots.tolist())) == 18 and plan.slots.max() < c.num_pages * 16
    c.advance(new)
    assert c.seq_lens == [17, 0, 1] == c.lengths.tolist()
    again = [2, 5, 0]
    c.reserve(again)
    plan = c.plan_prompts(again)
    assert plan.positions.tolist() == [17, 18, 0, 1, 2, 3, 4] and plan.cu_q.tolist() == [0, 2, 7, 7]
    assert plan.cu_k.tolist() == [0, 19, 24, 24]                # sequence 2 is not attended to
    assert torch.equal(plan.all_slots, torch.cat([slots_of(c, 0, 19), slots_of(c, 1, 5)]))
    assert torch.equal(plan.slots, torch.cat([slots_of(c, 0, 19)[17:], slots_of(c, 1, 5)]))
    c.advance(again)
    c.reserve([1, 1, 1])
    step = c.plan_step()
    assert step.positions.tolist() == [19, 5, 1] and step.lengths.tolist() == [20, 6, 2]
    assert step.slots.tolist() == [int(slots_of(c, b, n)[-1]) for b, n in enumerate((20, 6, 2))]


def test_a_full_sequence_has_no_slot_for_a_step():
    c = cache(2, 16)
    c.reserve([16, 3])
    c.advance([16, 3])
    assert c.plan_step().slots[0] == -1 and c.plan_step().slots[1] >= 0
    c.block_table.fill_(-1)                                   # no pages: nothing is written
    assert c.plan_step().slots.tolist() == [-1, -1]


def test_a_cache_refuses_what_does_not_fit_and_takes_pages_back():
    c = cache(3, 40, num_pages=4)
    for bad in ([41, 0, 0], [1, 1], [-1, 0, 0], [17, 17, 16]):
        with pytest.raises(ValueError, match="PagedKVCache"):
            c.reserve(bad)
        assert len(c._free) == 4 and (c.block_table == -1).all()
    c.reserve([17, 16, 1])
    c.advance([17, 16, 1])
    assert not c._free
    with pytest.raises(ValueError, match="are free"):
        c.reserve([0, 1, 0])
    held = set(c.block_table[0, :2].tolist())
    c.clear(0)
    assert set(c._free) == held and c.seq_lens == [0, 16, 1] == c.lengths.tolist() and (c.block_table[0] == -1).all()
    c.reserve([0, 1, 0])
    c.clear()
    assert sorted(c._free) == [0, 1, 2, 3] and c.seq_lens == [0, 0, 0]


def test_models_that_a_paged_cache_does_not_fit():
    from smlm_hip.model import ModelConfig, Transformer
    m = Transformer(ModelConfig(vocab_size=64, d_model=64, n_layers=1, n_heads=2, ffn_hidden=64, max_seq_len=32))
    with pytest.raises(ValueError, match="bf16"):             # on the CPU
        m.prefill(m.paged_cache(1), [torch.tensor([1, 2])])
    with pytest.raises(ValueError, match="max_len"):
        m.paged_cache(1, 33)
