"""The dense training operators without a GPU: argument checks of the library and the wrappers, before anything is
launched, and Transformer.loss where it runs the modules."""
import pytest
import torch
import torch.nn.functional as F

from smlm_hip import _lib, kernels
from smlm_hip.model import ModelConfig, Transformer

FAKE = 256                    # a 16-byte aligned address that is never read: the checks fail first
BIG = 1 << 60


def loss_call(**kw):
    ok = dict(x=FAKE, ldx=64, w=FAKE, ldw=64, t=FAKE, ignore=-100, reduction=_lib.REDUCE_MEAN, M=10, V=100, d=64, loss=FAKE,
              count=FAKE, lse=FAKE, ws=FAKE, bytes=BIG)
    return _lib.lib().smlm_linear_ce(*dict(ok, **kw).values(), None)


def test_linear_ce_refusals():
    for name in ("x", "w", "t", "loss", "count", "lse"):
        assert loss_call(**{name: None}) == _lib.EINVAL and "null" in _lib.last_error(), name
    for name in ("x", "w"):
        assert loss_call(**{name: FAKE + 8}) == _lib.EINVAL and "aligned" in _lib.last_error(), name
    assert loss_call(t=FAKE + 4) == _lib.EINVAL
    assert loss_call(ldx=56) == loss_call(ldw=60) == loss_call(ldx=68) == loss_call(ldw=(1 << 21) + 8) == _lib.EINVAL
    assert loss_call(M=-1) == loss_call(V=0) == loss_call(d=0) == loss_call(reduction=3) == loss_call(reduction=-1) == _lib.EINVAL
    assert loss_call(d=60) == loss_call(V=1 << 31) == loss_call(M=1 << 40) == loss_call(M=(1 << 30) + 1, d=8) == _lib.EUNSUPPORTED
    assert loss_call(ws=None) == loss_call(ws=FAKE + 8) == loss_call(bytes=100) == _lib.EINVAL
    assert "workspace" in _lib.last_error()
    assert loss_call(M=0, count=None, reduction=_lib.REDUCE_NONE) == _lib.OK and loss_call(M=0) == _lib.EINVAL


def test_linear_ce_backward_refusals():
    ok = dict(g=FAKE, count=None, per_token=0, x=FAKE, ldx=64, w=FAKE, ldw=64, t=FAKE, ignore=-100, lse=FAKE, M=10, V=100, d=64,
              dx=FAKE, dw=FAKE, ws=FAKE, bytes=BIG)

    def call(**kw):
        return _lib.lib().smlm_linear_ce_backward(*dict(ok, **kw).values(), None)

    for name in ("g", "x", "w", "t", "lse"):
        assert call(**{name: None}) == _lib.EINVAL and "null" in _lib.last_error(), name
    assert call(dx=None, dw=None) == _lib.EINVAL
    assert call(dx=FAKE + 8) == call(dw=FAKE + 8) == call(M=0) == call(ws=FAKE + 4) == call(bytes=1000) == _lib.EINVAL
    assert call(d=12) == _lib.EUNSUPPORTED


@pytest.mark.parametrize("M,V,d", [(1, 1, 8), (64, 32000, 384), (129, 50304, 384), (16384, 50304, 384), (100000, 65536, 64),
                                   (1 << 22, 1000, 8)])
def test_linear_ce_workspaces_are_bounded(M, V, d):
    """The gradient's pieces stay within 1 GiB (or 256 columns), and its parts within what 128 splits take."""
    lib = _lib.lib()
    assert 0 < lib.smlm_linear_ce_workspace(M, V, d, 0) <= M * 8 * 1024 + (M + 64) * 16 + 4096
    grad = lib.smlm_linear_ce_workspace(M, V, d, 1)
    assert 0 < grad <= max(1 << 30, M * 512) + 256 + 128 * M * d * 4
    assert lib.smlm_linear_ce_workspace(0, V, d, 1) == 0


def ffn_call(**kw):
    ok = dict(x=FAKE, ldx=64, w13=FAKE, ld13=64, w2=FAKE, ld2=96, M=10, d=64, hidden=96, o=64, y=FAKE, ws=FAKE, bytes=BIG)
    return _lib.lib().smlm_gated_ffn(*dict(ok, **kw).values(), None)


def test_gated_ffn_refusals():
    for name in ("x", "w13", "w2", "y"):
        assert ffn_call(**{name: None}) == _lib.EINVAL, name
        assert ffn_call(**{name: FAKE + 8}) == _lib.EINVAL, name
    assert ffn_call(ldx=60) == ffn_call(ld13=56) == ffn_call(ld2=100) == ffn_call(ld2=(1 << 21) + 8) == _lib.EINVAL
    assert ffn_call(d=60) == ffn_call(hidden=100, ld2=104) == ffn_call(o=4) == ffn_call(M=1 << 34) == _lib.EUNSUPPORTED
    assert ffn_call(M=-1) == ffn_call(d=0) == ffn_call(hidden=0) == ffn_call(o=0) == _lib.EINVAL
    assert ffn_call(ws=None) == ffn_call(bytes=64) == _lib.EINVAL
    assert ffn_call(M=0) == _lib.OK
    ok = dict(dy=FAKE, ldy=64, x=FAKE, ldx=64, w13=FAKE, ld13=64, w2=FAKE, ld2=96, M=10, d=64, hidden=96, o=64, dx=FAKE,
              dw13=FAKE, dw2=FAKE, ws=FAKE, bytes=BIG)

    def back(**kw):
        return _lib.lib().smlm_gated_ffn_backward(*dict(ok, **kw).values(), None)

    for name in ("dy", "x", "w13", "w2"):
        assert back(**{name: None}) == _lib.EINVAL, name
    for name in ("dy", "dx", "dw13", "dw2"):
        assert back(**{name: FAKE + 8}) == _lib.EINVAL, name
    assert back(dx=None, dw13=None, dw2=None) == back(M=0) == back(ldy=56) == back(bytes=64) == _lib.EINVAL


def test_pad_rows_refusals():
    def call(**kw):
        ok = dict(src=FAKE, ld=65, blocks=2, rows=5, cols=65, dst=FAKE, rows_out=8, cols_out=72)
        return _lib.lib().smlm_pad_rows(*dict(ok, **kw).values(), None)
    assert call(src=None) == call(dst=None) == call(dst=FAKE + 8) == call(src=FAKE + 1) == _lib.EINVAL
    assert call(ld=64) == call(blocks=0) == call(rows=9) == call(rows=-1) == call(cols=73) == call(cols_out=68) == _lib.EINVAL
    assert call(rows_out=1 << 41) == call(cols_out=1 << 31) == call(blocks=1 << 21) == call(rows_out=1 << 36) == _lib.EUNSUPPORTED


def test_rmsnorm_train_refusals():
    lib = _lib.lib()
    ok = dict(x=FAKE, xt=_lib.F32, delta=FAKE, dt=_lib.BF16, w=FAKE, wt=_lib.F32, eps=1e-5, M=10, C=64, xs=FAKE, h=FAKE,
              ht=_lib.BF16, rstd=FAKE)

    def call(**kw):
        return lib.smlm_rmsnorm_train(*dict(ok, **kw).values(), None)

    for name in ("x", "w", "xs", "h", "rstd"):
        assert call(**{name: None}) == _lib.EINVAL, name
        assert call(**{name: FAKE + 1}) == _lib.EINVAL, name
    assert call(xt=_lib.F16) == call(wt=_lib.I8) == call(ht=_lib.I64) == call(xt=_lib.BF16, dt=_lib.F32) == _lib.EINVAL
    assert call(M=-1) == call(C=0) == call(eps=-1.0) == call(eps=float("nan")) == _lib.EINVAL
    assert call(C=16385) == _lib.EUNSUPPORTED
    assert call(M=0) == call(M=0, delta=None, xs=None) == _lib.OK
    ok = dict(dxs=FAKE, dh=FAKE, ht=_lib.BF16, xs=FAKE, xt=_lib.F32, w=FAKE, wt=_lib.F32, rstd=FAKE, M=10, C=64, dx=FAKE,
              ddelta=FAKE, dt=_lib.BF16, dw=FAKE, parts=FAKE)

    def back(**kw):
        return lib.smlm_rmsnorm_train_backward(*dict(ok, **kw).values(), None)

    for name in ("xs", "w", "rstd", "dx", "parts"):
        assert back(**{name: None}) == _lib.EINVAL, name
    assert back(dxs=None, dh=None) == back(M=0) == back(xt=_lib.BF16, dt=_lib.F32) == back(dw=FAKE + 2) == _lib.EINVAL
    assert back(C=16385) == _lib.EUNSUPPORTED
    assert lib.smlm_rmsnorm_parts(1 << 30, 64) <= 1024 * 64 and lib.smlm_rmsnorm_parts(1, 7) == 7


def test_the_wrappers_want_a_gpu():
    x, w, t = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(30, 16, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: kernels.linear_cross_entropy(x, w, t), lambda: kernels.gated_ffn(x, w, w[:, :15].contiguous()),
                 lambda: kernels.add_rmsnorm_train(x, None, torch.nn.RMSNorm(16))):
        with pytest.raises(ValueError, match="device"):
            call()


def small(**kw):
    torch.manual_seed(3)
    return Transformer(ModelConfig(**dict(dict(vocab_size=67, d_model=32, n_layers=2, n_heads=2, ffn_hidden=48, max_seq_len=16),
                                          **kw)))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_on_the_cpu_is_the_modules(reduction):
    m = small()
    idx = torch.randint(0, 67, (2, 9), generator=torch.Generator().manual_seed(0))
    t = torch.roll(idx, -1, 1)
    t[:, -1] = 5
    logits, mean = m(idx, t)
    assert torch.equal(m.loss(idx, t), mean)
    t[0, 3] = -1
    got = m.loss(idx, t, ignore_index=-1, reduction=reduction)
    ref = F.cross_entropy(logits.view(-1, 67), t.view(-1), ignore_index=-1, reduction=reduction)
    assert torch.equal(got.reshape(-1), ref.reshape(-1)) and got.shape == (t.shape if reduction == "none" else ())
    got.sum().backward()
    assert m.tok_emb.weight.grad is not None


def test_loss_calls_a_watched_embedding_once():
    m, seen = small(), []
    m.tok_emb.register_forward_hook(lambda *a: seen.append(1))
    m.register_forward_hook(lambda *a: seen.append(2))
    m.loss(torch.zeros(1, 4, dtype=torch.int64), torch.ones(1, 4, dtype=torch.int64))
    assert seen == [1, 2]


def test_default_eps_is_that_of_fp32():
    """F.rms_norm's without one, for bf16 inputs too."""
    norm, x = torch.nn.RMSNorm(16), (torch.randn(5, 16, generator=torch.Generator().manual_seed(0)) * 2.0 ** -11).bfloat16()
    assert kernels._rms_eps(norm) == 2.0 ** -23 and kernels._rms_eps(torch.nn.RMSNorm(16, eps=1e-5)) == 1e-5
    got, ref = F.rms_norm(x, (16,)).double(), F.rms_norm(x.double(), (16,), eps=kernels._rms_eps(norm))
    assert ((got - ref).abs() <= 2 * 2.0 ** -8 * ref.abs()).all()


def test_loss_of_flat_targets_on_the_cpu():
    """Losses in the targets' shape."""
    m = small()
    idx = torch.randint(0, 67, (2, 9), generator=torch.Generator().manual_seed(0))
    t = torch.roll(idx, -1, 1)
    flat, each = m.loss(idx, t.view(-1), reduction="none"), m.loss(idx, t, reduction="none")
    assert flat.shape == (18,) and torch.equal(flat, each.view(-1)) and torch.equal(m.loss(idx, t.view(-1)), m.loss(idx, t))


class _DoubleAsBf16:
    """torch, with 64 bits where the model asks for bf16."""
    bfloat16 = torch.float64

    def __getattr__(self, name):
        return getattr(torch, name)


def _in_64_bits(monkeypatch):
    """Transformer.loss takes its kernels' way on the CPU in 64 bits, with the operators' formulas in their place; counts them."""
    import smlm_hip.model as model
    calls = {"loss": 0, "ffn": 0, "norm": 0}

    def loss(x, w, t, ignore_index, reduction):
        calls["loss"] += 1
        return F.cross_entropy((x @ w.T).flatten(0, -2), t.flatten(), ignore_index=ignore_index, reduction=reduction)

    def ffn(x, w13, w2):
        calls["ffn"] += 1
        a, b = (x @ w13.T).chunk(2, -1)
        return (F.silu(a) * b) @ w2.T

    def norm(x, delta, norm, out_dtype=None):
        calls["norm"] += 1
        x = x if delta is None else x + delta
        return x, F.rms_norm(x, norm.weight.shape, norm.weight, norm.eps)

    monkeypatch.setattr(model, "torch", _DoubleAsBf16())
    monkeypatch.setattr(Transformer, "_loss_kernels", lambda *a: True)
    for name, f in (("linear_cross_entropy", loss), ("gated_ffn", ffn), ("add_rmsnorm_train", norm)):
        monkeypatch.setattr(kernels, name, f)
    return calls


class _Sublayer(torch.nn.Module):
    """Something nonlinear in a memory or Engram layer's place (whose kernels need a GPU)."""

    def __init__(self, d):
        super().__init__()
        self.w = torch.nn.Parameter(torch.randn(d, d) * 0.4)

    def forward(self, x, *rest):
        return torch.sin(x @ self.w.T)


@pytest.mark.parametrize("memory,second,engram,counts", [((), (), (), (4, 9)), ((1, 2), (2,), (), (2, 10)), ((), (), (0, 3), (4, 9)),
                                                         ((0, 2, 3), (0, 3), (0, 1, 3), (1, 11))])
def test_loss_sums_and_norms_in_forwards_order(memory, second, engram, counts, monkeypatch):
    """Every residual add, norm and sublayer of the kernels' way, with sublayers where memory layers, second reads and Engram
    layers are: the loss and all gradients of forward, in 64 bits (a few thousand roundings of 2^-53 each)."""
    torch.manual_seed(3)
    m = Transformer(ModelConfig(vocab_size=67, d_model=32, n_layers=4, n_heads=2, ffn_hidden=48, max_seq_len=16))
    for i, blk in enumerate(m.layers):
        if i in memory:
            blk.is_memory, blk.ffn = True, _Sublayer(32)
        if i in second:
            blk.ffn_norm_r2, blk.ffn_r2 = torch.nn.RMSNorm(32, eps=1e-5), _Sublayer(32)
        if i in engram:
            blk.engram = _Sublayer(32)
    m.double().train()
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.copy_(p * 4.0 if p.dim() == 2 else p + 0.1 * torch.randn_like(p))
    idx = torch.randint(0, 67, (2, 9), generator=torch.Generator().manual_seed(0))
    t = torch.roll(idx, -1, 1)
    names, params = zip(*m.named_parameters())
    plain = F.cross_entropy(m(idx).view(-1, 67), t.view(-1))
    want = torch.autograd.grad(plain, params)
    calls = _in_64_bits(monkeypatch)
    loss = m.loss(idx, t)
    got = torch.autograd.grad(loss, params)
    assert calls == {"loss": 1, "ffn": counts[0], "norm": counts[1]}
    assert abs(loss.item() - plain.item()) <= 1e-11 * plain.item()
    for n, a, b in zip(names, got, want):
        assert 0 < float(b.norm()) and float((a - b).norm()) <= 1e-9 * float(b.norm()), n


def test_products_of_an_operand_form_that_is_not_there():
    """Contiguous features with strided tokens are refused, not run as another form (smlm::mm_launch of csrc/lm_mm.h)."""
    import ctypes

    class Args(ctypes.Structure):                     # MmArgs, by value on the stack: at least its size
        _fields_ = [("bytes", ctypes.c_int64 * 32)]

    class Plan(ctypes.Structure):
        _fields_ = [("shape", ctypes.c_int), ("splits", ctypes.c_int64)]

    launch = getattr(_lib.lib(), "_ZN4smlm9mm_launchENS_6MmArgsEbbRKNS_6MmPlanEP12ihipStream_tPKc")
    launch.restype = ctypes.c_int
    launch.argtypes = [Args, ctypes.c_bool, ctypes.c_bool, ctypes.POINTER(Plan), ctypes.c_void_p, ctypes.c_char_p]
    assert launch(Args(), True, False, ctypes.byref(Plan(3, 1)), None, b"product") == _lib.EUNSUPPORTED
    assert "strided tokens" in _lib.last_error()
