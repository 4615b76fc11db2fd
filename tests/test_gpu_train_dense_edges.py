"""Edges of the dense training operators on the GPU: default arguments, operands of one row, inputs that depend on each
other, what a backward gets back, replaced and watched sublayers, and every tile of the products.  Tolerances as in
test_gpu_train_dense.py."""
import ctypes
import itertools

import pytest
import torch
import torch.nn.functional as F

from smlm_hip import _lib, kernels
from test_gpu_train_dense import (BF16, DEV, F32, HALF, U32, batch, check_ffn, check_loss, close, ffn_inputs, lm, note, randn,
                                  rounding, run_ffn, run_loss, spied, targets)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- default epsilons
@pytest.mark.parametrize("xt,wt", itertools.product([F32, BF16], repeat=2))
def test_norm_default_eps(xt, wt):
    """nn.RMSNorm(C) without eps adds the epsilon of fp32, the type it computes in, whatever its input's: rows whose mean
    square is about as small tell it from any other."""
    M, C = 9, 40
    norm = torch.nn.RMSNorm(C, device=DEV, dtype=wt)
    x = randn(M, C, std=2.0 ** -11, dtype=xt).requires_grad_()
    g = randn(M, C, seed=4, dtype=xt)
    _, h = kernels.add_rmsnorm_train(x, None, norm)
    dx, dw = torch.autograd.grad(h, (x, norm.weight), g)
    s, w = x.detach().double(), norm.weight.detach().double()
    r = (s.square().mean(1, keepdim=True) + 2.0 ** -23).rsqrt()
    hat, k = s * r, (C + 16) * U32
    close(h.detach(), hat * w, (hat * w).abs() * (rounding(xt) + k) * 1.01, "h")
    close(F.rms_norm(x.detach(), (C,), norm.weight.detach()), hat * w, (hat * w).abs() * (2 * rounding(xt) + k) * 1.01, "torch's")
    gw = g.double() * w
    mean, mean_abs = (gw * hat).mean(1, keepdim=True), (gw * hat).abs().mean(1, keepdim=True)
    ref = (gw - hat * mean) * r
    close(dx, ref, (2 * k * r * (gw.abs() + hat.abs() * mean_abs) + rounding(xt) * ref.abs()) * 1.01, "dx")
    ref = (g.double() * hat).sum(0)
    close(dw, ref, ((g.double() * hat).abs().sum(0) * (M + C + 64) * U32 + rounding(wt) * ref.abs()) * 1.01, "dw")


def test_forward_norms_default_eps():
    """The forward-only norm and the decode linear's: the same bits as with that epsilon given."""
    C = 64
    norm, same = (torch.nn.RMSNorm(C, eps=e, device=DEV, dtype=BF16) for e in (None, 2.0 ** -23))
    x, w = randn(9, C, std=2.0 ** -11), randn(48, C, std=0.1, seed=2)
    assert torch.equal(kernels.add_rmsnorm(x, None, norm)[1], kernels.add_rmsnorm(x, None, same)[1])
    assert torch.equal(kernels.decode_linear(w, x, norm=norm), kernels.decode_linear(w, x, norm=same))
    close(kernels.add_rmsnorm(x, None, norm)[1], F.rms_norm(x.double(), (C,), None, 2.0 ** -23),
          2.0 * HALF * F.rms_norm(x.double(), (C,), None, 2.0 ** -23).abs(), "h")


# ------------------------------------------------------------------------------------------- operands of one row
def row(t):
    """The one row of t as a transposed column: strides (1, 1)."""
    t = t.reshape(-1, 1).contiguous().t()
    assert t.stride() == (1, 1)
    return t


def test_operands_of_one_row_have_any_row_stride():
    """Odd widths, so that the operands are padded: a weight of one row that is a transposed column, and the gradient of a
    sum, whose strides are 0."""
    x, w13, w2, g = ffn_inputs(1, 33, 65, 1)
    assert all(torch.equal(a, b) for a, b in zip(run_ffn(x, w13, w2, g), run_ffn(row(x), w13, row(w2), g)))
    ins = [t.detach().requires_grad_() for t in (x, w13, w2)]
    kernels.gated_ffn(*ins).sum().backward()
    want = run_ffn(x, w13, w2, torch.ones_like(g))[1:]
    assert all(torch.equal(t.grad, b) for t, b in zip(ins, want))
    x, w, t = randn(5, 33), randn(1, 33, std=0.3, seed=2), torch.zeros(5, dtype=torch.int64, device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(run_loss(x, w, t), run_loss(x, row(w), t)))


# --------------------------------------------------------------------------- inputs that depend on each other
@pytest.mark.parametrize("create", [False, True])
def test_loss_gradient_of_hidden_states_that_depend_on_the_weight(create):
    """Tied embeddings: the recorded gradient counts the way through the hidden states once, as the other does."""
    w = randn(20, 16, std=0.3, seed=2).requires_grad_()
    t, pick = targets(9, 20), targets(9, 20, seed=7)
    got, = torch.autograd.grad(kernels.linear_cross_entropy(2 * w[pick], w, t), w, create_graph=create)
    wd = w.detach().double().requires_grad_()
    ref, = torch.autograd.grad(F.cross_entropy(2 * wd[pick] @ wd.T, t), wd, create_graph=True)
    # bf16 roundings of dx, dw, their sum and of the rows that are picked more than once, each at most 2^-8
    assert float((got.double() - ref).norm() / ref.norm()) <= 8 * HALF
    if create:
        got, = torch.autograd.grad(got.float().square().sum(), w)
        ref, = torch.autograd.grad(ref.square().sum(), wd)
        assert float((got.double() - ref).norm() / ref.norm()) <= 16 * HALF


@pytest.mark.parametrize("create", [False, True])
def test_ffn_gradient_of_inputs_that_depend_on_each_other(create):
    """Input and second weight from the first one."""
    w13, g = randn(48, 16, std=0.3, seed=1).requires_grad_(), randn(9, 16, std=0.1, seed=3)
    got, = torch.autograd.grad(kernels.gated_ffn(4 * w13[:9], w13, w13[:24].t()), w13, g, create_graph=create)
    wd = w13.detach().double().requires_grad_()
    a, b = (4 * wd[:9] @ wd.T).chunk(2, 1)
    ref, = torch.autograd.grad((F.silu(a) * b) @ wd[:24], wd, g.double())
    assert float((got.double() - ref).norm() / ref.norm()) <= 8 * HALF


# -------------------------------------------------------------------------------------- what a backward gets back
def operators(odd):
    """Each operator with leaves and a gradient of its output; odd: sizes whose copies are saved too."""
    n = 33 if odd else 32
    x, w, t = randn(9, n), randn(40, n, std=0.3, seed=2), targets(9, 40)
    y, w13, w2, g = ffn_inputs(9, n, 25 if odd else 24, n)
    s, norm = randn(9, n, dtype=F32), torch.nn.RMSNorm(n, eps=1e-5, device=DEV)
    made = {"mean": ([x, w], lambda a: kernels.linear_cross_entropy(*a, t), torch.tensor(1.5, device=DEV)),
            "none": ([x, w], lambda a: kernels.linear_cross_entropy(*a, t, reduction="none"), randn(9, dtype=F32)),
            "ffn": ([y, w13, w2], lambda a: kernels.gated_ffn(*a), g),
            "norm": ([s, norm.weight], lambda a: kernels.add_rmsnorm_train(a[0], a[0], norm)[1], randn(9, n, seed=7, dtype=F32))}
    return {k: ([i.detach().requires_grad_() if i is not norm.weight else i for i in ins], f, g) for k, (ins, f, g) in made.items()}


CHANGES = {"host": lambda t: t.cpu(), "type": lambda t: t.double() if t.dtype == F32 else t.float(),
           "fewer": lambda t: t[:-1] if t.dim() else t[None], "flat": lambda t: t.reshape(-1)[None]}


@pytest.mark.parametrize("name,odd,change,create", itertools.product(["mean", "none", "ffn", "norm"], [False, True], CHANGES,
                                                                     [False, True]))
def test_saved_tensors_that_come_back_changed_are_refused(name, odd, change, create):
    """One saved tensor after the other comes back on the host, in another type or with other sizes."""
    note(name, odd, change, create)
    for k in itertools.count():
        count = itertools.count()
        ins, f, g = operators(odd)[name]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(count), t.detach()),
                                                      lambda p: CHANGES[change](p[1]) if p[0] == k else p[1]):
            out = f(ins)
        if k >= next(count):
            assert k > 0
            break
        with pytest.raises((RuntimeError, ValueError)):
            torch.autograd.grad(out, ins, g, create_graph=create)


@pytest.mark.parametrize("name,odd", itertools.product(["mean", "none", "ffn", "norm"], [False, True]))
def test_saved_tensors_that_come_back_elsewhere(name, odd):
    """From host memory, or in other strides: the same bits."""
    ins, f, g = operators(odd)[name]
    want = torch.autograd.grad(f(ins), ins, g)

    def turned(t):
        return t if t.dim() < 2 else t.repeat_interleave(2, 1)[:, ::2]

    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), turned)):
        with hooks:
            out = f(ins)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, ins, g), want))


def test_leaves_replaced_between_the_passes_are_refused():
    """A model moved to another type, or weights freed, after the forward pass."""
    for name, (ins, f, g) in operators(False).items():
        for i, new in itertools.product(range(len(ins)), (lambda t: t.to(BF16 if t.dtype == F32 else F32), lambda t: t[:0])):
            ins, f, g = operators(False)[name]
            out = f(ins)
            if name == "norm" and (i == 0 or new(ins[1]).numel()):
                continue                                 # the stream is kept as it was formed; weights of either type are read
            ins[i].data = new(ins[i].data)
            with pytest.raises((RuntimeError, ValueError)):
                torch.autograd.grad(out, ins, g)


# ------------------------------------------------------------------------- Transformer.loss and its sublayers
class Seen(torch.nn.Module):
    """A sublayer put in another's place, which notes its input's type."""

    def __init__(self, inner, types):
        super().__init__()
        self.inner, self.types = inner, types

    def forward(self, x, *rest):
        self.types.append(x.dtype)
        return self.inner(x, *rest)


class SeenLinear(torch.nn.Linear):
    def forward(self, x):
        self.types.append(x.dtype)
        return super().forward(x)


@pytest.mark.parametrize("how", ["watched", "projection watched", "replaced", "projection replaced"])
def test_model_loss_gives_other_attention_the_streams_type(how):
    """Under autocast the stream is fp32: what watches the attention's input or takes its place sees what forward gives."""
    m, types = lm(F32), []
    idx, t = batch()
    blk = m.layers[1]

    def see(module, args):
        types.append(args[0].dtype)

    if how == "watched":
        blk.attn.register_forward_pre_hook(see)
    elif how == "projection watched":
        blk.attn.wqkv.register_forward_pre_hook(see)
    elif how == "replaced":
        blk.attn = Seen(blk.attn, types)
    else:
        blk.attn.wqkv.__class__, blk.attn.wqkv.types = SeenLinear, types
    with torch.autocast("cuda", dtype=BF16):
        loss = m.loss(idx, t)
        _, plain = m(idx, t)
    assert types == [F32, F32]
    assert abs(loss.item() - plain.item()) <= 0.03 * plain.item()


def test_model_loss_targets_of_other_shapes_and_types(monkeypatch):
    """Targets as forward takes them: flat ones count for the tokens in order, and losses come in the targets' shape; what
    is not int64 goes the modules' way."""
    m = lm(BF16)
    idx, t = batch()
    calls = spied(monkeypatch)
    each = m.loss(idx, t, reduction="none")
    flat = m.loss(idx, t.view(-1), reduction="none")
    assert flat.shape == (t.numel(),) and torch.equal(flat, each.view(-1))
    assert torch.equal(m.loss(idx, t.view(-1)), m.loss(idx, t))
    assert calls["linear_cross_entropy"] == 4
    small = t.clamp(0, 255).to(torch.uint8)
    assert torch.equal(m.loss(idx, small), m(idx, small)[1])
    for bad in (t[:2], t.int()):
        with pytest.raises((ValueError, RuntimeError)):
            m.loss(idx, bad)


class Gives(torch.nn.Module):
    def __init__(self, value):
        super().__init__()
        self.value = torch.nn.Parameter(value) if torch.is_tensor(value) else value

    def forward(self, x, *rest):
        return self.value


def test_model_loss_with_sublayers_that_give_less_than_the_stream():
    """A sublayer that is switched off (0), or gives one row for all tokens: added as forward adds it."""
    m = lm(BF16)
    idx, t = batch()
    m.layers[0].attn, m.layers[1].ffn = Gives(0.0), Gives(randn(128))
    m.layers[2].ffn = Gives(randn(1, 33, 128, seed=3))
    loss, (_, plain) = m.loss(idx, t), m(idx, t)
    assert abs(loss.item() - plain.item()) <= 0.03 * plain.item()
    for blk in m.layers[1:]:
        v = blk.ffn.value
        got, want = (torch.autograd.grad(x, v, retain_graph=True)[0].double() for x in (loss, plain))
        # either path within the bf16 roundings of two layers and the loss, forward and back
        assert float((got - want).norm() / want.norm()) <= 32 * HALF


# --------------------------------------------------------------------------------- every tile of the products
class Plan(ctypes.Structure):
    _fields_ = [("shape", ctypes.c_int), ("splits", ctypes.c_int64)]


def plan(T, F, K, may_split):
    """The library's own choice (smlm::mm_plan of csrc/lm_mm.h)."""
    f = getattr(_lib.lib(), "_ZN4smlm7mm_planElllb")
    f.restype, f.argtypes = Plan, [ctypes.c_int64] * 3 + [ctypes.c_bool]
    p = f(T, F, K, may_split)
    return ("256 x 256", "384 x 128", "128 x 128", "64 x 64")[p.shape], p.splits > 1


def up(n, to=8):
    return -(-n // to) * to


def terms(M):
    return 2 if M <= 128 else 1


def loss_tiles(M, V, d):
    """(operands with contiguous k, tile, whether k is split, terms) of the loss' two products."""
    cols, d = up(V, 256), up(d)
    return {("tokens", *plan(M, d, cols, True), terms(M)), ("none", *plan(cols, d, M, False), terms(M))}


def ffn_tiles(M, d, h, o):
    """Of the block's four."""
    n, (d, h, o) = terms(M), map(up, (d, h, o))
    return {("both", *plan(M, o, h * n, True), n), ("tokens", *plan(M, d, 2 * h * n, True), n),
            ("none", *plan(2 * h, d, M * n, True), n), ("none", *plan(o, h, M * n, True), n)}


LOSS_TILES = [(64, 32000, 384), (2031, 32003, 201), (4096, 20011, 392), (2, 24157, 3393)]
FFN_TILES = [(2, 35, 36, 46), (70, 42, 2594, 2701), (76, 1794, 3641, 40), (312, 2128, 2885, 3336), (870, 73, 409, 50),
             (1347, 43, 3419, 1979), (7591, 524, 1643, 42), (14074, 33, 3882, 130), (14077, 392, 1001, 392),
             (15192, 535, 145, 779), (16318, 897, 286, 614), (32801, 384, 1024, 384)]


def test_the_sizes_below_take_every_tile():
    """Every tile in every form of operands with a bf16 result and, where a plan may split k, with fp32 parts; with two terms
    those that so few tokens take."""
    seen = set().union(*(loss_tiles(*s) for s in LOSS_TILES), *(ffn_tiles(*s) for s in FFN_TILES))
    tiles = ("256 x 256", "384 x 128", "128 x 128", "64 x 64")
    missing = set(itertools.product(("both", "tokens", "none"), tiles, (False, True), (1,))) - seen
    assert not missing
    two = {("both", "64 x 64", False), ("both", "64 x 64", True), ("both", "128 x 128", True), ("tokens", "64 x 64", False),
           ("tokens", "64 x 64", True), ("tokens", "128 x 128", True), ("tokens", "384 x 128", True),
           *(("none", t, False) for t in tiles)}
    assert {k[:3] for k in seen if k[3] == 2} >= two


@pytest.mark.parametrize("M,V,d", LOSS_TILES)
def test_loss_tiles(M, V, d):
    note("loss", M, V, d)
    check_loss(randn(M, d), randn(V, d, std=4.0 / d ** 0.5, seed=2), targets(M, V, ignored=0.1))


@pytest.mark.parametrize("M,d,h,o", FFN_TILES)
def test_ffn_tiles(M, d, h, o):
    note("ffn", M, d, h, o)
    check_ffn(*ffn_inputs(M, d, h, o))


@pytest.mark.parametrize("M", [200, 300, 1111])
def test_loss_weights_of_single_tokens(M):
    """A coefficient per token in the loss' tiles of 128 and 256 tokens; an ignored token's may be NaN."""
    V, d = 1500, 136
    note("loss", M, V, d)
    t, g = targets(M, V, ignored=0.2), randn(M, seed=5, dtype=F32)
    want = check_loss(randn(M, d), randn(V, d, std=0.3, seed=2), t, "none", g=g)
    g[t == -100] = float("nan")
    got = run_loss(randn(M, d), randn(V, d, std=0.3, seed=2), t, "none", g=g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
