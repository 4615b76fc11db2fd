"""The dense operators of a training step on the GPU (linear_cross_entropy, gated_ffn, add_rmsnorm_train) against their
definitions in 64 bits.  Tolerances are element by element, from the roundings that the operators document: a bf16
rounding moves a value by at most 2^-8 of it, so a product whose one operand G is rounded is off by at most 2^-8 |G| |W|, its
own rounding by 2^-8 of itself; fp32 sums of n products by n 2^-24 of the absolute products."""
import itertools

import pytest
import torch
import torch.nn.functional as F

from smlm_hip import kernels
from smlm_hip.capture import capture

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32
HALF = 2.0 ** -8                 # a bf16 rounding, relative
U32 = 2.0 ** -24                 # an fp32 one
# The smallest normal number of fp32 and bf16 both: the exponential and the matrix cores flush what is smaller, so that
# an element of G below it may count as zero (an error of at most TINY, times the other operand) and so may a result.
TINY = 2.0 ** -126


def half_between(tokens):
    """The rounding of what the products read back: up to 128 tokens as two bf16 terms, the second rounding what the first
    leaves."""
    return HALF * HALF if tokens <= 128 else HALF


def note(*what):
    print("[case]", *what, flush=True)


def randn(*shape, std=1.0, seed=0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def close(got, ref, tol, what):
    err = (got.double() - ref).abs() - tol
    at = err.argmax() if err.numel() else None
    assert err.numel() == 0 or float(err.max()) <= 0, \
        f"{what}: {got.flatten()[at].item()} against {ref.flatten()[at].item()}, allowed {tol.expand_as(ref).flatten()[at].item()}"


# ------------------------------------------------------------------------------------------------- the loss
def loss_reference(x, w, t, ignore=-100, reduction="mean", g=None):
    """Loss, gradients and their tolerances in 64 bits (x (M, d), w (V, d), t (M,), g the loss' gradient)."""
    x, w = x.double(), w.double()
    logits = x @ w.T
    size = (x.abs() @ w.abs().T).amax(1)
    lse = torch.logsumexp(logits, 1)
    valid = t != ignore
    at = torch.where(valid, t, 0).unsqueeze(1)
    each = torch.where(valid, lse - logits.gather(1, at).squeeze(1), 0.0)
    logit_err = (x.shape[1] + 32) * U32 * size           # a logit's, and with it the exponent's of every probability
    each_tol = torch.where(valid, 2 * logit_err + 16 * U32 * (1 + lse.abs()), 0.0)
    n = valid.sum()
    loss, tol = {"none": (each, each_tol), "sum": (each.sum(), each_tol.sum()),
                 "mean": (each.sum() / n, each_tol.sum() / n)}[reduction]
    tol = tol + 2 * U32 * loss.abs()
    c = valid.double() * (1.0 if g is None else g.double())
    if reduction == "mean":
        c = c / n
    p = torch.exp(logits - lse.unsqueeze(1))
    G = c.unsqueeze(1) * p.scatter_add(1, at, -torch.ones_like(at, dtype=torch.float64))
    G_tol = TINY + half_between(x.shape[0]) * G.abs() + c.abs().unsqueeze(1) * p * (2 * logit_err.unsqueeze(1) + 32 * U32) * 1.01
    dx, dw = G @ w, G.T @ x
    k = (w.shape[0] + 64) * U32
    dx_tol = (G_tol + k * G.abs()) @ w.abs() * 1.01 + HALF * dx.abs() * 1.01 + TINY
    k = (x.shape[0] + 64) * U32
    dw_tol = (G_tol + k * G.abs()).T @ x.abs() * 1.01 + HALF * dw.abs() * 1.01 + TINY
    return (loss, tol), (dx, dx_tol), (dw, dw_tol)


def run_loss(x, w, t, reduction="mean", ignore=-100, g=None):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = kernels.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    return loss.detach(), dx, dw


def check_loss(x, w, t, reduction="mean", ignore=-100, g=None):
    d = x.shape[-1]
    loss, dx, dw = run_loss(x, w, t, reduction, ignore, g)
    gf = None if g is None else g.reshape(-1)
    (l, lt), (rx, xt), (rw, wt) = loss_reference(x.reshape(-1, d), w, t.reshape(-1), ignore, reduction, gf)
    assert loss.dtype == F32 and dx.dtype == dw.dtype == BF16 and dx.shape == x.shape and dw.shape == w.shape
    close(loss.reshape(l.shape), l, lt, "loss")
    close(dx.reshape(-1, d), rx, xt, "dx")
    close(dw, rw, wt, "dw")
    return loss, dx, dw


def targets(M, V, seed=1, ignored=0.0, ignore=-100):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (M,), generator=g)
    t[torch.rand(M, generator=g) < ignored] = ignore
    return t.to(DEV)


@pytest.mark.parametrize("M,V,d", [(1, 1, 8), (1, 2, 1), (1, 1000, 384), (2, 127, 32), (63, 128, 64), (64, 129, 31),
                                   (65, 500, 40), (128, 1001, 72), (129, 1025, 201), (200, 640, 384), (256, 4096, 256),
                                   (257, 3001, 136), (700, 2050, 100), (1000, 32003, 64)])
def test_loss_sizes(M, V, d):
    note("loss", M, V, d)
    check_loss(randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V))


@pytest.mark.parametrize("reduction,ignored", itertools.product(["mean", "sum", "none"], [0.0, 0.4, 1.0]))
def test_loss_reductions(reduction, ignored):
    note("loss", reduction, ignored)
    M, V, d = 150, 777, 96
    t = targets(M, V, ignored=ignored)
    g = randn(M, seed=5, dtype=F32) if reduction == "none" else torch.tensor(1.75, device=DEV)
    if ignored == 1.0:
        loss, dx, dw = run_loss(randn(M, d), randn(V, d, std=0.3, seed=2), t, reduction, g=g)
        assert torch.isnan(loss).all() if reduction == "mean" else torch.equal(loss, torch.zeros_like(loss))
        assert not dx.any() and not dw.any()
        return
    check_loss(randn(M, d), randn(V, d, std=0.3, seed=2), t, reduction, g=g)


def test_loss_other_ignore_index_and_leading_shape():
    x, w, t = randn(3, 5, 7, 48), randn(300, 48, std=0.3, seed=2), targets(105, 300, ignored=0.3, ignore=0).view(3, 5, 7)
    loss, dx, dw = check_loss(x, w, t, "none", ignore=0, g=randn(3, 5, 7, dtype=F32).abs())
    assert loss.shape == t.shape and not loss[t == 0].any() and not dx[t == 0].any()


def test_loss_of_one_token_without_a_dimension():
    x, w, t = randn(48), randn(300, 48, std=0.3, seed=2), torch.tensor(7, device=DEV)
    loss, dx, _ = check_loss(x, w, t)
    assert loss.shape == () and dx.shape == (48,)


@pytest.mark.parametrize("layout", ["rows", "columns", "offset", "transposed"])
def test_loss_strided_operands(layout):
    """Rows apart are read as they are; other layouts are copied."""
    M, V, d = 90, 400, 64

    def lay(t):
        if layout == "rows":
            return torch.cat([t, t + 1], 1)[:, :d]
        if layout == "columns":
            return t.repeat_interleave(2, 1)[:, ::2]
        if layout == "offset":
            return torch.cat([t[:, :1], t], 1)[:, 1:]
        return t.T.contiguous().T

    x, w, t = randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V)
    a, b = run_loss(x, w, t), run_loss(lay(x), lay(w), torch.stack([t, t], 1)[:, 0])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_loss_in_several_pieces_of_the_vocabulary():
    """More than 1 GiB of logits' gradient: 57,000 tokens x 10,000 columns in two pieces."""
    M, V, d = 57000, 10000, 16
    note("loss", M, V, d)
    check_loss(randn(M, d), randn(V, d, std=0.5, seed=2), targets(M, V, ignored=0.1))


def test_loss_of_few_tokens_over_a_very_large_vocabulary():
    """Two pieces of at most 2^21 columns: the products take no wider rows."""
    M, V, d = 3, (1 << 21) + 300, 8
    note("loss", M, V, d)
    t = targets(M, V)
    t[1] = V - 1
    check_loss(randn(M, d), randn(V, d, std=0.5, seed=2), t)


def test_loss_excluded_vocabulary_row():
    """A row whose logit is -inf for every token counts for nothing; as a target its loss is inf and the gradients of all
    rows are still finite: softmax - 1 at the target."""
    M, V, d = 40, 300, 32
    x, w, t = randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V)
    t[t == 5] = 6
    x[:, 0], w[5, 0] = 1.0, float("-inf")
    w[5, 1:] = 0
    t[7] = 5
    loss, _, dw = run_loss(x, w, t, "none", g=torch.ones(M, device=DEV))
    kept = torch.arange(V, device=DEV) != 5
    others = torch.where(t == 5, -100, t - (t > 5).long())
    (l, lt), _, (rw, wt) = loss_reference(x, w[kept], others, -100, "none", torch.ones(M, device=DEV))
    assert torch.isposinf(loss[7])
    close(torch.where(t == 5, 0.0, loss), l, lt, "loss")
    p = torch.softmax(x[7].double() @ w[kept].double().T, 0)
    more = p.unsqueeze(1) * x[7].double()              # the excluded target's token: its probabilities, no 1 among the kept
    close(dw[kept], rw + more, wt + 2 * HALF * (more.abs() + rw.abs()) + 2.0 ** -12 * more.abs() + TINY, "dw")
    assert torch.equal(dw[5], -x[7])


def test_loss_large_logits_and_certain_tokens():
    """Logits of thousands: probabilities of exactly 1 and 0; no overflow, a loss of 0 and no gradient where the target has
    all of it."""
    M, V, d = 70, 600, 32
    x, w = randn(M, d, std=40.0), randn(V, d, std=20.0, seed=2)
    best = (x.double() @ w.double().T).argmax(1)
    loss, dx, dw = run_loss(x, w, best, "none", g=torch.ones(M, device=DEV))
    assert torch.isfinite(loss).all() and float(loss.min()) >= 0
    check_loss(x, w, targets(M, V), "none", g=torch.ones(M, device=DEV))
    check_loss(x, w, best, "mean")


def test_loss_infinite_and_nan_rows_stay_their_own():
    M, V, d = 80, 300, 32
    x, w, t = randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V)
    clean = kernels.linear_cross_entropy(x, w, t, reduction="none")
    x[3, 5], x[9, 0] = float("nan"), float("inf")
    loss = kernels.linear_cross_entropy(x, w, t, reduction="none")
    bad = torch.zeros(M, dtype=torch.bool, device=DEV)
    bad[3] = bad[9] = True
    assert torch.isnan(loss[bad]).all() and torch.equal(loss[~bad], clean[~bad])


def test_loss_targets_outside_the_vocabulary_are_nan():
    M, V, d = 40, 200, 32
    x, w, t = randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V)
    t[4], t[17], t[30] = V, -1, 1 << 40
    loss, dx, _ = run_loss(x, w, t, "none", g=torch.ones(M, device=DEV))
    bad = torch.zeros(M, dtype=torch.bool, device=DEV)
    bad[[4, 17, 30]] = True
    assert torch.isnan(loss[bad]).all() and torch.isfinite(loss[~bad]).all()
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_without_tokens(reduction):
    x, w = randn(0, 16).requires_grad_(), randn(30, 16).requires_grad_()
    loss = kernels.linear_cross_entropy(x, w, torch.empty(0, dtype=torch.int64, device=DEV), reduction=reduction)
    assert torch.isnan(loss) if reduction == "mean" else not loss.sum()
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    assert dx.shape == x.shape and not dw.any()


def test_loss_partial_gradients_and_no_grad():
    x, w, t = randn(70, 64), randn(333, 64, std=0.3, seed=2), targets(70, 333)
    loss, dx, dw = run_loss(x, w, t)
    only_x = torch.autograd.grad(kernels.linear_cross_entropy(x.requires_grad_(), w, t), x)[0]
    only_w = torch.autograd.grad(kernels.linear_cross_entropy(x.detach(), w.requires_grad_(), t), w)[0]
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    with torch.no_grad():
        again = kernels.linear_cross_entropy(x, w, t)
    assert torch.equal(again, loss) and not again.requires_grad


def test_loss_gradient_against_differences():
    """The gradient's step along itself changes the loss by its squared length (bf16 inputs, steps of whole bf16 values)."""
    M, V, d = 64, 300, 64
    x, w, t = randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V)
    _, dx, dw = run_loss(x, w, t, "sum", g=torch.tensor(1.0, device=DEV))
    for i, grad in ((0, dx), (1, dw)):
        step = (2.0 ** -5 * grad.float() / grad.float().norm()).to(BF16).float()
        ops = [[x.float(), w.float()], [x.float(), w.float()]]
        ops[0][i], ops[1][i] = ops[0][i] + step, ops[1][i] - step
        up, down = ((F.cross_entropy(a.double() @ b.double().T, t, reduction="sum")) for a, b in ops)
        # third order in the step, and the gradient's own roundings
        assert abs(float(up - down) / 2 - float((grad.float() * step).sum())) <= 0.01 * float(up - down) / 2


def test_loss_same_bits_and_other_stream():
    M, V, d = 500, 5000, 128
    x, w, t = randn(M, d), randn(V, d, std=0.3, seed=2), targets(M, V, ignored=0.2)
    first = run_loss(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run_loss(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    third = run_loss(x, w, t)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, second, third))


def test_loss_recorded_gradient():
    """create_graph differentiates the PyTorch ops: the gradient's gradient of a small loss."""
    x, w, t = randn(6, 16).requires_grad_(), randn(20, 16, std=0.3, seed=2).requires_grad_(), targets(6, 20)
    dx, = torch.autograd.grad(kernels.linear_cross_entropy(x, w, t), x, create_graph=True)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    rx, = torch.autograd.grad(F.cross_entropy(xd @ wd.T, t), xd, create_graph=True)
    got, = torch.autograd.grad(dx.float().square().sum(), w)
    ref, = torch.autograd.grad(rx.square().sum(), wd)
    assert float((got.double() - ref).norm() / ref.norm()) <= 0.02


def test_loss_recorded_gradient_of_targets_outside_the_vocabulary():
    x, w, t = randn(6, 16).requires_grad_(), randn(20, 16, std=0.3, seed=2).requires_grad_(), targets(6, 20)
    t[2], t[4] = 20, -7
    for create in (False, True):
        dx, = torch.autograd.grad(kernels.linear_cross_entropy(x, w, t, reduction="sum"), x, create_graph=create)
        assert torch.isnan(dx[[2, 4]]).all() and torch.isfinite(dx[[0, 1, 3, 5]]).all()


def test_recorded_gradients_keep_fp32_under_autocast():
    x, w, t = randn(6, 16).requires_grad_(), randn(20, 16, std=0.3, seed=2).requires_grad_(), targets(6, 20)
    y, w13, w2, g = ffn_inputs(9, 16, 24, 16)
    y = y.requires_grad_()
    got = []
    for on in (False, True):
        with torch.autocast("cuda", dtype=BF16, enabled=on):
            got.append(torch.autograd.grad(kernels.linear_cross_entropy(x, w, t), (x, w), create_graph=True)
                       + torch.autograd.grad(kernels.gated_ffn(y, w13, w2), y, g, create_graph=True))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ---------------------------------------------------------------------------------------------- the FFN block
def ffn_reference(x, w13, w2, g):
    x, w13, w2, g = (t.double() for t in (x, w13, w2, g))
    d, h, M = x.shape[1], w2.shape[1], x.shape[0]
    a, b = (x @ w13.T).chunk(2, 1)
    ea, eb = ((x.abs() @ w13.abs().T) * (d + 4) * U32).chunk(2, 1)
    s = torch.sigmoid(a)
    act, ds = a * s, s + a * s * (1 - s)
    hid = act * b
    # |silu'| <= 1.1 and |silu''| <= 0.5; 2^-20 for the sigmoid
    act_tol = 1.1 * ea + 2.0 ** -20 * act.abs()
    half = half_between(M)
    hid_tol = TINY + half * hid.abs() + 1.01 * (act_tol * b.abs() + act.abs() * eb)
    dh = g @ w2
    dh_err = (g.abs() @ w2.abs()) * (w2.shape[0] + 4) * U32
    dab = torch.cat([dh * b * ds, dh * act], 1)
    ds_tol = 0.5 * ea + 2.0 ** -20 * (s + a.abs())
    dab_tol = TINY + half * dab.abs() + 1.01 * torch.cat([dh_err * (b * ds).abs() + (dh * b).abs() * ds_tol + (dh * ds).abs() * eb,
                                                   dh_err * act.abs() + dh.abs() * act_tol], 1)

    def product(p, tol, q, n):
        ref = p @ q
        return ref, 1.01 * ((tol + (n + 64) * U32 * p.abs()) @ q.abs() + HALF * ref.abs())

    return (product(hid, hid_tol, w2.T, h), product(dab, dab_tol, w13, 2 * h),
            product(dab.T, dab_tol.T, x, M), tuple(t.T for t in product(hid.T, hid_tol.T, g, M)))


def run_ffn(x, w13, w2, g):
    ins = [t.detach().requires_grad_() for t in (x, w13, w2)]
    y = kernels.gated_ffn(*ins)
    return (y.detach(), *torch.autograd.grad(y, ins, g))


def check_ffn(x, w13, w2, g):
    got = run_ffn(x, w13, w2, g)
    ref = ffn_reference(x.reshape(-1, x.shape[-1]), w13, w2, g.reshape(-1, g.shape[-1]))
    for name, t, (r, tol), like in zip(("y", "dx", "dw13", "dw2"), got, ref, (g, x, w13, w2)):
        assert t.shape == like.shape and t.dtype == BF16
        close(t.reshape(r.shape), r, tol, name)
    return got


def ffn_inputs(M, d, h, o, seed=0):
    return (randn(M, d, seed=seed), randn(2 * h, d, std=1.2 / d ** 0.5, seed=seed + 1),
            randn(o, h, std=h ** -0.5, seed=seed + 2), randn(M, o, std=0.1, seed=seed + 3))


@pytest.mark.parametrize("M,d,h,o", [(1, 8, 8, 8), (1, 1, 1, 1), (1, 384, 1024, 384), (3, 33, 65, 17), (48, 384, 1024, 384),
                                     (63, 64, 64, 64), (64, 40, 72, 40), (65, 72, 200, 136), (129, 100, 130, 100),
                                     (256, 384, 1000, 384), (700, 392, 1001, 200), (1111, 256, 512, 256),
                                     (4096, 128, 640, 128), (9000, 64, 1024, 72)])
def test_ffn_sizes(M, d, h, o):
    note("ffn", M, d, h, o)
    check_ffn(*ffn_inputs(M, d, h, o))


def test_ffn_leading_shape_and_strides():
    x, w13, w2, g = ffn_inputs(60, 64, 72, 48)
    want = check_ffn(x.view(3, 4, 5, 64), w13, w2, g.view(3, 4, 5, 48))
    wide = lambda t: torch.cat([t, t], 1)[:, :t.shape[1]]  # noqa: E731
    shifted = lambda t: torch.cat([t[:, :1], t], 1)[:, 1:]  # noqa: E731
    turned = lambda t: t.T.contiguous().T  # noqa: E731
    for lay in (wide, shifted, turned):
        got = run_ffn(lay(x), lay(w13), lay(w2), lay(g))
        assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(want, got))


def test_ffn_of_one_vector_and_of_none():
    x, w13, w2, g = ffn_inputs(1, 64, 72, 48)
    got = run_ffn(x[0], w13, w2, g[0])
    assert got[0].shape == (48,) and got[1].shape == (64,)
    got = run_ffn(x[:0], w13, w2, g[:0])
    assert got[0].shape == (0, 48) and not got[2].any() and not got[3].any()


def test_ffn_partial_gradients_and_same_bits():
    x, w13, w2, g = ffn_inputs(300, 128, 200, 96)
    y, dx, dw13, dw2 = run_ffn(x, w13, w2, g)
    for i, want in ((0, dx), (1, dw13), (2, dw2)):
        ins = [t.detach() for t in (x, w13, w2)]
        ins[i].requires_grad_()
        out = kernels.gated_ffn(*ins)
        assert torch.equal(out, y) and torch.equal(torch.autograd.grad(out, ins[i], g)[0], want)
    with torch.no_grad():
        assert torch.equal(kernels.gated_ffn(x, w13, w2), y)


def test_ffn_saturated_gates():
    """Pre-activations far on either side of the sigmoid's range: no overflow, gates of exactly 0 and 1."""
    x, w13, w2, g = ffn_inputs(100, 64, 128, 64)
    y, dx, dw13, dw2 = run_ffn(x * 64, w13 * 8, w2, g)
    assert all(torch.isfinite(t).all() for t in (y, dx, dw13, dw2))
    check_ffn(x * 64, w13 * 8, w2, g)


def test_ffn_nan_stays_in_its_row():
    x, w13, w2, g = ffn_inputs(100, 64, 128, 64)
    y, dx, _, _ = run_ffn(x, w13, w2, g)
    x[7, 3] = float("nan")
    y2, dx2, _, _ = run_ffn(x, w13, w2, g)
    keep = torch.arange(100, device=DEV) != 7
    assert torch.isnan(y2[7]).all() and torch.equal(y2[keep], y[keep]) and torch.equal(dx2[keep], dx[keep])


def test_ffn_recorded_gradient():
    x, w13, w2, g = ffn_inputs(9, 16, 24, 16)
    ins = [t.detach().requires_grad_() for t in (x, w13, w2)]
    dx, = torch.autograd.grad(kernels.gated_ffn(*ins), ins[0], g, create_graph=True)
    got, = torch.autograd.grad(dx.float().square().sum(), ins[1])
    dbl = [t.detach().double().requires_grad_() for t in (x, w13, w2)]
    a, b = (dbl[0] @ dbl[1].T).chunk(2, 1)
    rx, = torch.autograd.grad((F.silu(a) * b) @ dbl[2].T, dbl[0], g.double(), create_graph=True)
    ref, = torch.autograd.grad(rx.square().sum(), dbl[1])
    assert float((got.double() - ref).norm() / ref.norm()) <= 0.02


# ---------------------------------------------------------------------------------------------------- the norm
def norm_of(C, dtype, seed=9, eps=1e-5):
    n = torch.nn.RMSNorm(C, eps=eps, device=DEV, dtype=dtype)
    with torch.no_grad():
        n.weight.copy_(randn(C, seed=seed, dtype=F32).abs() + 0.5)
    return n


def run_norm(x, delta, norm, out, gx, gh):
    ins = [x.detach().requires_grad_(), None if delta is None else delta.detach().requires_grad_(), norm.weight]
    xs, h = kernels.add_rmsnorm_train(ins[0], ins[1], norm, out_dtype=out)
    outs = [(o, g) for o, g in ((xs, gx), (h, gh)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], [t for t in ins if t is not None], [g for _, g in outs])
    return xs.detach(), h.detach(), got


def rounding(dtype):
    return HALF if dtype == BF16 else U32


def check_norm(M, C, xt, dt, wt, ht, with_gx=True, with_gh=True):
    x, delta = randn(M, C, std=2.0, dtype=xt), None if dt is None else randn(M, C, seed=3, dtype=dt)
    norm = norm_of(C, wt)
    gx = randn(M, C, seed=4, dtype=xt) if with_gx else None
    gh = randn(M, C, seed=5, dtype=ht) if with_gh else None
    xs, h, got = run_norm(x, delta, norm, ht, gx, gh)
    if delta is None:
        assert torch.equal(xs, x)
    else:
        assert torch.equal(xs, (x.float() + delta.float()).to(xt))
    assert xs.dtype == xt and h.dtype == ht
    s, w = xs.double(), norm.weight.detach().double()
    r = (s.square().mean(1, keepdim=True) + norm.eps).rsqrt()
    hat = s * r
    k = (C + 16) * U32                                        # the sum of the squares, halved by the root, and the rest
    close(h, hat * w, (hat * w).abs() * (rounding(ht) + k) * 1.01, "h")
    gh = torch.zeros_like(s) if gh is None else gh.double()
    res = torch.zeros_like(s) if gx is None else gx.double()
    gw = gh * w
    mean, mean_abs = (gw * hat).mean(1, keepdim=True), (gw * hat).abs().mean(1, keepdim=True)
    dx = (gw - hat * mean) * r + res
    tol = 2 * k * r * (gw.abs() + hat.abs() * mean_abs) + 4 * U32 * res.abs()
    close(got[0], dx, (tol + rounding(xt) * dx.abs()) * 1.01, "dx")
    dw, n = (gh * hat).sum(0), (M + C + 64) * U32
    close(got[-1], dw, ((gh * hat).abs().sum(0) * n + rounding(wt) * dw.abs()) * 1.01, "dw")
    if delta is not None:
        close(got[1], dx, (tol + rounding(dt) * dx.abs()) * 1.01, "ddelta")


TYPES = [(F32, BF16, F32, BF16), (F32, F32, F32, F32), (F32, None, BF16, F32), (BF16, BF16, BF16, BF16),
         (BF16, None, F32, BF16), (BF16, BF16, F32, F32)]


@pytest.mark.parametrize("M,C", [(1, 1), (1, 384), (2, 7), (5, 8), (64, 384), (33, 511), (9, 512), (17, 513), (300, 1001),
                                 (11, 1024), (7, 1025), (20, 2048), (6, 2049), (5, 4097), (3, 16384), (4097, 392),
                                 (20000, 24), (70, 9), (33, 64), (3, 100), (130, 128), (1000, 129), (9, 255), (41, 257),
                                 (2, 1500), (5, 4104), (7, 8191), (4, 8200), (3, 16383)])
def test_norm_sizes(M, C):
    note("norm", M, C)
    for types in TYPES:
        check_norm(M, C, *types)


@pytest.mark.parametrize("with_gx,with_gh", [(False, True), (True, False)])
@pytest.mark.parametrize("types", TYPES)
def test_norm_one_gradient_absent(types, with_gx, with_gh):
    if not with_gh:
        x, delta = randn(6, 40, dtype=types[0]), None if types[1] is None else randn(6, 40, seed=3, dtype=types[1])
        norm, gx = norm_of(40, types[2]), randn(6, 40, seed=4, dtype=types[0])
        ins = [x.requires_grad_(), norm.weight] + ([] if delta is None else [delta.requires_grad_()])
        xs, _ = kernels.add_rmsnorm_train(x, delta, norm, out_dtype=types[3])
        got = torch.autograd.grad(xs, ins, gx)
        assert torch.equal(got[0], gx) and not got[1].any()
        return
    check_norm(6, 40, *types, with_gx=with_gx, with_gh=with_gh)


def test_norm_strides_and_shapes():
    norm = norm_of(48, F32)
    x, d = randn(4, 5, 48, dtype=F32), randn(4, 5, 48, seed=3)
    want = kernels.add_rmsnorm_train(x, d, norm, out_dtype=BF16)
    turned = kernels.add_rmsnorm_train(x.transpose(0, 1).contiguous().transpose(0, 1), d.repeat_interleave(2, 2)[..., ::2], norm,
                                       out_dtype=BF16)
    assert all(torch.equal(a, b) for a, b in zip(want, turned))
    flat = kernels.add_rmsnorm_train(x[0, 0], d[0, 0], norm, out_dtype=BF16)
    assert all(torch.equal(a, b[0, 0]) for a, b in zip(flat, want))
    none = kernels.add_rmsnorm_train(x[:0].requires_grad_(), d[:0], norm)
    dx, dw = torch.autograd.grad(none[1].sum() + none[0].sum(), (none[0], norm.weight), allow_unused=True)
    assert not dw.any()


def test_norm_offset_rows():
    """Rows that start on any element: the loads need no alignment beyond their elements'."""
    flat, norm = randn(1 + 40 * 96, dtype=BF16), norm_of(96, BF16)
    x = flat[1:].view(40, 96)
    a, b = kernels.add_rmsnorm_train(x, None, norm), kernels.add_rmsnorm_train(x.clone(), None, norm)
    assert torch.equal(a[1], b[1])


def test_norm_zero_and_infinite_rows():
    norm = norm_of(64, F32)
    x = randn(5, 64, dtype=F32)
    x[1], x[3, 4] = 0, float("inf")
    x.requires_grad_()
    _, h = kernels.add_rmsnorm_train(x, None, norm)
    ref = F.rms_norm(x, (64,), norm.weight, norm.eps)
    assert torch.equal(torch.isnan(h), torch.isnan(ref)) and not h[1].any()
    dx, = torch.autograd.grad(h[:3].sum(), x)
    assert torch.isfinite(dx[:3]).all()


def test_norm_recorded_gradient():
    norm, x, d = norm_of(24, F32), randn(5, 24, dtype=F32).requires_grad_(), randn(5, 24, seed=3, dtype=F32).requires_grad_()
    g = randn(5, 24, seed=4, dtype=F32)
    xs, h = kernels.add_rmsnorm_train(x, d, norm)
    dx, = torch.autograd.grad((h * g).sum() + xs.square().sum(), x, create_graph=True)
    got, = torch.autograd.grad(dx.square().sum(), norm.weight)
    xd, wd = (x + d).detach().double().requires_grad_(), norm.weight.detach().double().requires_grad_()
    hd = F.rms_norm(xd, (24,), wd, norm.eps)
    rx, = torch.autograd.grad((hd * g.double()).sum() + xd.square().sum(), xd, create_graph=True)
    ref, = torch.autograd.grad(rx.square().sum(), wd)
    assert float((got.double() - ref).norm() / ref.norm()) <= 1e-4


# ------------------------------------------------------------------------------------------------- together
def block(x, delta, t, norm, w13, w2, emb):
    """Norm, FFN, norm and loss: the tail of a training pass."""
    x, h = kernels.add_rmsnorm_train(x, delta, norm, out_dtype=BF16)
    delta = kernels.gated_ffn(h, w13, w2)
    _, h = kernels.add_rmsnorm_train(x, delta, norm, out_dtype=BF16)
    return kernels.linear_cross_entropy(h, emb, t)


def block_inputs(M=200, d=96, h=160, V=700):
    _, w13, w2, _ = ffn_inputs(1, d, h, d)
    return (randn(M, d, dtype=F32), randn(M, d, seed=3), targets(M, V, ignored=0.1), norm_of(d, F32), w13, w2,
            randn(V, d, std=0.2, seed=8))


def leaves(x, delta, t, norm, w13, w2, emb):
    return [v.requires_grad_() for v in (x, delta, norm.weight, w13, w2, emb)]


def test_a_run_of_them_together():
    ins = block_inputs()
    ls = leaves(*ins)
    loss = block(*ins)
    got = torch.autograd.grad(loss, ls)
    x, delta, nw, w13, w2, emb = (v.detach().double().requires_grad_() for v in ls)
    xs = x + delta
    h = F.rms_norm(xs, nw.shape, nw, 1e-5)
    a, b = (h @ w13.T).chunk(2, 1)
    xs = xs + (F.silu(a) * b) @ w2.T
    ref_loss = F.cross_entropy(F.rms_norm(xs, nw.shape, nw, 1e-5) @ emb.T, ins[2])
    ref = torch.autograd.grad(ref_loss, (x, delta, nw, w13, w2, emb))
    assert abs(loss.item() - ref_loss.item()) <= 2e-3 * ref_loss.item()
    for name, p, q in zip(("x", "delta", "norm", "w13", "w2", "emb"), got, ref):
        # a chain of eight bf16 roundings, each at most 2^-8 of its value
        assert float((p.double() - q).norm() / q.norm()) <= 8 * HALF, name


def test_captured_and_replayed_with_new_inputs():
    """Forward and gradient in one graph; replays see new inputs and match the eager calls bit for bit, with eager work of
    the same sizes in between."""
    ins = block_inputs()
    static = [v.clone() if torch.is_tensor(v) else v for v in ins]
    ls = leaves(*static)

    def step():
        loss = block(*static)
        return [loss.detach(), *torch.autograd.grad(loss, ls)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with capture(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            static[0].copy_(randn(*ins[0].shape, seed=50 + k, dtype=F32))
            static[4].copy_(randn(*ins[4].shape, std=0.1, seed=60 + k))
            static[2].copy_(targets(ins[2].numel(), 700, seed=70 + k, ignored=0.3))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_two_graphs_share_nothing():
    """Two captured calls replayed in turn: each keeps its own workspace and results."""
    made = []
    for seed in (0, 1):
        x, w, t = randn(130, 64, seed=seed), randn(900, 64, std=0.3, seed=seed + 5), targets(130, 900, seed=seed)
        want = run_loss(x, w, t)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run_loss(x, w, t)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with capture(graph):
            out = run_loss(x, w, t)
        made.append((graph, out, want, (x, w, t)))                     # a graph reads its inputs where they were
    for _ in range(3):
        for graph, *_ in made:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in made:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


# --------------------------------------------------------------------------------------------------- refusals
def bulk(rows, cols, std=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(rows, cols, dtype=BF16, device=DEV).normal_(0, std, generator=g)


def test_ffn_past_2_31_elements():
    """1,100,000 x 2,048 gradients of a and b: the last rows against the reference; of the others dy is 0, so that the
    weights' gradients are those of the last rows alone."""
    M, d, h, o, n = 1100000, 16, 1024, 16, 700
    note("ffn", M, d, h, o)
    x, (_, w13, w2, _) = bulk(M, d), ffn_inputs(1, d, h, o)
    g = torch.zeros(M, o, dtype=BF16, device=DEV)
    g[-n:] = randn(n, o, std=0.1, seed=3)
    y, dx, dw13, dw2 = run_ffn(x, w13, w2, g)
    ref = ffn_reference(x[-n:], w13, w2, g[-n:])
    assert not dx[:-n].any()
    for name, t, (r, tol) in zip(("y", "dx", "dw13", "dw2"), (y[-n:], dx[-n:], dw13, dw2), ref):
        close(t, r, tol, name)


def test_loss_past_2_31_elements():
    """2,200,000 x 1,000 states, of which the last few count, over a small vocabulary."""
    M, V, d, n = 2200000, 300, 1000, 500
    note("loss", M, V, d)
    x, w = bulk(M, d), randn(V, d, std=0.1, seed=2)
    t = torch.full((M,), -100, device=DEV)
    t[-n:] = targets(n, V)
    loss, dx, dw = run_loss(x, w, t, "sum")
    (l, lt), (rx, xt), (rw, wt) = loss_reference(x[-n:], w, t[-n:], -100, "sum")
    assert not dx[:-n].any()
    for name, got, r, tol in (("loss", loss, l, lt), ("dx", dx[-n:], rx, xt), ("dw", dw, rw, wt)):
        close(got, r, tol, name)


def test_norm_past_2_31_elements():
    M, C, n = 2200000, 1001, 300
    note("norm", M, C)
    norm = norm_of(C, F32)
    x, gh = bulk(M, C), torch.zeros(M, C, dtype=BF16, device=DEV)
    gh[-n:] = randn(n, C, seed=5)
    xs, h, (dx, dw) = run_norm(x, None, norm, BF16, None, gh)
    small = run_norm(x[-n:], None, norm, BF16, None, gh[-n:])
    assert torch.equal(h[-n:], small[1]) and torch.equal(dx[-n:], small[2][0]) and not dx[:-n].any()
    # the same terms in another order: n sums of fp32
    hat = small[1].double() / norm.weight.detach().double()
    close(dw, small[2][1].double(), 2 * (n + 64) * U32 * (gh[-n:].double() * hat).abs().sum(0) + TINY, "dw")


def test_lazily_negated_views():
    """Views whose sign is yet to be applied (a conjugate's imaginary part is one) count with it, gradients too."""
    x, w, t = randn(40, 24), randn(60, 24, std=0.3, seed=2), targets(40, 60)
    neg = torch._neg_view
    assert all(torch.equal(a, b) for a, b in zip(run_loss(neg(x), neg(w), t, "none", g=neg(randn(40, dtype=F32))),
                                                 run_loss(-x, -w, t, "none", g=-randn(40, dtype=F32))))
    ins = ffn_inputs(40, 24, 32, 16)
    assert all(torch.equal(a, b) for a, b in zip(run_ffn(*map(neg, ins)), run_ffn(*(-i for i in ins))))
    n = torch.nn.RMSNorm(24, eps=1e-5, device=DEV)
    z = torch.complex(randn(40, 24, dtype=F32), randn(40, 24, seed=3, dtype=F32)).conj().imag
    assert z.is_neg()
    a, b = kernels.add_rmsnorm_train(z, z, n), kernels.add_rmsnorm_train(z.clone().resolve_neg(), z.resolve_neg(), n)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_traces():
    x, w, t = randn(8, 16), randn(20, 16), targets(8, 20)
    _, w13, w2, _ = ffn_inputs(8, 16, 16, 16)
    n = torch.nn.RMSNorm(16, device=DEV)
    for f in (lambda x: kernels.linear_cross_entropy(x, w, t), lambda x: kernels.gated_ffn(x, w13, w2),
              lambda x: kernels.add_rmsnorm_train(x, None, n)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,), check_trace=False)
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.vmap(f)(torch.stack([x, x]))


def test_refusals():
    x, w, t = randn(4, 16), randn(30, 16), targets(4, 30)
    for bad in (lambda: kernels.linear_cross_entropy(x.float(), w, t), lambda: kernels.linear_cross_entropy(x, w.float(), t),
                lambda: kernels.linear_cross_entropy(x, w[:, :8], t), lambda: kernels.linear_cross_entropy(x, w, t.int()),
                lambda: kernels.linear_cross_entropy(x, w, t[:3]), lambda: kernels.linear_cross_entropy(x, w[:0], t),
                lambda: kernels.linear_cross_entropy(x, w, t, reduction="max"),
                lambda: kernels.linear_cross_entropy(x, w.cpu(), t), lambda: kernels.gated_ffn(x.float(), w, w),
                lambda: kernels.gated_ffn(x, w, randn(16, 16)), lambda: kernels.gated_ffn(x, w[:, :8], randn(16, 15)),
                lambda: kernels.gated_ffn(x, w.cpu(), randn(16, 15)),
                lambda: kernels.add_rmsnorm_train(x, x.float(), norm_of(16, F32)),
                lambda: kernels.add_rmsnorm_train(x, x[:2], norm_of(16, F32)),
                lambda: kernels.add_rmsnorm_train(x, None, norm_of(8, F32)),
                lambda: kernels.add_rmsnorm_train(x.half(), None, norm_of(16, F32)),
                lambda: kernels.add_rmsnorm_train(x, None, norm_of(16, F32), out_dtype=torch.float16),
                lambda: kernels.add_rmsnorm_train(x, None, torch.nn.RMSNorm(16, elementwise_affine=False))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------ Transformer.loss
def lm(dtype=F32, **kw):
    from smlm_hip.model import ModelConfig, Transformer
    torch.manual_seed(5)
    canon = kw.pop("canon", None)
    m = Transformer(ModelConfig(**dict(dict(vocab_size=517, d_model=128, n_layers=3, n_heads=2, ffn_hidden=200,
                                            max_seq_len=64), **kw)), ngram_canon=canon)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 2:
                p.mul_(4.0)                   # logits that matter
    return m.to(DEV).to(dtype)


def batch(V=517, seed=0, ignored=True):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, V, (3, 33), generator=g)
    t = torch.roll(idx, -1, 1)
    if ignored:
        t[:, -1], t[1, 20:] = -100, -100
    return idx.to(DEV), t.to(DEV)


def named_grads(m, loss):
    names, ps = zip(*[(n, p) for n, p in m.named_parameters() if p.requires_grad])
    return dict(zip(names, torch.autograd.grad(loss, ps, allow_unused=True)))


def spied(monkeypatch):
    """How often the three operators ran."""
    calls = {"linear_cross_entropy": 0, "gated_ffn": 0, "add_rmsnorm_train": 0}
    for name in calls:
        fn = getattr(kernels, name)

        def wrapped(*a, _fn=fn, _name=name, **k):
            calls[_name] += 1
            return _fn(*a, **k)

        monkeypatch.setattr(kernels, name, wrapped)
    return calls


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_model_loss_against_64_bits(dtype, monkeypatch):
    """Loss and gradients as near to a 64-bit model's as the module path's, whose bf16 roundings are more."""
    m = lm(dtype)
    idx, t = batch()
    ref = lm(F32).cpu().double()
    ref.load_state_dict({k: v.cpu().double() for k, v in m.state_dict().items()})
    for a, b in zip(ref.layers, m.layers):
        a.attn.rope.cos, a.attn.rope.sin = b.attn.rope.cos.cpu().double(), b.attn.rope.sin.cpu().double()
    import smlm_hip.model as model
    monkeypatch.setattr(model, "_attention", lambda q, k, v, mask: F.scaled_dot_product_attention(q, k, v, attn_mask=mask))
    logits = ref(idx.cpu())
    ref_loss = F.cross_entropy(logits.view(-1, 517), t.view(-1).cpu())
    want = named_grads(ref, ref_loss)
    calls = spied(monkeypatch)
    with torch.autocast("cuda", dtype=BF16, enabled=dtype == F32):
        loss = m.loss(idx, t)
        assert calls == {"linear_cross_entropy": 1, "gated_ffn": 3, "add_rmsnorm_train": 7}
        _, plain = m(idx, t)
    assert loss.dtype == F32 and abs(loss.item() - ref_loss.item()) <= 1.5 * abs(plain.item() - ref_loss.item()) + 4 * HALF
    got, base = named_grads(m, loss), named_grads(m, plain)
    for n, r in want.items():
        err = lambda g: float((g.cpu().double() - r).norm() / r.norm())  # noqa: E731
        assert got[n].dtype == dtype and err(got[n]) <= 1.25 * err(base[n]) + 2 * HALF, (n, err(got[n]), err(base[n]))


@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_model_loss_scores_text_without_gradients(reduction):
    m = lm(BF16).eval()
    idx, t = batch()
    with torch.no_grad():
        got, logits = m.loss(idx, t, reduction=reduction), m(idx)
    ref = F.cross_entropy(logits.double().view(-1, 517), t.view(-1), reduction="none").view(t.shape)
    if reduction == "sum":
        assert abs(got.item() - ref.sum().item()) <= 0.02 * ref.sum().item()
        return
    assert got.shape == t.shape and not got.requires_grad and not got[t == -100].any()
    # the module path rounds its logits (of size s) to bf16 and both round the hidden state
    s = logits.double().abs().amax(-1)
    assert ((got.double() - ref).abs() <= 8 * HALF * (1 + s)).all()


def test_model_loss_with_memory_and_engram_layers(monkeypatch):
    """Memory layers get the stream's type, Engram layers the summed stream; the table's row-sparse gradients arrive."""
    m = lm(F32, d_model=64, n_heads=2, ffn_hidden=96, n_layers=4, mem_layers=[1, 2], mem_n_keys=16, mem_heads=2, mem_knn=4,
           mem_k_dim=32, mem_share_values=True, mem_round_layers=[2], eng_layers=[0, 3], eng_heads=2, eng_head_dim=8,
           eng_rows=101, canon=torch.arange(517)).train()
    idx, t = batch()
    calls = spied(monkeypatch)
    state = {k: v.clone() for k, v in m.state_dict().items()}
    with torch.autocast("cuda", dtype=BF16):
        loss = m.loss(idx, t)
        assert calls == {"linear_cross_entropy": 1, "gated_ffn": 2, "add_rmsnorm_train": 10}
        got = named_grads(m, loss)
        m.load_state_dict(state)
        _, plain = m(idx, t)
        want = named_grads(m, plain)
    assert abs(loss.item() - plain.item()) <= 0.03 * plain.item()
    for n, g in want.items():
        assert (g is None) == (got[n] is None), n


@pytest.mark.parametrize("watch", ["norm", "ffn", "block", "head", "subclass", "final", "embedding", "model"])
def test_model_loss_keeps_watched_modules(watch, monkeypatch):
    m = lm(BF16)
    idx, t = batch()
    seen = []
    target = {"norm": m.layers[1].ffn_norm, "ffn": m.layers[1].ffn.w2, "block": m.layers[1], "head": m.lm_head,
              "final": m.norm, "embedding": m.tok_emb, "model": m}.get(watch)
    if target is not None:
        target.register_forward_hook(lambda *a: seen.append(1))
    else:
        class Other(torch.nn.Parameter):
            pass
        m.layers[1].ffn.w13.weight = Other(m.layers[1].ffn.w13.weight.detach())
    calls = spied(monkeypatch)
    loss = m.loss(idx, t)
    _, plain = m(idx, t)
    assert abs(loss.item() - plain.item()) <= 0.03 * plain.item()
    if target is not None:
        assert len(seen) == 2                              # once in each
    expected = {"norm": (1, 3, 6), "ffn": (1, 2, 7), "block": (1, 2, 5), "head": (0, 0, 0), "subclass": (1, 2, 7),
                "final": (0, 0, 0), "embedding": (0, 0, 0), "model": (0, 0, 0)}[watch]
    assert tuple(calls.values()) == expected, calls


def test_model_loss_follows_function_transforms():
    """Under a function mode the modules run, and it sees their ops."""
    from torch.overrides import TorchFunctionMode

    class Count(TorchFunctionMode):
        n = 0

        def __torch_function__(self, func, types, args=(), kwargs=None):
            Count.n += func is F.cross_entropy
            return func(*args, **(kwargs or {}))

    m = lm(BF16)
    idx, t = batch()
    with Count(), torch.no_grad():
        m.loss(idx, t)
    assert Count.n == 1


def test_model_trains_on_the_loss():
    """Ten steps on one batch run and change every parameter."""
    m = lm(F32).train()
    idx, t = batch()
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3)
    for _ in range(10):
        with torch.autocast("cuda", dtype=BF16):
            loss = m.loss(idx, t)
        loss.backward()
        opt.step()
        opt.zero_grad()
    assert torch.isfinite(loss) and all(not torch.equal(p, before[n]) for n, p in m.named_parameters())
