"""The dense operators of a training step, as cases that can be timed and checked: the language model's loss over its
vocabulary without stored logits, the gated feed-forward block, and the residual add with RMSNorm, each with its
gradients.  Sizes are the package's configurations (d_model 384, ffn 1024, vocabularies of 32,000 and 50,304) and odd ones
around them."""
import math
import os
import sys

import torch
import torch.nn.functional as F

own = False

DEV = torch.device("cuda")
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100
EPS = 1e-5


def _kernels():
    path = os.path.join(os.getcwd(), "sparse-memory-lm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from smlm_hip import kernels
    return kernels


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the loss of one short sequence, as when fine-tuning on single examples: launches and the weight's gradient
        {"name": "loss_small", "kind": "loss", "tokens": 64, "vocab": 32000, "width": 384, "ignored": 0.0,
         "reduction": "mean", "grad": True},
        # the loss of a training micro-batch (4 x 1024 tokens, the default vocabulary)
        {"name": "loss_train", "kind": "loss", "tokens": 4096, "vocab": 50304, "width": 384, "ignored": 0.0,
         "reduction": "mean", "grad": True},
        # four such micro-batches in one step
        {"name": "loss_large", "kind": "loss", "tokens": 16384, "vocab": 50304, "width": 384, "ignored": 0.0,
         "reduction": "mean", "grad": True},
        # padded sequences of odd lengths (3 x 677), an odd vocabulary and width, summed over accumulation steps
        {"name": "loss_ragged", "kind": "loss", "tokens": 2031, "vocab": 32003, "width": 201, "ignored": 0.3,
         "reduction": "sum", "grad": True},
        # held-out text scored token by token: no gradient
        {"name": "loss_score", "kind": "loss", "tokens": 8192, "vocab": 32000, "width": 384, "ignored": 0.05,
         "reduction": "none", "grad": False},
        # the feed-forward block of one short sequence
        {"name": "ffn_small", "kind": "ffn", "tokens": 48, "width": 384, "hidden": 1024},
        # of a training micro-batch
        {"name": "ffn_train", "kind": "ffn", "tokens": 4096, "width": 384, "hidden": 1024},
        # of eight
        {"name": "ffn_large", "kind": "ffn", "tokens": 32768, "width": 384, "hidden": 1024},
        # odd everywhere: 7 x 2011 tokens, a width and a hidden size off every tile
        {"name": "ffn_odd", "kind": "ffn", "tokens": 14077, "width": 392, "hidden": 1001},
        # the norm of one short sequence of a bf16 model
        {"name": "norm_small", "kind": "norm", "tokens": 64, "width": 384, "x": "bf16", "delta": "bf16", "weight": "bf16",
         "out": "bf16"},
        # the norm of a step of 32 sequences under bf16 autocast: fp32 residual stream, bf16 sublayers
        {"name": "norm_train", "kind": "norm", "tokens": 32768, "width": 384, "x": "fp32", "delta": "bf16",
         "weight": "fp32", "out": "bf16"},
        # a wide odd stream, the first norm of a model (nothing to add)
        {"name": "norm_odd", "kind": "norm", "tokens": 9001, "width": 1001, "x": "bf16", "delta": None, "weight": "fp32",
         "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "ffn", "norm"])
    if kind == "loss":
        width = rng.choice([8 * rng.randint(4, 64), 8 * rng.randint(4, 64), rng.randint(33, 511)])
        vocab = rng.choice([_log(rng, 500, 65536), 8 * _log(rng, 64, 8192)])
        most = 16384 * 50304 * 384 // (vocab * width)
        return {"kind": kind, "tokens": min(_log(rng, 1, 16384), most), "vocab": vocab, "width": width,
                "ignored": rng.choice([0.0, 0.0, 0.1, 0.6]), "reduction": rng.choice(["mean", "mean", "sum", "none"]),
                "grad": rng.random() < 0.75}
    if kind == "ffn":
        width = rng.choice([8 * rng.randint(4, 64), 8 * rng.randint(4, 64), rng.randint(33, 511)])
        hidden = rng.choice([64 * rng.randint(1, 32), 8 * rng.randint(8, 256), rng.randint(65, 2047)])
        most = 32768 * 384 * 1024 // (width * hidden)
        return {"kind": kind, "tokens": min(_log(rng, 1, 32768), most), "width": width, "hidden": hidden}
    width = rng.choice([8 * rng.randint(4, 256), 8 * rng.randint(4, 64), rng.randint(1, 2047)])
    x = rng.choice(["fp32", "bf16"])
    return {"kind": kind, "tokens": min(_log(rng, 1, 131072), 65536 * 384 // width), "width": width, "x": x,
            "delta": rng.choice([None, "bf16", x]), "weight": rng.choice(["fp32", "bf16"]),
            "out": rng.choice(["bf16", x])}


# --------------------------------------------------------------------------------------------------- the states
def _randn(*shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, device=DEV).mul_(std).to(dtype)


def prepare(c, seed):
    torch.manual_seed(seed)
    M, d, bf16 = c["tokens"], c["width"], torch.bfloat16
    if c["kind"] == "loss":
        V = c["vocab"]
        w = _randn(V, d, std=0.06, dtype=bf16)
        # word-like frequencies, and hidden states that lean towards their target as a trained model's do
        t = torch.rand(M, device=DEV).mul_(math.log(V)).exp_().long().sub_(1).clamp_(0, V - 1)
        t = torch.randperm(V, device=DEV)[t]
        x = torch.randn(M, d, device=DEV).add_(w[t].float(), alpha=5.0).to(bf16)
        t = torch.where(torch.rand(M, device=DEV) < c["ignored"], torch.full_like(t, IGNORE), t)
        s = {"c": c, "x": x.requires_grad_(c["grad"]), "w": w.requires_grad_(c["grad"]), "t": t}
        if c["reduction"] == "none" and c["grad"]:
            s["g"] = torch.rand(M, device=DEV).add_(0.5)       # weights of the single tokens
        return s
    if c["kind"] == "ffn":
        h = c["hidden"]
        return {"c": c, "x": _randn(M, d, dtype=bf16).requires_grad_(),
                "w13": _randn(2 * h, d, std=1.2 / math.sqrt(d), dtype=bf16).requires_grad_(),
                "w2": _randn(d, h, std=1.0 / math.sqrt(h), dtype=bf16).requires_grad_(),
                "g": _randn(M, d, std=1e-3, dtype=bf16)}
    x, out = DTYPES[c["x"]], DTYPES[c["out"]]
    norm = torch.nn.RMSNorm(d, eps=EPS, device=DEV, dtype=DTYPES[c["weight"]])
    with torch.no_grad():
        norm.weight.uniform_(0.5, 1.5)
    s = {"c": c, "norm": norm, "x": _randn(M, d, std=2.0, dtype=x).requires_grad_(), "delta": None,
         "gx": _randn(M, d, std=1e-3, dtype=x), "gh": _randn(M, d, std=1e-3, dtype=out)}
    if c["delta"] is not None:
        s["delta"] = _randn(M, d, dtype=DTYPES[c["delta"]]).requires_grad_()
    return s


# ----------------------------------------------------------------------------------------------------- the pass
def run(s):
    kind = s["c"]["kind"]
    if kind == "loss":
        return _loss_own(s) if own else _loss_plain(s)
    if kind == "ffn":
        return _ffn_own(s) if own else _ffn_plain(s)
    return _norm_own(s) if own else _norm_plain(s)


def _loss_own(s):
    c = s["c"]
    loss = _kernels().linear_cross_entropy(s["x"], s["w"], s["t"], ignore_index=IGNORE, reduction=c["reduction"])
    if not c["grad"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s.get("g"))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


@torch.no_grad()
def _loss_plain(s):
    c, x, w, t = s["c"], s["x"].float(), s["w"].float(), s["t"]
    valid = t != IGNORE
    at = torch.where(valid, t, torch.zeros_like(t)).unsqueeze(1)
    logits = x @ w.T
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at).squeeze(1)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    each = torch.where(valid, (total.log() + top).squeeze(1) - picked, torch.zeros_like(picked))
    coef = valid.float()
    if c["reduction"] == "mean":
        loss, coef = each.sum() / valid.sum(), coef / valid.sum()
    elif c["reduction"] == "sum":
        loss = each.sum()
    else:
        loss = each
    if not c["grad"]:
        return {"loss": loss}
    if "g" in s:
        coef = coef * s["g"]
    coef = coef.unsqueeze(1)
    g = p.mul_(coef / total).scatter_add_(1, at, -coef)
    return {"loss": loss, "dx": (g @ w).to(s["x"].dtype), "dw": (g.T @ x).to(s["w"].dtype)}


def _ffn_own(s):
    y = _kernels().gated_ffn(s["x"], s["w13"], s["w2"])
    dx, dw13, dw2 = torch.autograd.grad(y, (s["x"], s["w13"], s["w2"]), s["g"])
    return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}


@torch.no_grad()
def _ffn_plain(s):
    x, w13, w2, g = s["x"].float(), s["w13"].float(), s["w2"].float(), s["g"].float()
    a, b = (x @ w13.T).chunk(2, 1)
    sig = 1.0 / (1.0 + (-a).exp())
    act = a * sig
    h = act * b
    dh = g @ w2
    dab = torch.cat([dh * b * (sig + act * (1.0 - sig)), dh * act], 1)
    bf16 = s["x"].dtype
    return {"y": (h @ w2.T).to(bf16), "dx": (dab @ w13).to(bf16), "dw13": (dab.T @ x).to(bf16),
            "dw2": (g.T @ h).to(bf16)}


def _norm_own(s):
    out = DTYPES[s["c"]["out"]]
    xs, h = _kernels().add_rmsnorm_train(s["x"], s["delta"], s["norm"], out_dtype=out)
    inputs = [s["x"], s["norm"].weight] + ([] if s["delta"] is None else [s["delta"]])
    got = torch.autograd.grad((xs, h), inputs, (s["gx"], s["gh"]))
    return {"xs": xs.detach(), "h": h.detach(), **dict(zip(("dx", "dw", "ddelta"), got))}


@torch.no_grad()
def _norm_plain(s):
    x, delta, w, gh = s["x"], s["delta"], s["norm"].weight.float(), s["gh"].float()
    xs = x if delta is None else (x.float() + delta.float()).to(x.dtype)     # the stream as it is stored
    xf = xs.float()
    r = (xf.square().mean(1, keepdim=True) + EPS).rsqrt()
    hat = xf * r
    gw = gh * w
    dx = (gw - hat * (gw * hat).mean(1, keepdim=True)) * r + s["gx"].float()
    got = {"xs": xs.detach(), "h": (hat * w).to(DTYPES[s["c"]["out"]]), "dx": dx.to(x.dtype),
           "dw": (gh * hat).sum(0).to(s["norm"].weight.dtype)}
    if delta is not None:
        got["ddelta"] = dx.to(delta.dtype)
    return got


# ----------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    double = lambda t: None if t is None else t.detach().double().requires_grad_()  # noqa: E731
    if c["kind"] == "loss":
        x, w = double(s["x"]), double(s["w"])
        loss = F.cross_entropy(x @ w.T, s["t"], ignore_index=IGNORE, reduction=c["reduction"])
        if not c["grad"]:
            return {"loss": loss.detach()}
        dx, dw = torch.autograd.grad(loss, (x, w), None if "g" not in s else s["g"].double())
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    if c["kind"] == "ffn":
        x, w13, w2 = double(s["x"]), double(s["w13"]), double(s["w2"])
        a, b = (x @ w13.T).chunk(2, 1)
        y = (F.silu(a) * b) @ w2.T
        dx, dw13, dw2 = torch.autograd.grad(y, (x, w13, w2), s["g"].double())
        return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}
    x, delta, w = double(s["x"]), double(s["delta"]), double(s["norm"].weight)
    xs = x if delta is None else x + delta
    if c["x"] != "fp32":
        xs = xs + (xs.to(s["x"].dtype).double() - xs).detach()               # the stream as it is stored
    h = F.rms_norm(xs, (c["width"],), w, EPS)
    inputs = [x, w] + ([] if delta is None else [delta])
    got = torch.autograd.grad((xs, h), inputs, (s["gx"].double(), s["gh"].double()))
    return {"xs": xs.detach(), "h": h.detach(), **dict(zip(("dx", "dw", "ddelta"), got))}


# ------------------------------------------------------------------------------------------------------- the work
def work(c):
    M, d = c["tokens"], c["width"]
    if c["kind"] == "loss":
        V, losses = c["vocab"], c["tokens"] if c["reduction"] == "none" else 1
        read, written, products = 2 * (M + V) * d + 8 * M, 4 * losses, 1
        if c["grad"]:
            written += 2 * (M + V) * d
            products = 3
        return {"bytes": read + written, "flops": 2 * products * M * V * d}
    if c["kind"] == "ffn":
        h = c["hidden"]
        return {"bytes": 2 * (2 * M * d + 3 * h * d) + 2 * (2 * M * d + 3 * h * d), "flops": 2 * 9 * M * d * h}
    size = {None: 0, "fp32": 4, "bf16": 2}
    x, delta, out, weight = (size[c[k]] for k in ("x", "delta", "out", "weight"))
    # forward: x, delta in, h and (with a delta) the stream out; gradient: its two gradients and the stream in, dx, ddelta out
    forward = M * d * (x + delta + out + (x if delta else 0))
    return {"bytes": forward + M * d * (out + x + x + x + delta) + 2 * weight * d, "flops": 20 * M * d}
