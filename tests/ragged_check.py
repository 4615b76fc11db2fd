"""The operators of serving sequences of different lengths, written plainly in 64 bits: what tests/test_gpu_ragged.py and
tests/test_ragged_host.py compare with."""
import math

import torch

bf16 = torch.bfloat16
HALF = 2.0 ** -8           # half a step of bf16, relative


def rotate(x, cos, sin, interleaved):
    """x (N, heads, dim) double, cos, sin (N, half) double: the first 2 * half dims of each head rotated."""
    out, half = x.clone(), cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[:, i:i + 1], sin[:, i:i + 1]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()


def values(codes, scale):
    """What 4-bit rows stand for: (..., dim / 2) uint8 and (..., 2) step, lowest."""
    return scale[..., 1:].double() + scale[..., :1].double() * unpack(codes)


def quantized(x):
    """Random 4-bit rows for x (..., dim): codes (..., dim / 2) uint8 and scale (..., 2) bf16."""
    x = x.double()
    lo = x.amin(-1, keepdim=True).to(bf16)
    step = ((x.amax(-1, keepdim=True) - lo.double()) / 15).to(bf16)
    c = ((x - lo.double()) / step.double()).round().clamp(0, 15)
    c = torch.where(step > 0, c, torch.zeros_like(c)).to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4, torch.cat([step, lo], -1)


def attention(q, k, v, seen, scale):
    """q (T, H, D), k, v (S, Hk, D) double, seen (T, S) bool: y (T, H, D), and the weighted sum of |v| that bounds what
    rounding the weights costs.  Rows that see nothing are zeros; what is masked does not count, whatever it holds."""
    share = q.shape[1] // k.shape[1]
    y, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(q.shape[1]):
        kh, vh = k[:, h // share], v[:, h // share]
        for t in range(q.shape[0]):
            at = seen[t].nonzero().flatten()
            if len(at):
                w = torch.softmax(kh[at] @ q[t, h] * scale, 0)
                y[t, h], bound[t, h] = w @ vh[at], w @ vh[at].abs()
    return y, bound


def causal(T, S):
    return torch.ones(T, S, dtype=torch.bool).tril(S - T)


def sample(x, u, temperature, top_k, top_p, min_p):
    """The token of one row x (V,) at u.  Masses are weights in whole multiples of 2^-45 of the largest, as sample_tokens defines
    them: a token of weight below 2^-46 is not drawn at u = 0 either, where its weight in 64 bits, e^-700 still above 0, is."""
    x = x.double().clone()
    x[~(x > -3.389e38)] = -3.3895313892515355e38
    V = len(x)
    order = sorted(range(V), key=lambda i: (-float(x[i]), i)) if V < 300 else torch.sort(x, descending=True, stable=True).indices.tolist()
    if not temperature > 0:
        return order[0]
    order = torch.tensor(order[:top_k] if 0 < top_k < V else order)
    w = ((x[order] - x[order[0]]) / temperature).exp()
    n, mass = len(w), (w * 2.0 ** 45).round()
    if top_p < 1:
        before = torch.cat([torch.zeros(1, dtype=torch.float64), mass.cumsum(0)[:-1]])
        n = max(1, int((before < top_p * mass.sum()).sum()))
    n = max(1, min(n, int((w >= min_p).sum())))
    kept, place = order[:n].sort()
    mass = mass[:n][place].cumsum(0)
    return int(kept[min(int((mass <= u * float(mass[-1])).sum()), n - 1)])


def f32(v):
    """A Python number as the fp32 that a call takes it for."""
    return float(torch.tensor(v, dtype=torch.float32))


def bound_of(y, weighted):
    """The output's rounding, the probabilities' twice (in the sum of values and in their own), and fp32 sums."""
    return HALF * y.abs() + 2.1 * HALF * weighted + 1e-30


__all__ = ["math", "rotate", "values", "unpack", "quantized", "attention", "causal", "sample", "bound_of", "f32", "HALF"]
