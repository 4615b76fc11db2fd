"""The operators of serving sequences of different lengths, as cases that can be timed and checked: keys and values appended
to a paged cache with the position rotation on the way (and read back from it), causal attention over packed prompts with
grouped heads, single-token attention over the paged cache in bf16 or 4 bits, and sampling from given random numbers.  Sizes
are the package's configurations (6 heads of 64, vocabularies of 32,000 and 50,304), grouped heads of 64 and 128, and odd
lengths around them."""
import math
import os
import random
import sys

import torch

own = False

DEV = torch.device("cuda")
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
THETA = 10000.0


def _kernels():
    path = os.path.join(os.getcwd(), "sparse-memory-lm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from smlm_hip import kernels
    return kernels


# ---------------------------------------------------------------------------------------------------- the cases
# seqs sequences with `longest` tokens at most, the lengths spread below it by `spread` (0: all as long as the longest)
def listed():
    return [
        # one decode step of a small batch of the default model: latency
        {"name": "append_step", "kind": "append", "kv": "bf16", "seqs": 16, "new": 1, "longest": 700, "spread": 0.8, "heads": 6,
         "kv_heads": 6, "dim": 64, "rot": 64, "interleaved": False, "page": 64},
        # the prompts of a batch of the default model in one pass
        {"name": "append_prompts", "kind": "append", "kv": "bf16", "seqs": 16, "new": 0, "longest": 1024, "spread": 0.6,
         "heads": 6, "kv_heads": 6, "dim": 64, "rot": 64, "interleaved": False, "page": 64},
        # a later piece of long prompts, grouped heads, over a 4-bit cache: appended, then all of the keys and values read back
        # for the prompt attention
        {"name": "append_chunk_q4", "kind": "append", "kv": "q4", "seqs": 4, "new": 509, "longest": 6000, "spread": 0.5,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16},
        # a few short prompts of the default model: latency
        {"name": "prompt_short", "kind": "prompt", "seqs": 3, "longest": 61, "spread": 0.5, "cached": 0, "heads": 6,
         "kv_heads": 6, "dim": 64},
        # a batch of prompts up to the default model's longest
        {"name": "prompt_batch", "kind": "prompt", "seqs": 32, "longest": 1024, "spread": 0.95, "cached": 0, "heads": 6,
         "kv_heads": 6, "dim": 64},
        # long documents on grouped heads of 128, one of them behind a cached beginning
        {"name": "prompt_long", "kind": "prompt", "seqs": 2, "longest": 6001, "spread": 0.3, "cached": 1500, "heads": 32,
         "kv_heads": 8, "dim": 128},
        # one sequence of the default model: latency
        {"name": "decode_one", "kind": "decode", "kv": "bf16", "seqs": 1, "longest": 700, "spread": 0.0, "heads": 6,
         "kv_heads": 6, "dim": 64, "page": 64},
        # a batch of them, lengths from a few tokens to the longest
        {"name": "decode_batch", "kind": "decode", "kv": "bf16", "seqs": 256, "longest": 1024, "spread": 0.99, "heads": 6,
         "kv_heads": 6, "dim": 64, "page": 64},
        # a batch of longer ones on grouped heads over a 4-bit cache of small pages
        {"name": "decode_q4_batch", "kind": "decode", "kv": "q4", "seqs": 48, "longest": 8191, "spread": 0.9, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16},
        # two very long ones: the walk is split
        {"name": "decode_q4_long", "kind": "decode", "kv": "q4", "seqs": 2, "longest": 131072, "spread": 0.01, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64},
        # the next token of one sequence, the usual settings
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 50304, "type": "bf16", "each": False, "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # a full batch, every sequence with settings of its own
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 50304, "type": "bf16", "each": True, "temperature": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.02},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(6, 6, 64), (6, 6, 64), (12, 12, 32), (3, 3, 128), (8, 1, 64), (9, 3, 64), (32, 8, 128), (16, 2, 128), (20, 4, 32)]


def draw(rng):
    kind = rng.choice(["append", "prompt", "decode", "sample"])
    if kind == "sample":
        vocab = rng.choice([32000, 50304, _log(rng, 100, 131072)])
        return {"kind": kind, "rows": min(_log(rng, 1, 512), 256 * 50304 // vocab), "vocab": vocab,
                "type": rng.choice(["bf16", "fp32"]), "each": rng.random() < 0.5,
                "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.6]), "top_k": rng.choice([0, 0, 1, 20, 50, _log(rng, 1, vocab)]),
                "top_p": rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.999]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1, 0.5])}
    heads, kv_heads, dim = rng.choice(HEADS)
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "spread": round(rng.uniform(0.0, 0.99), 3)}
    if kind == "prompt":
        seqs = _log(rng, 1, 128)
        longest = min(_log(rng, 2, 8192), int(14000 * math.sqrt(32 / heads)) // seqs)
        return dict(c, seqs=seqs, longest=longest, cached=rng.choice([0, 0, _log(rng, 1, longest)]) if seqs * longest < 4000 else 0)
    c.update(kv=rng.choice(["bf16", "q4"]), page=rng.choice([16, 32, 64, 128, 256]))
    row = kv_heads * dim
    if kind == "decode":
        seqs = _log(rng, 1, 512)
        return dict(c, seqs=seqs, longest=max(1, min(_log(rng, 1, 131072), 48 * 8191 * 1024 // (seqs * row))))
    seqs = _log(rng, 1, 256)
    longest = max(4, min(_log(rng, 4, 8192), 16 * 1024 * 1024 // (seqs * (heads + 2 * kv_heads) * dim)))
    return dict(c, seqs=seqs, longest=longest, new=rng.choice([0, 1, 1, rng.randint(1, longest)]),
                rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3)


# --------------------------------------------------------------------------------------------------- the states
def _lengths(c):
    """The sequences' lengths: the first is the longest, the others spread below it."""
    rng, n = random.Random(17), c["longest"]
    return [n] + [max(1, n - int(rng.random() * c["spread"] * n)) for _ in range(c["seqs"] - 1)]


def _randn(*shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).mul_(std).to(dtype)


def _ints(values, dtype):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _table(lengths, page):
    """A block table over pages handed out in no order, and how many pages there are."""
    need = [-(-n // page) for n in lengths]
    total, widest = sum(need) + 3, max(need)
    ids, table, at = torch.randperm(total), torch.zeros(len(lengths), widest, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table.to(DEV), total


def _quantized(x):
    """Rows x (..., dim) fp32 or wider as 4-bit codes (..., dim), and each row's step and lowest value in bf16."""
    bf16 = torch.bfloat16
    lo = x.amin(-1, keepdim=True).to(bf16)
    step = ((x.amax(-1, keepdim=True) - lo.to(x.dtype)) / 15.0).to(bf16)
    code = ((x - lo.to(x.dtype)) / step.to(x.dtype)).round().clamp(0, 15)
    return torch.where(step > 0, code, torch.zeros_like(code)).to(torch.uint8), torch.cat([step, lo], -1)


def _packed(code):
    """Two codes a byte: dim 2 i in the low half of byte i."""
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(packed, scale, dtype=torch.float32):
    """The values that 4-bit rows stand for."""
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).to(dtype)
    return scale[..., 1:].to(dtype) + scale[..., :1].to(dtype) * code


def _pages(c, total):
    """Pages in use by other and earlier tokens: (k, v), or (k, v, k_scale, v_scale) of 4 bits."""
    shape = (total, c["kv_heads"], c["page"], c["dim"])
    # keys have a few channels that stand out, as a trained model's do
    k, v = _randn(*shape), _randn(*shape)
    k[..., ::29] *= 4
    if c["kv"] == "bf16":
        return [k, v]
    (ck, sk), (cv, sv) = _quantized(k.float()), _quantized(v.float())
    return [_packed(ck), _packed(cv), sk, sv]


def prepare(c, seed):
    torch.manual_seed(seed)
    H, Hk, D = (c.get(key) for key in ("heads", "kv_heads", "dim"))
    s = {"c": c}
    if c["kind"] == "sample":
        B, V = c["rows"], c["vocab"]
        # scores that decay with a token's rank, as a language model's do, over a permuted vocabulary
        decay = torch.arange(1, V + 1, device=DEV).float().log_().mul_(-1.1)
        logits = torch.randn(B, V, device=DEV).add_(decay[torch.randperm(V, device=DEV)]).add_(9.0)
        s.update(logits=logits.to(DTYPES[c["type"]]), u=torch.rand(B, device=DEV))
        for key, dtype, spread in (("temperature", torch.float32, 0.5), ("top_p", torch.float32, 0.2), ("min_p", torch.float32, 1.0)):
            s[key] = torch.rand(B, device=DEV).mul_(-spread).add_(1).mul_(c[key]).to(dtype) if c["each"] else c[key]
        s["top_k"] = torch.randint(0, max(2, 2 * c["top_k"]), (B,), dtype=torch.int32, device=DEV) if c["each"] else c["top_k"]
        return s
    lengths = _lengths(c)
    if c["kind"] == "prompt":
        # queries over the last tokens of each sequence; a cached beginning has keys and values only (of every second one)
        cached = [c["cached"] if i % 2 == 0 else 0 for i in range(len(lengths))]
        cu_q, cu_k = [0], [0]
        for n, m in zip(lengths, cached):
            cu_q.append(cu_q[-1] + n)
            cu_k.append(cu_k[-1] + n + m)
        N, S = cu_q[-1], cu_k[-1]
        if any(cached):
            s.update(k=_randn(S, Hk, D), v=_randn(S, Hk, D), cu_k=_ints(cu_k, torch.int32))
        else:                                       # the values as they lie in the projection's rows
            rows = _randn(S, (H + 2 * Hk) * D)
            s.update(k=_randn(S, Hk, D), v=rows[:, (H + Hk) * D:].view(S, Hk, D), cu_k=None)
        return dict(s, q=_randn(N, H, D), cu_q=_ints(cu_q, torch.int32))
    page = c["page"]
    table, total = _table(lengths, page)
    s["pages"] = _pages(c, total)
    if c["kind"] == "decode":
        return dict(s, q=_randn(c["seqs"], H, D), table=table, lengths=_ints(lengths, torch.int32))
    new = [n if c["new"] == 0 else min(c["new"], n) for n in lengths]
    def at(seq, n):                                 # positions, and where these lie in the pages
        rows, pos = _ints(seq, torch.int64), _ints(n, torch.int64)
        return pos, table[rows, pos // page].long() * page + pos % page
    tokens = [(b, p) for b, n in enumerate(lengths) for p in range(n - new[b], n)]
    s["positions"], s["slots"] = at(*zip(*tokens))
    if c["kv"] == "q4":
        s["all"] = at(*zip(*((b, p) for b, n in enumerate(lengths) for p in range(n))))[1]
    inv = THETA ** (-torch.arange(0, c["rot"], 2, device=DEV).double() / c["rot"])
    angle = torch.outer(torch.arange(c["longest"], device=DEV).double(), inv)
    return dict(s, cos=angle.cos().float(), sin=angle.sin().float(), qkv=_randn(len(tokens), (H + 2 * Hk) * D))


# ----------------------------------------------------------------------------------------------------- the pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    c, kernels = s["c"], _kernels()
    if c["kind"] == "append":
        q, _ = kernels.paged_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["pages"], c["heads"],
                                    interleaved=c["interleaved"])
        if c["kv"] == "bf16":
            return {"q": q, "k_pages": s["pages"][0], "v_pages": s["pages"][1]}
        k, v = kernels.paged_gather(s["pages"], s["all"])
        return {"q": q, "k": k, "v": v}
    if c["kind"] == "prompt":
        return {"y": kernels.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])}
    if c["kind"] == "decode":
        return {"y": kernels.paged_attention(s["q"], s["pages"], s["table"], s["lengths"])}
    return {"token": kernels.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])}


@torch.no_grad()
def _run_plain(s):
    kind = s["c"]["kind"]
    if kind == "append":
        return _append_plain(s)
    if kind == "prompt":
        return _prompt_plain(s)
    if kind == "decode":
        return _decode_plain(s)
    return _sample_plain(s)


def _rotated(x, cos, sin, interleaved):
    """x (N, heads, dim) with the first 2 * cos.shape[1] dims of each head rotated, in x's type."""
    half = cos.shape[1]
    cos, sin, rest = cos.unsqueeze(1), sin.unsqueeze(1), x[..., 2 * half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _append_plain(s):
    c = s["c"]
    H, Hk, page, bf16 = c["heads"], c["kv_heads"], c["page"], torch.bfloat16
    q, k, v = s["qkv"].float().view(-1, H + 2 * Hk, c["dim"]).split([H, Hk, Hk], 1)
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q, k = _rotated(q, cos, sin, c["interleaved"]).to(bf16), _rotated(k, cos, sin, c["interleaved"])
    of, at = s["slots"] // page, s["slots"] % page
    if c["kv"] == "bf16":
        s["pages"][0][of, :, at] = k.to(bf16)
        s["pages"][1][of, :, at] = v.to(bf16)
        return {"q": q, "k_pages": s["pages"][0], "v_pages": s["pages"][1]}
    (ck, sk), (cv, sv) = _quantized(k), _quantized(v)
    for pages, rows in zip(s["pages"], (_packed(ck), _packed(cv), sk, sv)):
        pages[of, :, at] = rows
    of, at = s["all"] // page, s["all"] % page
    kp, vp, ks, vs = (pages[of, :, at] for pages in s["pages"])
    return {"q": q, "k": _values(kp, ks).to(bf16), "v": _values(vp, vs).to(bf16)}


def _prompt_plain(s):
    q, k, v, cu_q = s["q"].float(), s["k"].float(), s["v"].float(), s["cu_q"].long()
    cu_k = cu_q if s["cu_k"] is None else s["cu_k"].long()
    N, H, D = q.shape
    S, Hk, _ = k.shape
    i, j = torch.arange(N, device=DEV), torch.arange(S, device=DEV)
    of_q, of_k = torch.searchsorted(cu_q[1:], i, right=True), torch.searchsorted(cu_k[1:], j, right=True)
    last = cu_k[of_q + 1] - cu_q[of_q + 1] + i       # the last key that a query sees
    seen = (of_q.unsqueeze(1) == of_k) & (j <= last.unsqueeze(1))
    q = q.view(N, Hk, H // Hk, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)
    p = torch.matmul(q, k.permute(1, 2, 0).contiguous()).mul_(D ** -0.5).view(H, N, S)
    p = p.masked_fill_(~seen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(Hk, -1, S), v.transpose(0, 1).contiguous()).view(H, N, D) / total
    return {"y": y.transpose(0, 1).to(s["q"].dtype).contiguous()}


def _decode_plain(s):
    c, table = s["c"], s["table"].long()
    B, H, D = s["q"].shape
    Hk = c["kv_heads"]
    k, v = (pages[table].transpose(1, 2) for pages in s["pages"][:2])      # (B, kv heads, blocks, page, ...)
    if c["kv"] == "q4":
        k, v = (_values(x, pages[table].transpose(1, 2)) for x, pages in zip((k, v), s["pages"][2:]))
    k, v = (x.float().reshape(B * Hk, -1, D) for x in (k, v))
    q = s["q"].float().view(B * Hk, H // Hk, D)
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, H, -1)
    p = p.masked_fill_((torch.arange(p.shape[2], device=DEV) >= s["lengths"].unsqueeze(1)).unsqueeze(1), -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(B * Hk, H // Hk, -1), v).view(B, H, D) / total
    return {"y": y.to(s["q"].dtype)}


def _column(v, B):
    return v.double().unsqueeze(1) if torch.is_tensor(v) else torch.full((B, 1), float(v), dtype=torch.float32, device=DEV).double()


def _sample_plain(s):
    x, u = s["logits"].double(), s["u"].double().unsqueeze(1)
    B, V = x.shape
    temperature, k, p, low = (_column(s[key], B) for key in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(x, dim=1, descending=True, stable=True)          # ties: the lowest index first
    w = ((x - x[:, :1]) / torch.where(temperature > 0, temperature, torch.ones_like(temperature))).exp()
    rank = torch.arange(V, device=DEV)
    keep = (k == 0) | (rank < k)
    w = torch.where(keep, w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    keep = keep & ((p >= 1) | (before < p * w.sum(1, keepdim=True))) & (w >= low) & ((temperature > 0) | (rank < 1))
    keep[:, 0] = True
    w = torch.where(keep, w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w).cumsum(1)                # over the vocabulary in its own order
    return {"token": (w > u * w[:, -1:]).to(torch.uint8).argmax(1)}


# ----------------------------------------------------------------------------------------------------- in 64 bits
@torch.no_grad()
def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "append":
        return _append_exact(s)
    if c["kind"] == "prompt":
        q, k, v, cu_q = s["q"].double(), s["k"].double(), s["v"].double(), s["cu_q"].tolist()
        cu_k = cu_q if s["cu_k"] is None else s["cu_k"].tolist()
        y = torch.zeros_like(q)
        for b in range(c["seqs"]):
            T, S = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
            hidden = torch.ones(T, S, dtype=torch.bool, device=DEV).triu(S - T + 1)
            for h in range(c["heads"]):
                g = h // (c["heads"] // c["kv_heads"])
                score = q[cu_q[b]:cu_q[b + 1], h] @ k[cu_k[b]:cu_k[b + 1], g].T / math.sqrt(c["dim"])
                y[cu_q[b]:cu_q[b + 1], h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v[cu_k[b]:cu_k[b + 1], g]
        return {"y": y}
    if c["kind"] == "decode":
        q, y = s["q"].double(), torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lengths"].tolist()):
            ids = s["table"][b].long()
            if c["kv"] == "q4":
                k, v = (_values(x[ids], z[ids], torch.float64) for x, z in zip(s["pages"][:2], s["pages"][2:]))
            else:
                k, v = (x[ids].double() for x in s["pages"])
            k, v = (x.transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n] for x in (k, v))
            share = c["heads"] // c["kv_heads"]
            for g in range(c["kv_heads"]):
                of = slice(g * share, (g + 1) * share)
                y[b, of] = torch.softmax(q[b, of] @ k[g].T / math.sqrt(c["dim"]), 1) @ v[g]
        return {"y": y}
    return {"token": _sample_exact(s)}


def _append_exact(s):
    c = s["c"]
    H, Hk, page = c["heads"], c["kv_heads"], c["page"]
    rows = s["qkv"].double().view(-1, H + 2 * Hk, c["dim"])
    # a rotation of each pair as a product of complex numbers
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]].unsqueeze(1)
    n = c["rot"] // 2
    head = rows[:, :H + Hk, :c["rot"]]
    pairs = head.unflatten(-1, (n, 2)) if c["interleaved"] else head.unflatten(-1, (2, n)).transpose(-1, -2)
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    rows[:, :H + Hk, :c["rot"]] = (pairs if c["interleaved"] else pairs.transpose(-1, -2)).flatten(-2)
    q, k, v = rows.split([H, Hk, Hk], 1)
    where = (s["slots"] // page, slice(None), s["slots"] % page)
    if c["kv"] == "bf16":
        pages = [x.double() for x in s["pages"]]
        pages[0][where], pages[1][where] = k, v
        return {"q": q, "k_pages": pages[0], "v_pages": pages[1]}
    for x, codes, scales in ((k, s["pages"][0], s["pages"][2]), (v, s["pages"][1], s["pages"][3])):
        code, scale = _quantized(x)
        codes[where], scales[where] = _packed(code), scale
    where = (s["all"] // page, slice(None), s["all"] % page)
    k, v = (_values(s["pages"][i][where], s["pages"][i + 2][where], torch.float64) for i in (0, 1))
    return {"q": q, "k": k, "v": v}


def _sample_exact(s):
    x, u = s["logits"].double(), s["u"].double()
    B, V = x.shape
    got = []
    for b in range(B):
        T, k, p, low = (float(_column(s[key], B)[b]) for key in ("temperature", "top_k", "top_p", "min_p"))
        ids = torch.sort(-x[b], stable=True).indices
        if T == 0:
            got.append(int(ids[0]))
            continue
        ids = ids[:int(k)] if k else ids
        prob = torch.softmax(x[b][ids] / T, 0)
        n = len(ids)
        if p < 1:
            n = max(1, int((prob.cumsum(0) - prob < p).sum()))
        n = max(1, min(n, int((prob >= low * prob[0]).sum())))
        ids, at = torch.sort(ids[:n])
        mass = prob[:n][at].cumsum(0)
        got.append(int(ids[min(int((mass <= u[b] * mass[-1]).sum()), n - 1)]))
    return torch.tensor(got, device=DEV)


# ------------------------------------------------------------------------------------------------------- the work
def work(c):
    if c["kind"] == "sample":
        size = 2 if c["type"] == "bf16" else 4
        return {"bytes": c["rows"] * (c["vocab"] * size + 12), "flops": 4 * c["rows"] * c["vocab"]}
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    lengths = _lengths(c)
    if c["kind"] == "prompt":
        cached = [c["cached"] if i % 2 == 0 else 0 for i in range(len(lengths))]
        pairs = sum(n * (n + 1) // 2 + n * m for n, m in zip(lengths, cached))
        return {"bytes": 2 * D * (2 * H * sum(lengths) + 2 * Hk * sum(n + m for n, m in zip(lengths, cached))),
                "flops": 4 * D * H * pairs}
    row = 2 * D if c["kv"] == "bf16" else D // 2 + 4
    if c["kind"] == "decode":
        return {"bytes": 2 * row * Hk * sum(lengths) + 4 * D * H * c["seqs"] + 4 * sum(-(-n // c["page"]) + 1 for n in lengths),
                "flops": 4 * D * H * sum(lengths)}
    new = sum(n if c["new"] == 0 else min(c["new"], n) for n in lengths)
    moved = new * (2 * D * (2 * H + 2 * Hk) + 2 * row * Hk + 16 + 4 * c["rot"])
    if c["kv"] == "q4":                             # and the cache read back
        moved += sum(lengths) * (2 * Hk * (row + 2 * D) + 8)
    return {"bytes": moved, "flops": new * 6 * D * (H + Hk)}
