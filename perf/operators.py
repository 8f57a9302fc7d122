"""The operators of serving in 8 bits whose speed is measured: what a decode step does to and with a cache of e4m3 keys and values,
and the norm that hands 8-bit rows to a projection with block-scaled fp8 weights.

``store``   per-head norm and rotation of the packed qkv projection; keys and values quantised into the paged cache, queries in bf16
``expand``  the pages of sequences read back as bf16 pages, in order: what prompt attention reads when a prefix is cached
``decode``  attention of one new token per sequence over the paged 8-bit cache
``norm``    root-mean-square norm with the residual's addition, and an output in e4m3 with a scale for every 128 entries

A cache holds, for every token and head, 128 e4m3 codes and one byte b that scales them by 2^(b - 127).  The scale is the smallest
power of two with which no entry exceeds 448, the largest e4m3 number.

``own``: the framework's kernels; otherwise the same mathematics in plain torch.
"""
import math
import random

import torch

own = False

D = 128                       # head size
EPS = 1e-6
E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one user's newest token: all latency
        {"name": "store 1", "op": "store", "tokens": 1, "pad": 0, "heads": 16, "kv_heads": 8, "block": 256},
        # a decode step of a thinned-out batch, padded to its graph
        {"name": "store 61", "op": "store", "tokens": 61, "pad": 3, "heads": 32, "kv_heads": 8, "block": 256},
        # a long prompt
        {"name": "store 4001", "op": "store", "tokens": 4001, "pad": 0, "heads": 32, "kv_heads": 8, "block": 64},
        # a follow-up question: the conversation so far is cached
        {"name": "expand 1", "op": "expand", "seqs": 1, "lo": 700, "hi": 700, "kv_heads": 8, "block": 256},
        # a token budget of ragged prompts
        {"name": "expand 28", "op": "expand", "seqs": 28, "lo": 100, "hi": 1024, "kv_heads": 8, "block": 256},
        # requests behind a shared system prompt of 4096 tokens
        {"name": "expand 8", "op": "expand", "seqs": 8, "lo": 4352, "hi": 4352, "kv_heads": 8, "block": 256},
        # one user, some way into a conversation: latency again
        {"name": "decode 1", "op": "decode", "seqs": 1, "pad": 0, "lo": 3001, "hi": 3001, "heads": 32, "kv_heads": 8, "block": 256},
        # a few users of a model with five query heads to a key head
        {"name": "decode 13", "op": "decode", "seqs": 13, "pad": 3, "lo": 200, "hi": 2000, "heads": 40, "kv_heads": 8, "block": 64},
        # steady state of the 256-request benchmark workload
        {"name": "decode 256", "op": "decode", "seqs": 256, "pad": 0, "lo": 100, "hi": 1500, "heads": 16, "kv_heads": 8, "block": 256},
        # long documents and a wide group of heads
        {"name": "decode 9 long", "op": "decode", "seqs": 9, "pad": 0, "lo": 9000, "hi": 32000, "heads": 64, "kv_heads": 8, "block": 256},
        # a decode step's rows before a projection
        {"name": "norm 61", "op": "norm", "rows": 61, "hidden": 4096, "residual": True},
        # many rows of an odd number
        {"name": "norm 8191", "op": "norm", "rows": 8191, "hidden": 2560, "residual": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["store", "expand", "decode", "norm"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (40, 8), (64, 8), (8, 1), (5, 1), (4, 2), (12, 4)])
    block = rng.choice([16, 32, 64, 256, 256])
    if op == "store":
        tokens = _log(rng, 1, 4001 * 48 // (heads + 2 * kv_heads) if heads > 32 else 4001)
        return {"op": op, "tokens": tokens, "pad": rng.randint(0, 15) if tokens <= 512 else 0, "heads": heads, "kv_heads": kv_heads, "block": block}
    if op == "norm":
        hidden = rng.choice([1024, 2048, 2560, 4096, 5120])
        return {"op": op, "rows": _log(rng, 1, 8191 * 2560 // hidden), "hidden": hidden, "residual": rng.random() < 0.7}
    if op == "expand":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, min(8192, 8 * 4352 * 8 // (seqs * kv_heads)))
        return {"op": op, "seqs": seqs, "lo": rng.randint(1, hi), "hi": hi, "kv_heads": kv_heads, "block": block}
    seqs = _log(rng, 1, 256)
    hi = _log(rng, 1, min(32000, 9 * 20500 * 8 // (seqs * kv_heads)))
    return {"op": op, "seqs": seqs, "pad": rng.randint(0, 15), "lo": rng.randint(1, hi), "hi": hi, "heads": heads, "kv_heads": kv_heads, "block": block}


def _lengths(case):
    """The sequences' lengths, spread evenly from lo to hi."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    op = case["op"]
    if op == "store":
        T, H, kv = case["tokens"], case["heads"], case["kv_heads"]
        return {"bytes": T * (2 * (H + 2 * kv) * D + 2 * H * D + 2 * kv * (D + 1) + 4 * D + 8), "flops": T * (H + kv) * D * 10}
    if op == "norm":
        n = case["rows"] * case["hidden"]
        return {"bytes": n * (7 if case["residual"] else 3) + n // 32, "flops": 8 * n}
    keys = sum(_lengths(case))
    if op == "expand":
        return {"bytes": keys * case["kv_heads"] * 2 * (D + 1 + 2 * D), "flops": keys * case["kv_heads"] * 2 * D}
    return {"bytes": keys * case["kv_heads"] * 2 * (D + 1) + case["seqs"] * case["heads"] * D * 4, "flops": keys * case["heads"] * 4 * D}


# --------------------------------------------------------------------------------------------------------------- inputs
class Step:
    """What the attention calls read of a step."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _quantise(x):
    """fp32 [..., 128] -> (e4m3 codes, scale bytes)."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1))                   # amax = mantissa 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > 0.875).int()                          # 448 = 0.875 2^9
    e = torch.where(mantissa == 0, -126, e).clamp(-126, 127)
    return torch.ldexp(x, -e[..., None]).to(E4M3), (e + 127).to(torch.uint8)


def _pages(case, gen):
    """A cache's number of blocks, and the sequences' tables: blocks in shuffled order, -1 behind the last."""
    lens = torch.tensor(_lengths(case), device="cuda")
    lens = lens[torch.randperm(case["seqs"], generator=gen, device="cuda")]
    need = -(-lens // case["block"])
    width = int(need.max())
    total = int(need.sum())
    order = torch.randperm(total + 3, generator=gen, device="cuda")[:total]
    slot = torch.arange(width, device="cuda")
    live = slot[None] < need[:, None]
    first = need.cumsum(0) - need
    tables = torch.where(live, order[(first[:, None] + slot[None]).clamp(max=total - 1)], -1)
    return total, lens.int(), tables.int()


def _cache(blocks, case, gen, spread):
    """Codes and scale bytes of keys or values whose heads have sizes of their own."""
    shape = (blocks, case["kv_heads"], case["block"])
    size = torch.exp(spread * torch.randn(*shape, 1, generator=gen, device="cuda"))
    return _quantise(torch.randn(*shape, D, generator=gen, device="cuda") * size)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if op == "norm":
        n, h = case["rows"], case["hidden"]
        return {"op": op, "x": randn(n, h).to(BF16), "residual": (4 * randn(n, h)).to(BF16) if case["residual"] else None,
                "weight": (1 + 0.2 * randn(h)).to(BF16)}
    if op == "store":
        T, H, kv, bs = case["tokens"], case["heads"], case["kv_heads"], case["block"]
        blocks = -(-T // bs) + 2
        slots = torch.randperm(blocks, generator=gen, device="cuda")[:, None] * bs + torch.arange(bs, device="cuda")
        start = random.Random(seed).randrange(0, 512)
        positions = torch.arange(start, start + T, device="cuda")
        pad = torch.zeros(case["pad"], dtype=torch.int64, device="cuda")
        angles = torch.outer(torch.arange(5120, dtype=torch.float64), 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
        return {"op": op, "heads": H, "kv_heads": kv, "live": T, "qkv": randn(T + case["pad"], (H + 2 * kv) * D).to(BF16),
                "q_weight": (1 + 0.2 * randn(D)).to(BF16), "k_weight": (1 + 0.2 * randn(D)).to(BF16),
                "table": torch.cat((angles.cos(), angles.sin()), -1).float().cuda(),
                "positions": torch.cat((positions, pad)).int(), "slots": torch.cat((slots.reshape(-1)[:T], pad - 1)).int(),
                "codes": torch.zeros(2, blocks, kv, bs, D, dtype=torch.uint8, device="cuda").view(E4M3),
                "scales": torch.zeros(2, blocks, kv, bs, dtype=torch.uint8, device="cuda")}
    total, lens, tables = _pages(case, gen)
    k, ks = _cache(total + 3, case, gen, 0.3)
    v, vs = _cache(total + 3, case, gen, 0.5)
    state = {"op": op, "k": k, "ks": ks, "v": v, "vs": vs, "lens": lens, "tables": tables, "pages": total}
    if op == "decode":
        n, pad = case["seqs"], case["pad"]
        state["lens"] = torch.cat((lens, lens.new_zeros(pad)))
        state["tables"] = torch.cat((tables, tables.new_full((pad, tables.shape[1]), -1)))
        state["q"] = (2 * randn(n + pad, case["heads"], D)).to(BF16)
        state["step"] = Step(is_prefill=False, num_seqs=n, padded_seqs=n + pad, table_width=tables.shape[1], max_seqlen_k=case["hi"],
                             block_tables=state["tables"], context_lens=state["lens"])
    return state


# --------------------------------------------------------------------------------------------------------------- a pass
_handle = None


def _ops():
    global _handle
    if _handle is None:
        from tinyllmforge_b200.ops.cuda import CudaOps
        _handle = CudaOps()
    return _handle


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from tinyllmforge_b200.ops.quant import Fp8KVCache
    ops, op = _ops(), s["op"]
    if op == "store":
        kc, vc = (Fp8KVCache(s["codes"][i], s["scales"][i]) for i in (0, 1))
        q = ops.qk_norm_rope_store(s["qkv"], s["q_weight"], s["k_weight"], EPS, s["table"], s["positions"], s["slots"], kc, vc, s["heads"],
                                   s["kv_heads"], D)
        return {"q": q, "codes": s["codes"], "scales": s["scales"].view(E8M0)}
    if op == "norm":
        rows, stream = ops.rms_norm_fp8(s["x"], s["residual"], s["weight"], EPS)
        return {"rows": rows.q, "scale": rows.scale[:, :s["x"].shape[0]], "stream": stream}
    kc, vc = Fp8KVCache(s["k"], s["ks"]), Fp8KVCache(s["v"], s["vs"])
    if op == "expand":
        k, v, tables = ops.expand_kv(kc, vc, s["tables"], s["lens"], s["pages"])
        return {"k": k, "v": v, "tables": tables}
    return ops.attention(s["q"], kc, vc, s["step"], D ** -0.5)


def _values(codes, scales):
    return torch.ldexp(codes.float(), scales.int()[..., None] - 127)


def _norm_rotate(x, weight, cos, sin):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _run_plain(s):
    op = s["op"]
    if op == "store":
        H, kv, T, live = s["heads"], s["kv_heads"], s["qkv"].shape[0], s["live"]
        q, k, v = s["qkv"].view(T, H + 2 * kv, D).split([H, kv, kv], 1)
        cs = s["table"][s["positions"].long()][:, None]
        q = _norm_rotate(q, s["q_weight"], cs[..., :D // 2], cs[..., D // 2:])
        k = _norm_rotate(k, s["k_weight"], cs[..., :D // 2], cs[..., D // 2:])
        codes, scales = _quantise(torch.stack((k, v.float()))[:, :live])
        bs = s["codes"].shape[3]
        slots = s["slots"][:live].long()
        s["codes"].view(torch.uint8)[:, slots // bs, :, slots % bs] = codes.view(torch.uint8).transpose(0, 1)
        s["scales"][:, slots // bs, :, slots % bs] = scales.transpose(0, 1)
        return {"q": q.to(BF16), "codes": s["codes"], "scales": s["scales"].view(E8M0)}
    if op == "norm":
        x = s["x"] if s["residual"] is None else s["residual"].add_(s["x"])
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["weight"].float()
        parts = y.view(y.shape[0], -1, 128)
        most = parts.abs().amax(-1)
        scale = torch.where(most > 0, most / 448, 1.0)
        return {"rows": (parts / scale[..., None]).to(E4M3).view(y.shape), "scale": scale.t(), "stream": x}
    tables, lens = s["tables"].long(), s["lens"].long()
    bs = s["k"].shape[2]
    if op == "expand":
        need = -(-lens // bs)
        slot = torch.arange(tables.shape[1], device="cuda")
        first = need.cumsum(0) - need
        page = torch.arange(s["pages"], device="cuda")
        of = torch.searchsorted(first + need, page, right=True)          # the sequence of a page
        at = page - first[of]
        left = (lens[of] - at * bs)[:, None, None, None] > torch.arange(bs, device="cuda")[:, None]
        from_block = tables[of, at]
        k, v = (torch.where(left, _values(s[c][from_block], s[x][from_block]), 0.0).to(BF16) for c, x in (("k", "ks"), ("v", "vs")))
        return {"k": k, "v": v, "tables": torch.where(slot < need[:, None], first[:, None] + slot, -1).int()}
    n, H = s["q"].shape[:2]
    kv, keys = s["k"].shape[1], tables.shape[1] * bs
    block = tables.clamp(min=0)
    k = _values(s["k"][block], s["ks"][block]).transpose(2, 3).reshape(n, keys, kv, D).transpose(1, 2)
    q = s["q"].float().view(n, kv, H // kv, D)
    scores = q @ k.transpose(2, 3) * D ** -0.5
    del k
    seen = (torch.arange(keys, device="cuda") < lens[:, None])[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    p = torch.where(seen, torch.exp(scores - scores.amax(-1, keepdim=True)), 0.0)
    v = _values(s["v"][block], s["vs"][block]).transpose(2, 3).reshape(n, keys, kv, D).transpose(1, 2)
    total = p.sum(-1, keepdim=True)
    return (p @ v / torch.where(total > 0, total, 1.0)).to(BF16).view(n, H * D)


# --------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The results in 64 bits, sequence by sequence; what is held in 8 bits as it was before it was rounded to them."""
    s, op = prepare(case, seed), case["op"]
    F64 = torch.float64
    if op == "store":
        H, kv, T, live, bs = case["heads"], case["kv_heads"], s["qkv"].shape[0], s["live"], case["block"]
        heads = s["qkv"].to(F64).view(T, H + 2 * kv, D)
        at = s["table"].to(F64)[s["positions"].long()].view(T, 1, 2, D // 2)

        def head(x, w):
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.to(F64)
            z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * torch.complex(at[:, :, 0], at[:, :, 1])
            return torch.cat((z.real, z.imag), -1)

        q = head(heads[:, :H], s["q_weight"])
        codes = torch.zeros(s["codes"].shape, dtype=F64, device="cuda")
        scales = torch.full(s["scales"].shape, 2.0 ** -127, dtype=F64, device="cuda")
        slots = s["slots"][:live].long()
        for i, x in enumerate((head(heads[:, H:H + kv], s["k_weight"]), heads[:, H + kv:])):
            x = x[:live]
            step = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 448)).clamp(-126, 127))
            codes[i, slots // bs, :, slots % bs] = x / step[..., None]
            scales[i, slots // bs, :, slots % bs] = step
        return {"q": q, "codes": codes, "scales": scales}
    if op == "norm":
        x = s["x"].to(F64)
        stream = x if s["residual"] is None else x + s["residual"].to(F64)
        held = stream.to(BF16).to(F64)                                   # the stream is held in bf16, and the norm is the held stream's
        y = held / (held.square().mean(1, keepdim=True) + EPS).sqrt() * s["weight"].to(F64)
        scale = torch.stack([part.abs().amax(1) for part in y.split(128, 1)]) / 448
        scale[scale == 0] = 1
        return {"rows": y / scale.t().repeat_interleave(128, 1), "scale": scale, "stream": stream}
    bs, lens = case["block"], s["lens"].tolist()

    def sequence(codes, scales, i):
        blocks = s["tables"][i, :-(-lens[i] // bs)].long()
        x = codes[blocks].to(F64) * torch.pow(2.0, scales[blocks].to(F64) - 127)[..., None]
        return x.transpose(0, 1).reshape(case["kv_heads"], -1, D)[:, :lens[i]]

    if op == "expand":
        out = {}
        for name, x in (("k", "ks"), ("v", "vs")):
            pages = []
            for i, n in enumerate(lens):
                rows = sequence(s[name], s[x], i)
                full = torch.zeros(case["kv_heads"], -(-n // bs) * bs, D, dtype=F64, device="cuda")
                full[:, :n] = rows
                pages.append(full.view(case["kv_heads"], -1, bs, D).transpose(0, 1))
            out[name] = torch.cat(pages)
        tables, at = torch.full(s["tables"].shape, -1, dtype=torch.int32, device="cuda"), 0
        for i, n in enumerate(lens):
            need = -(-n // bs)
            tables[i, :need] = torch.arange(at, at + need, device="cuda")
            at += need
        return {**out, "tables": tables}
    out = torch.zeros(len(lens), case["heads"], D, dtype=F64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for i, n in enumerate(lens):
        if n:
            k, v = (sequence(s[c], s[x], i).repeat_interleave(group, 0) for c, x in (("k", "ks"), ("v", "vs")))
            scores = torch.einsum("hd,hkd->hk", s["q"][i].to(F64), k) / math.sqrt(D)
            out[i] = torch.einsum("hk,hkd->hd", torch.softmax(scores, -1), v)
    return out.view(len(lens), -1)
