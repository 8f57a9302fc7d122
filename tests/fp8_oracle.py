"""What an 8-bit KV cache and 8-bit rows stand for, in 64 bits and entry by entry; shared by the CPU and GPU tests."""
import math

import torch

F64 = torch.float64
E4M3 = torch.float8_e4m3fn


def values(codes, scales):
    """fp64 values of codes [..., d] with scale bytes [...]."""
    scale = torch.pow(2.0, scales.to(F64) - 127)
    scale[scales == 255] = math.nan
    return codes.to(F64) * scale[..., None]


def check_quantised(codes, scales, want, slack):
    """codes and scales of fp64 heads ``want``, which the code under test knows up to ``slack`` (fp64, one per head, absolute)."""
    top = want.abs().amax(-1)
    step = torch.pow(2.0, scales.to(F64) - 127)
    assert (448 * step >= top - slack).all(), "an entry exceeds 448"
    larger = scales > 1
    assert (224 * step < top + slack)[larger].all(), "a smaller scale would do"
    got = values(codes, scales)
    # half a step of e4m3: 2^-4 of the value, and 2^-10 of the scale among the subnormals
    allowed = torch.maximum(want.abs() * 2.0 ** -4, step[..., None] * 2.0 ** -10) + slack[..., None]
    assert ((got - want).abs() <= allowed).all(), "beyond half a step"


def head(x, weight, eps, table, positions):
    """fp64 [T, heads, 128] -> normed (weight may be None) and rotated (table may be None)."""
    x = x.to(F64)
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.to(F64)
    if table is not None:
        cs = table.to(F64)[positions.long()][:, None]
        z = torch.complex(x[..., :64], x[..., 64:]) * torch.complex(cs[..., :64], cs[..., 64:])
        x = torch.cat((z.real, z.imag), -1)
    return x


def attention(q, k, v, scale):
    """One token's attention in fp64: q [H, d], k and v [heads, n, d] -> (out [H, d], allowed error [H, d]).

    Allowed: half a step of bf16 of the result (2^-8).  Every weight may be rounded to 11 bits (half a step 2^-11) and is off by the error
    of its score: sums of 128 products in fp32, 2^-24 of the sum of their absolute values each, with the factors' roundings no more than 2^-20
    of that sum.  Both act on the mean of the |values|, once in the sum and once in what it is divided by; sums over the tokens in
    fp32 add 2^-16 of it at most."""
    g = q.shape[0] // k.shape[0]
    k, v, q = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0), q.to(F64)
    s = torch.einsum("hd,hnd->hn", q, k) * scale
    size = (torch.einsum("hd,hnd->hn", q.abs(), k.abs()) * abs(scale)).amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    out = torch.einsum("hn,hnd->hd", p, v)
    spread = torch.einsum("hn,hnd->hd", p, v.abs())
    return out, out.abs() * 2.0 ** -8 + 2 * spread * (2.0 ** -11 + 2.0 ** -20 * size + 2.0 ** -16)


def sequence(cache, table_row, n):
    """fp64 [kv_heads, n, 128]: the first n tokens of a sequence of an Fp8KVCache."""
    bs = cache.shape[2]
    blocks = table_row[:-(-n // bs)].long()
    x = values(cache.codes.view(torch.uint8)[blocks].view(E4M3), cache.scales[blocks])
    return x.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n]


def norm_rows(x, residual, weight, eps):
    """fp64 (normed rows, stream): the stream is held in the rows' type."""
    s = x.to(F64) if residual is None else (x.to(F64) + residual.to(F64)).to(x.dtype).to(F64)
    return s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * weight.to(F64), s


def check_rows(rows, want):
    """Fp8Rows of fp64 rows ``want`` known up to 2^-18 of themselves (a sum of squares, a root and two products in fp32)."""
    M, K = want.shape
    parts = want.view(M, K // 128, 128)
    top = parts.abs().amax(-1)
    scale = rows.scale[:, :M].t().to(F64)
    ideal = torch.where(top > 0, top / 448, torch.ones_like(top))
    assert ((scale - ideal).abs() <= ideal * 2.0 ** -18).all()
    got = rows.q.to(F64).view(M, K // 128, 128) * scale[..., None]
    allowed = torch.maximum(parts.abs() * 2.0 ** -4, scale[..., None] * 2.0 ** -10) + top[..., None] * 2.0 ** -18
    assert ((got - parts).abs() <= allowed).all()
