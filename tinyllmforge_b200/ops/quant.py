"""Tensors held in 8 bits.  The reference has no quantised path.

* Block-scaled fp8 weights (``quantization="fp8_block"``): e4m3 values with one fp32 scale per 128 x 128 block, bf16 activations
  quantised on the fly per token and per 128 input features, or handed over by the norm before them as ``Fp8Rows``.
* The 8-bit KV cache (``kv_cache_dtype="fp8"``): e4m3 codes with one power-of-two scale per token and head.
"""
from __future__ import annotations

import torch

BLOCK = 128
E4M3_MAX = 448.0


class Fp8BlockWeight:
    """A linear weight ``[N, K]`` stored as e4m3 + block scales ``[ceil(N / 128), K / 128]``."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
        self.q, self.scale = q.contiguous(), scale.contiguous()
        self.shape = tuple(q.shape)
        self.dtype = torch.bfloat16
        self.device = q.device

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Fp8BlockWeight":
        N, K = w.shape
        if K % BLOCK:
            raise ValueError(f"in_features ({K}) must be a multiple of {BLOCK} for fp8_block")
        nb = -(-N // BLOCK)
        wf = torch.zeros(nb * BLOCK, K, dtype=torch.float32, device=w.device)
        wf[:N] = w.float()
        blocks = wf.view(nb, BLOCK, K // BLOCK, BLOCK)
        amax = blocks.abs().amax(dim=(1, 3))
        scale = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
        q = (blocks / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(nb * BLOCK, K)[:N].to(torch.float8_e4m3fn)
        return cls(q, scale)

    def dequantize(self) -> torch.Tensor:
        N, K = self.shape
        s = self.scale.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)
        return self.q.float() * s

    def __getitem__(self, idx):        # row slices at block granularity (gate / up halves)
        raise TypeError("slice the bf16 weight before quantising")


def quantize_activations_ref(x: torch.Tensor):
    """Per token, per 128 features: (e4m3 values, scales [K / 128, M]).  Oracle of the CUDA quantiser."""
    M, K = x.shape
    xb = x.float().view(M, K // BLOCK, BLOCK)
    amax = xb.abs().amax(-1)
    s = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    q = (xb / s[..., None]).view(M, K).to(torch.float8_e4m3fn)
    return q, s.t().contiguous()


class Fp8Rows:
    """Activations ``[M, K]`` as e4m3 values ``q`` with fp32 scales ``scale`` ``[K / 128, >= M]``, one per row and 128 columns: what a
    projection with an ``Fp8BlockWeight`` multiplies.  ``dtype``: the type of the projection's result."""

    __slots__ = ("q", "scale", "dtype")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        if q.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32 or q.dim() != 2 or scale.dim() != 2:
            raise ValueError("Fp8Rows: e4m3 values [M, K] and fp32 scales [K / 128, >= M] expected")
        (M, K), (groups, columns) = q.shape, scale.shape
        if K != groups * BLOCK or columns < M:
            raise ValueError(f"Fp8Rows: scales {tuple(scale.shape)} do not belong to values {tuple(q.shape)}")
        self.q, self.scale, self.dtype = q, scale, dtype

    @classmethod
    def of(cls, q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> "Fp8Rows":
        """Of tensors that belong together by their making."""
        rows = object.__new__(cls)
        rows.q, rows.scale, rows.dtype = q, scale, dtype
        return rows

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    def dequantize(self) -> torch.Tensor:
        M, K = self.shape
        return (self.q.float().view(M, K // BLOCK, BLOCK) * self.scale[:, :M].t()[..., None]).view(M, K)


def linear_fp8_ref(x: "torch.Tensor | Fp8Rows", w: Fp8BlockWeight) -> torch.Tensor:
    """What the fp8 kernel computes, in fp32: quantised activations times quantised weights."""
    if isinstance(x, Fp8Rows):
        return (x.dequantize() @ w.dequantize().t()).to(x.dtype)
    q, s = quantize_activations_ref(x)
    xd = q.float().view(x.shape[0], -1, BLOCK) * s.t()[..., None]
    return (xd.view(x.shape[0], -1) @ w.dequantize().t()).to(x.dtype)


def quantize_heads(x: torch.Tensor):
    """fp32 ``[..., d]`` -> (e4m3 codes ``[..., d]``, scale bytes ``[...]``) of an 8-bit KV cache: a byte b stands for 2^(b - 127), the
    smallest power of two (not below 2^-126) with which no entry exceeds 448.  A finite head stays finite: under the largest scale, 2^120,
    entries from 248 on are held as 240, which is within half a step of them (256 would be infinite).  A head with an entry that is
    not finite has NaN in every code, and 255 (NaN)."""
    amax = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)                               # amax = mantissa 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > E4M3_MAX / 512).to(exponent.dtype)
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(-126, 127)
    bad = ~torch.isfinite(amax)
    most = torch.where(e == 120, 240.0, E4M3_MAX)[..., None]
    codes = torch.ldexp(x, -e[..., None]).clamp(-most, most).masked_fill(bad[..., None], float("nan")).to(torch.float8_e4m3fn)
    return codes, (e + 127).masked_fill(bad, 255).to(torch.uint8)


class Fp8KVCache:
    """Keys or values in 8 bits: e4m3 ``codes`` ``[..., block_size, head_dim]`` and a byte of ``scales`` ``[..., block_size]`` per token and
    head (see ``quantize_heads``).  One layer's half is ``[blocks, kv_heads, block_size, head_dim]``, as the bf16 cache is; leading
    dimensions are indexed as a tensor's are, and the parts share the memory."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.uint8:
            raise ValueError(f"Fp8KVCache: float8_e4m3fn codes and uint8 scales expected, got {codes.dtype} and {scales.dtype}")
        if codes.shape[:-1] != scales.shape:
            raise ValueError(f"Fp8KVCache: scales {tuple(scales.shape)} do not belong to codes {tuple(codes.shape)}")
        if codes.device != scales.device:
            raise ValueError("Fp8KVCache: codes and scales on one device expected")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return self.codes.shape

    @property
    def dtype(self):
        return self.codes.dtype

    @property
    def device(self):
        return self.codes.device

    @classmethod
    def zeros(cls, *shape: int, device="cpu") -> "Fp8KVCache":
        return cls(torch.zeros(*shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                   torch.zeros(*shape[:-1], dtype=torch.uint8, device=device))

    @property
    def code_bytes(self) -> torch.Tensor:
        return self.codes.view(torch.uint8)

    def __getitem__(self, idx) -> "Fp8KVCache":
        return Fp8KVCache(self.code_bytes[idx].view(torch.float8_e4m3fn), self.scales[idx])

    def dequantize(self) -> torch.Tensor:
        """fp32 values."""
        scale = torch.ldexp(torch.ones_like(self.scales, dtype=torch.float32), self.scales.int() - 127)
        return self.codes.float() * scale.masked_fill(self.scales == 255, float("nan"))[..., None]
