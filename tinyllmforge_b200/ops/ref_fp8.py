"""Plain-PyTorch ops of an 8-bit KV cache and of norms with 8-bit rows: the CPU path and the oracle of ``ops/cuda_fp8.py``.

Everything between an op's operands and the one rounding of its result is fp32.
"""
from __future__ import annotations

import torch

from .quant import Fp8KVCache, Fp8Rows, quantize_activations_ref, quantize_heads


def store_kv(k, v, k_cache: Fp8KVCache, v_cache: Fp8KVCache, slot_mapping) -> None:
    """k, v fp32 [T, kv_heads, d]; a slot < 0 is passed over."""
    bs = k_cache.shape[2]
    slots = slot_mapping.long()
    keep = slots >= 0
    blk, off = slots[keep] // bs, slots[keep] % bs
    for x, cache in ((k, k_cache), (v, v_cache)):
        codes, scales = quantize_heads(x[keep])
        cache.code_bytes[blk, :, off] = codes.view(torch.uint8)
        cache.scales[blk, :, off] = scales


def qk_norm_rope_store(qkv, q_weight, k_weight, eps, table, positions, slot_mapping, k_cache, v_cache, num_heads, num_kv_heads, head_dim, do_rope=True):
    """``ref.qk_norm_rope_store`` into an 8-bit cache, without roundings on the way; q is rounded to the type of ``qkv``."""
    from .ref import apply_rope
    T = qkv.shape[0]
    q, k, v = qkv.float().split([num_heads * head_dim, num_kv_heads * head_dim, num_kv_heads * head_dim], dim=-1)

    def head(x, weight):
        x = x.reshape(T, -1, head_dim)
        if weight is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
        return apply_rope(x, positions, table) if do_rope else x

    store_kv(head(k, k_weight), v.reshape(T, num_kv_heads, head_dim), k_cache, v_cache, slot_mapping)
    return head(q, q_weight).to(qkv.dtype)


def expand_kv(k_cache, v_cache, block_tables, context_lens, num_pages, dtype=torch.bfloat16):
    """The sequences' pages in order: (keys, values) ``[num_pages, kv_heads, block_size, d]``, entries behind a sequence's last token zero,
    and the page numbers ``[sequences, width]``, -1 behind the last."""
    bs = k_cache.shape[2]
    out = [torch.zeros(num_pages, *k_cache.shape[1:], dtype=dtype, device=k_cache.device) for _ in range(2)]
    tables = torch.full(block_tables.shape, -1, dtype=torch.int32, device=block_tables.device)
    at = 0
    for s, n in enumerate(context_lens.tolist()):
        for j in range(-(-n // bs)):
            live = min(bs, n - j * bs)
            for x, cache in zip(out, (k_cache, v_cache)):
                x[at, :, :live] = cache[int(block_tables[s, j])].dequantize()[:, :live].to(dtype)
            tables[s, j] = at
            at += 1
    return out[0], out[1], tables


def rms_norm_fp8(x, residual, weight, eps):
    """(``Fp8Rows`` of the normed rows, new residual): ``add_rms_norm`` whose normed rows are quantised per 128 columns, from fp32."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    y = s.float()
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    return Fp8Rows(*quantize_activations_ref(y), dtype=x.dtype), s
