"""One-kernel cases of an 8-bit KV cache and of norms with 8-bit rows (see ``kernel_case``): sizes of the Qwen3-8B layers.

Every entry returns (callable, bytes, flops): what the operation has to move and to multiply, each input read once and each output written once.
"""
from __future__ import annotations

import torch

BF = torch.bfloat16
D, BLOCK = 128, 256


def _cache(blocks, kv_heads):
    from ..ops.quant import Fp8KVCache, quantize_heads
    return Fp8KVCache(*quantize_heads(torch.randn(blocks, kv_heads, BLOCK, D, device="cuda")))


class _Step:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _step(B, ctx, longest=0):
    """B sequences of ctx tokens; the table has room for ``longest`` (captured steps of the engine: for ``max_model_len``)."""
    need, width = -(-ctx // BLOCK), -(-max(ctx, longest) // BLOCK)
    tables = torch.full((B, width), -1, dtype=torch.int32)
    tables[:, :need] = torch.randperm(B * need, dtype=torch.int32).view(B, need)
    return _Step(is_prefill=False, num_seqs=B, padded_seqs=B, table_width=width, max_seqlen_k=ctx, blocks=B * need, block_tables=tables.cuda(),
                 context_lens=torch.full((B,), ctx, dtype=torch.int32, device="cuda"))


def _decode(ops, B, ctx, heads, kv_heads, longest=0):
    step = _step(B, ctx, longest)
    kc, vc = (_cache(step.blocks, kv_heads) for _ in range(2))
    q = torch.randn(B, heads, D, device="cuda").to(BF)
    return (lambda: ops.attention(q, kc, vc, step, D ** -0.5)), 2 * B * ctx * kv_heads * (D + 1) + 4 * q.numel(), 4 * B * ctx * heads * D


def _decode_qkv(ops, B, ctx, heads, kv_heads):
    from ..ops.ref import rope_table
    step = _step(B, ctx)
    kc, vc = (_cache(step.blocks, kv_heads) for _ in range(2))
    qkv = torch.randn(B, (heads + 2 * kv_heads) * D, device="cuda").to(BF)
    w, table = torch.ones(D, device="cuda", dtype=BF), rope_table(ctx, D, 1e6, "cuda")
    return ((lambda: ops.decode_attention_qkv(qkv, w, w, 1e-6, table, kc, vc, step, heads, D ** -0.5)),
            2 * B * ctx * kv_heads * (D + 1) + 2 * qkv.numel() + 2 * B * heads * D, 4 * B * ctx * heads * D)


def _expand(ops, B, ctx, kv_heads):
    step = _step(B, ctx)
    kc, vc = (_cache(step.blocks, kv_heads) for _ in range(2))
    return ((lambda: ops.expand_kv(kc, vc, step.block_tables, step.context_lens, step.blocks)),
            2 * B * ctx * kv_heads * (D + 1 + 2 * D), 0)


def _store(ops, T, heads, kv_heads):
    from ..ops.quant import Fp8KVCache
    from ..ops.ref import rope_table
    qkv = torch.randn(T, (heads + 2 * kv_heads) * D, device="cuda").to(BF)
    w = torch.ones(D, device="cuda", dtype=BF)
    table, at = rope_table(T, D, 1e6, "cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    kc, vc = (Fp8KVCache.zeros(-(-T // BLOCK), kv_heads, BLOCK, D, device="cuda") for _ in range(2))
    return ((lambda: ops.qk_norm_rope_store(qkv, w, w, 1e-6, table, at, at, kc, vc, heads, kv_heads, D)),
            T * (2 * (heads + 2 * kv_heads) * D + 2 * heads * D + 2 * kv_heads * (D + 1) + 4 * D), 0)


def _norm(ops, M, H):
    x, r = (torch.randn(M, H, device="cuda").to(BF) for _ in range(2))
    w = torch.ones(H, device="cuda", dtype=BF)
    return (lambda: ops.rms_norm_fp8(x, r, w, 1e-6)), 7 * M * H + M * H // 32, 0


CASES = {
    "fp8_decode": lambda ops: _decode(ops, 256, 800, 32, 8),
    "fp8_decode_g8": lambda ops: _decode(ops, 64, 2304, 64, 8),
    "fp8_decode_few": lambda ops: _decode(ops, 4, 3000, 32, 8),
    "fp8_decode_qkv": lambda ops: _decode_qkv(ops, 1, 1000, 32, 8),
    "fp8_decode_qkv_16": lambda ops: _decode_qkv(ops, 16, 768, 32, 8),
    "fp8_decode_16": lambda ops: _decode(ops, 16, 768, 32, 8),
    "fp8_decode_16_wide": lambda ops: _decode(ops, 16, 768, 32, 8, longest=4096),
    "fp8_expand": lambda ops: _expand(ops, 8, 4352, 8),
    "fp8_store": lambda ops: _store(ops, 16384, 32, 8),
    "norm_fp8": lambda ops: _norm(ops, 16384, 4096),
}
