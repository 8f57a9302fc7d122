"""CUDA ops that keep keys, values and normed rows in 8 bits (types: ``ops/quant.py``).

Queries and results are bf16, heads have 128 entries, cache blocks 16 tokens or more (a power of two).
"""
from __future__ import annotations

import torch

from .quant import Fp8KVCache, Fp8Rows

_DECODE_MODES = {"auto": 0, "flat": 1, "chunked": 2}


def expand_pages(tokens: int, block_size: int) -> int:
    """Pages that a portion of several sequences has at most, for a step's budget of ``tokens``."""
    return max(1, tokens // block_size)


def expand_portions(lens, block_size: int, tokens: int):
    """(begin, end, pages): the sequences, in order, that a prompt's attention reads back together: as many as have ``expand_pages`` pages,
    one at least."""
    begin = 0
    while begin < len(lens):
        end, pages = begin, 0
        while end < len(lens) and (end == begin or pages + -(-lens[end] // block_size) <= expand_pages(tokens, block_size)):
            pages += -(-lens[end] // block_size)
            end += 1
        yield begin, end, pages
        begin = end


def largest_portion(max_seqs: int, max_len: int, block_size: int, tokens: int) -> int:
    """Pages of the largest portion of any step of up to ``max_seqs`` sequences of up to ``max_len`` tokens."""
    one = -(-max_len // block_size)
    return max(one, min(expand_pages(tokens, block_size), max_seqs * one))


class Fp8Ops:
    """Mixed into ``CudaOps`` (uses its ``C``, ``status``, ``device`` and ``num_sms``)."""

    @staticmethod
    def _halves(k_cache, v_cache) -> tuple:
        if not (isinstance(k_cache, Fp8KVCache) and isinstance(v_cache, Fp8KVCache)):
            raise TypeError("keys and values must both be held in 8 bits, or neither")
        return k_cache.codes, k_cache.scales, v_cache.codes, v_cache.scales

    def store_fp8(self, qkv, q_weight, k_weight, eps, table, positions, slot_mapping, k_cache, v_cache, num_heads, do_rope=True):
        """``qk_norm_rope_store`` into an 8-bit cache: what is stored is rounded once, from fp32, and so is q.  The slots of a call are
        distinct; a negative one is passed over."""
        return self.C.fp8_store(qkv, q_weight, k_weight, eps, table if do_rope else None, positions, slot_mapping,
                                *self._halves(k_cache, v_cache), num_heads, self.status)

    def expand_kv(self, k_cache, v_cache, block_tables, context_lens, num_pages):
        """The sequences' pages read back, in order: (keys, values) bf16 ``[num_pages, kv_heads, block_size, 128]``, exact, entries behind a
        sequence's last token zero; and the page numbers ``[sequences, width]``, -1 behind the last.  ``num_pages``: at least the
        pages of all sequences (pages without a sequence are left as they are); one too many for it is reported and left out."""
        return self.C.fp8_expand(*self._halves(k_cache, v_cache), block_tables, context_lens, num_pages, self.status)

    def decode_attention_fp8(self, q, k_cache, v_cache, batch, scale):
        """``decode_attention_mode``: "flat" equal shares over the GPU, "chunked" a cluster of CTAs per sequence and KV head, "auto" by size."""
        return self.C.decode_fp8(q, *self._halves(k_cache, v_cache), batch.block_tables, batch.context_lens, scale, self.status,
                                 _DECODE_MODES.get(self.decode_attention_mode, 2))

    def decode_attention_qkv_fp8(self, qkv, q_weight, k_weight, eps, table, k_cache, v_cache, batch, num_heads, scale, do_rope=True):
        """``decode_attention_qkv`` over an 8-bit cache: ``store_fp8`` at positions length - 1 and ``decode_attention_fp8`` in one, with their bits.
        It knows only the "chunked" partition, whatever ``decode_attention_mode`` is."""
        return self.C.decode_fp8_qkv(qkv, q_weight, k_weight, eps, table if do_rope else None, *self._halves(k_cache, v_cache), batch.block_tables,
                                     batch.context_lens, num_heads, scale, self.status)

    def prefill_attention_fp8(self, q, k_cache, v_cache, batch, scale):
        """Prompts: the sequences' pages are read back and attended to by the bf16 kernels, the pages of one portion
        (``expand_portions``) at a time."""
        T, H, D = q.shape
        out = torch.empty(T, H * D, dtype=q.dtype, device=q.device)
        bs, lens = k_cache.shape[2], getattr(batch, "key_lens", None)
        if lens is None:                          # lengths unknown on the host: as long as the table is wide
            lens = [min(batch.max_seqlen_k, batch.block_tables.shape[1] * bs)] * batch.num_seqs
        for begin, end, pages in expand_portions(lens[:batch.num_seqs], bs, self.expand_tokens):
            part = slice(begin, end)
            if pages:                             # (sequences without keys have no queries either)
                k, v, tables = self.expand_kv(k_cache, v_cache, batch.block_tables[part], batch.context_lens[part], pages)
                self.C.prefill_attention(q, k, v, batch.cu_seqlens_q[begin:end + 1], batch.context_lens[part], tables, out, end - begin,
                                         batch.max_seqlen_q, scale, self.status)
                del k, v, tables                  # before the next portion asks for its own
        return out

    # ------------------------------------------------------------------ norms with 8-bit rows
    def takes_fp8_rows(self, weight, rows: int) -> bool:
        """Whether a projection with this weight multiplies 8-bit rows (with many rows fp8 weights are expanded and rows stay bf16)."""
        return not isinstance(weight, torch.Tensor) and not self._expands_fp8(weight, rows)

    def rms_norm_fp8(self, x, residual, weight, eps):
        """(``Fp8Rows`` of the normed rows, residual): ``add_rms_norm`` whose normed rows leave in 8 bits, quantised from fp32 per 128 columns.
        ``residual`` is updated in place and returned; without one x is."""
        q, scale = self.C.rms_norm_fp8(x, residual, weight, eps)
        return Fp8Rows.of(q, scale, x.dtype), x if residual is None else residual
