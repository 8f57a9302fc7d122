"""Keys, values and normed rows in 8 bits on the PyTorch op set: formats, refusals, ops against 64 bits, the engine."""
import pathlib
import random
import re
import types
import weakref

import fp8_oracle as oracle
import pytest
import torch

from tinyllmforge_b200 import LLM, Config, SamplingParams, preset
from tinyllmforge_b200.ops import ref
from tinyllmforge_b200.ops.quant import Fp8BlockWeight, Fp8KVCache, Fp8Rows, linear_fp8_ref, quantize_heads
from tinyllmforge_b200.utils.synth import write_checkpoint

F64 = torch.float64


def test_heads_take_the_smallest_power_of_two_that_holds_them():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(300, 128, generator=g) * torch.exp(20 * torch.randn(300, 1, generator=g))
    codes, scales = quantize_heads(x)
    oracle.check_quantised(codes, scales, x.to(F64), torch.zeros(300, dtype=F64))


@pytest.mark.parametrize("top,byte", [(448.0, 127), (448.0 * (1 + 2 ** -23), 128), (449.0, 128), (224.0, 126), (1.0, 119), (1.75, 119), (1.75 + 2 ** -22, 120),
                                      (0.0, 1), (2.0 ** -140, 1), (3e38, 247), (448.0 * 2.0 ** -126, 1), (449.0 * 2.0 ** -126, 2)])
def test_scale_bytes_at_the_borders(top, byte):
    x = torch.zeros(2, 128)
    x[0, 5], x[1, 77] = top, -top
    codes, scales = quantize_heads(x)
    assert scales.tolist() == [byte, byte]
    assert torch.equal(codes[0].float()[5], -codes[1].float()[77])


@pytest.mark.parametrize("top,value", [(247.0, 240.0), (248.0, 240.0), (248.0 + 2 ** -16, 240.0), (255.0, 240.0), (256.0 - 2 ** -16, 240.0), (231.0, 224.0), (233.0, 240.0)])
def test_the_largest_finite_heads_stay_finite(top, value):
    """Entries in units of 2^120, the largest scale that 32 bits give: 256 of them would be infinite, and 240 is within half a step (2^-4)
    of everything below."""
    x = torch.full((2, 128), 2.0 ** 118)
    x[0, 5], x[1, 77] = top * 2.0 ** 120, -top * 2.0 ** 120
    codes, scales = quantize_heads(x)
    assert scales.tolist() == [247, 247] and codes[0].float()[5] == value and codes[1].float()[77] == -value
    v = Fp8KVCache(codes, scales).dequantize()
    assert v.isfinite().all() and v.to(torch.bfloat16).isfinite().all()
    oracle.check_quantised(codes, scales, x.to(F64), torch.zeros(2, dtype=F64))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_heads_that_are_not_finite_read_back_as_nan(bad):
    x = torch.ones(3, 4, 128)
    x[1, 2, 7] = bad
    cache = Fp8KVCache(*quantize_heads(x))
    v = cache.dequantize()
    assert cache.scales[1, 2] == 255 and v[1, 2].isnan().all()
    v[1, 2] = 1.0
    assert torch.equal(v, torch.ones_like(v))


def test_cache_parts_share_memory_and_mismatches_are_refused():
    cache = Fp8KVCache.zeros(3, 2, 5, 2, 16, 8)
    part = cache[1, 0]
    assert part.shape == (5, 2, 16, 8)
    part.code_bytes[2, 1, 3] = 0x38                     # 1.0
    part.scales[2, 1, 3] = 128
    assert cache.dequantize()[1, 0, 2, 1, 3].tolist() == [2.0] * 8 and int(cache.code_bytes.count_nonzero()) == 8
    codes, scales = cache.codes, cache.scales
    for c, s in ((codes.float(), scales), (codes, scales.int()), (codes, scales[:, :1]), (codes[..., :4], scales[..., :4])):
        with pytest.raises(ValueError):
            Fp8KVCache(c, s)
    for q, s in ((torch.zeros(3, 256), torch.zeros(2, 4)), (torch.zeros(3, 200).to(oracle.E4M3), torch.zeros(2, 4)),
                 (torch.zeros(3, 256).to(oracle.E4M3), torch.zeros(2, 2)), (torch.zeros(3, 256).to(oracle.E4M3), torch.zeros(3, 4))):
        with pytest.raises(ValueError):
            Fp8Rows(q, s)


def _stored(T, H, kv, d, bs, blocks, slots, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (H + 2 * kv) * d, generator=g)
    w = [1 + 0.2 * torch.randn(d, generator=g) for _ in range(2)]
    table = ref.rope_table(64, d, 1e4)
    pos = torch.randint(0, 64, (T,), generator=g, dtype=torch.int32)
    kc, vc = Fp8KVCache.zeros(blocks, kv, bs, d), Fp8KVCache.zeros(blocks, kv, bs, d)
    q = ref.RefOps.qk_norm_rope_store(qkv, *w, 1e-6, table, pos, torch.tensor(slots, dtype=torch.int32), kc, vc, H, kv, d)
    return qkv.view(T, H + 2 * kv, d), w, table, pos, q, kc, vc


def test_store_writes_quantised_heads_and_passes_over_negative_slots():
    H, kv, d, bs = 4, 2, 128, 16
    slots = [17, -1, 40, 3, 16]
    x, w, table, pos, q, kc, vc = _stored(5, H, kv, d, bs, 4, slots)
    want_k = oracle.head(x[:, H:H + kv], w[1], 1e-6, table, pos)
    close = (q.to(F64) - oracle.head(x[:, :H], w[0], 1e-6, table, pos)).abs().amax()
    assert close < 1e-5
    written = torch.zeros(4, kv, bs, dtype=torch.bool)
    for t, s in enumerate(slots):
        if s >= 0:
            at = (s // bs, slice(None), s % bs)
            for cache, want in ((kc, want_k[t]), (vc, x[t, H + kv:].to(F64))):
                oracle.check_quantised(cache.codes[at], cache.scales[at], want, want.abs().amax(-1) * 2.0 ** -18)
            written[at] = True
    assert not kc.scales[~written].any() and not vc.code_bytes[~written].any()


def test_attention_is_that_of_the_values_the_cache_stands_for():
    g = torch.Generator().manual_seed(1)
    kc, vc = (Fp8KVCache(*quantize_heads(torch.randn(9, 2, 16, 64, generator=g))) for _ in range(2))
    q = torch.randn(8, 6, 64, generator=g)

    class B:
        cu_seqlens_q, context_lens = torch.tensor([0, 5, 8]), torch.tensor([33, 3])
        block_tables, num_seqs = torch.tensor([[4, 0, 7], [2, -1, -1]]), 2

    got = ref.RefOps.attention(q, kc, vc, B, 0.2)
    assert torch.equal(got, ref.RefOps.attention(q, kc.dequantize(), vc.dequantize(), B, 0.2))


def test_expanded_pages_are_the_cache_in_order():
    g = torch.Generator().manual_seed(2)
    kc, vc = (Fp8KVCache(*quantize_heads(torch.randn(9, 2, 16, 8, generator=g))) for _ in range(2))
    tables = torch.tensor([[4, 0, 7], [-1, -1, -1], [2, 4, -1]], dtype=torch.int32)
    k, v, t = ref.RefOps.expand_kv(kc, vc, tables, torch.tensor([33, 0, 32]), 6)
    assert t.tolist() == [[0, 1, 2], [-1] * 3, [3, 4, -1]]
    for x, c in ((k, kc), (v, vc)):
        full = c.dequantize()
        for page, block in ((0, 4), (1, 0), (3, 2), (4, 4)):
            assert torch.equal(x[page].float(), full[block])
        assert torch.equal(x[2, :, :1].float(), full[7, :, :1]) and not x[2, :, 1:].any() and not x[5].any()


@pytest.mark.parametrize("residual", [False, True])
def test_normed_rows_in_8_bits(residual):
    g = torch.Generator().manual_seed(3)
    x, r = (torch.randn(7, 384, generator=g).bfloat16() for _ in range(2))
    x[3], r[3] = 0, 0
    w = (1 + 0.2 * torch.randn(384, generator=g)).bfloat16()
    rows, s = ref.RefOps.rms_norm_fp8(x, r if residual else None, w, 1e-6)
    want, stream = oracle.norm_rows(x, r if residual else None, w, 1e-6)
    oracle.check_rows(rows, want)
    assert torch.equal(s.to(F64), stream) and rows.scale[:, 3].tolist() == [1.0] * 3
    weight = Fp8BlockWeight.quantize(torch.randn(128, 384, generator=g))
    y = linear_fp8_ref(rows, weight)
    assert y.dtype == torch.bfloat16 and torch.allclose(y.float(), rows.dequantize() @ weight.dequantize().t(), rtol=2 ** -7, atol=1e-3)


def _llm(**kw):
    base = dict(hf_config=preset("tiny", hidden_size=256, intermediate_size=512), load_format="dummy", skip_tokenizer_init=True, device="cpu",
                kvcache_block_size=16, max_model_len=256, max_num_batched_tokens=256, num_kvcache_blocks=64, kv_cache_dtype="fp8")
    return LLM("x", **{**base, **kw})


def _tokens(prompts, **kw):
    llm = _llm(**kw)
    outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True), use_tqdm=False)
    cache, cached = llm.worker.model.kv_cache, llm.stats.to_dict()["prefix_cached_tokens"]
    llm.exit()
    return [o["token_ids"] for o in outs], cache, cached


@pytest.mark.parametrize("quantization", [None, "fp8_block"])
def test_engine_serves_from_an_8_bit_cache(quantization):
    rng = random.Random(0)
    prompts = [[rng.randrange(4096) for _ in range(n)] for n in (5, 40, 100)]
    prompts.append(prompts[-1][:64] + [1, 2, 3])
    whole, cache, cached = _tokens(prompts, quantization=quantization)
    assert isinstance(cache, Fp8KVCache) and cached >= 64 and all(len(t) == 8 for t in whole)
    chunked, _, _ = _tokens(prompts, quantization=quantization, max_num_batched_tokens=32, chunked_prefill=True)
    # a prompt attends to the values the cache stands for, however it was cut; only the order of fp32 sums differs
    assert sum(a == b for s, t in zip(whole, chunked) for a, b in zip(s, t)) >= 0.9 * 32
    plain, cache, _ = _tokens(prompts, kv_cache_dtype=None, quantization=quantization)
    assert isinstance(cache, torch.Tensor) and len(plain) == 4


def test_two_ranks_serve_from_8_bit_caches_of_their_heads(tmp_path):
    path = str(tmp_path / "tiny")
    write_checkpoint(path, preset("tiny"), seed=0, std=0.2, norm_std=0.1)
    rng = random.Random(1)
    prompts = [[rng.randrange(4096) for _ in range(n)] for n in (5, 40, 100)]
    tokens = []
    for size in (1, 2):
        llm = LLM(path, device="cpu", kvcache_block_size=16, max_model_len=256, max_num_batched_tokens=256, num_kvcache_blocks=64, kv_cache_dtype="fp8",
                  tensor_parallel_size=size)
        tokens.append([o["token_ids"] for o in llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True), use_tqdm=False)])
        assert llm.worker.model.kv_cache.shape[3] == 2 // size         # KV heads of a rank
        llm.exit()
    # the ranks' sums are added in another order: 2^-24 of an entry, which moves few codes over a border
    assert sum(a == b for s, t in zip(*tokens) for a, b in zip(s, t)) >= 0.9 * 24


def test_block_bytes_and_norms_in_8_bits_follow_the_options():
    llm = _llm(quantization="fp8_block")
    m = llm.worker.model
    assert m.kv_block_bytes(16) == 2 * 2 * 16 * 2 * 65 and m.expansion_bytes(10) == 2 * 10 * 2 * 64 * 4 and m.norms_fp8
    llm.exit()
    for kw in (dict(quantization="fp8_block", kv_cache_dtype=None), dict(quantization=None)):
        llm = _llm(**kw)
        assert not llm.worker.model.norms_fp8
        llm.exit()


def test_options_that_do_not_go_with_an_8_bit_cache_are_refused():
    from tinyllmforge_b200.models.goselix_config import GoselixConfig, example_dict
    with pytest.raises(ValueError, match="kv_cache_dtype must be"):
        Config("x", hf_config=preset("tiny"), device="cpu", kv_cache_dtype="int8")
    with pytest.raises(ValueError, match="not available for GoselixConfig"):
        Config("x", hf_config=GoselixConfig.from_dict(example_dict(2048)), device="cpu", kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="heads of 128"):
        Config("x", hf_config=preset("tiny"), device="cuda", kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="bfloat16"):
        Config("x", hf_config=preset("qwen3-0.6b"), device="cuda", dtype="float32", kv_cache_dtype="fp8")
    assert Config("x", hf_config=preset("qwen3-0.6b"), device="cuda", kv_cache_dtype="fp8").kv_cache_dtype == "fp8"


def test_decode_steps_store_where_attention_reads():
    """A sequence whose blocks were reserved beyond its newest token: the step's slot is in the block of that token, in every later step too."""
    from tinyllmforge_b200 import SamplingParams
    from tinyllmforge_b200.engine.request import Request
    from tinyllmforge_b200.engine.step_batch import DecodeBuilder, build_decode
    reqs = []
    for n, table in ((5, [3, 7, 1]), (16, [2, 0]), (17, [5, 4])):
        r = Request(list(range(n)), SamplingParams(temperature=0.0))
        r.block_table = table
        reqs.append(r)
    builder = DecodeBuilder(16)
    for i in range(12):
        want = [r.block_table[(len(r) - 1) // 16] * 16 + (len(r) - 1) % 16 for r in reqs]
        for step in (build_decode(reqs, 16), builder.build(reqs, 0, 0, None, None)):
            at, size = step.offsets["slot_mapping"]
            assert step.buf[at:at + size].tolist() == want
        for r in reqs:
            r.append_token(1)


def _prompt_ops(tokens, bs):
    """The prompt attention of the GPU over stand-ins of its kernels; ``most``: pages that were read back and alive at once, ``portions``: (sequences, pages)."""
    from tinyllmforge_b200.ops.cuda_fp8 import Fp8Ops
    ops, alive = Fp8Ops(), weakref.WeakSet()
    ops.expand_tokens, ops.status, ops.portions, ops.most = tokens, None, [], 0

    def expand(kc, ks, vc, vs, tables, lens, pages, status):
        out = tuple(torch.empty(pages, 1, bs, 128, dtype=torch.bfloat16) for _ in range(2))
        alive.update(out)
        ops.most = max(ops.most, sum(t.shape[0] for t in alive))
        return (*out, tables.clone())

    def attend(q, k, v, cu, lens, tables, out, n, *rest):
        ops.portions.append((n, k.shape[0]))

    ops.C = types.SimpleNamespace(fp8_expand=expand, prefill_attention=attend)
    return ops


def test_a_portions_pages_are_freed_before_the_next_is_read_back():
    """A step of several portions holds the pages of one at a time: that much is in the peak that the cache is sized after."""
    bs, lens = 16, [64, 48, 16, 100, 33, 0, 128]
    ops = _prompt_ops(128, bs)
    cache = Fp8KVCache.zeros(4, 1, bs, 128)

    class B:
        num_seqs, max_seqlen_q, key_lens = len(lens), 1, lens
        block_tables, context_lens = torch.zeros(len(lens), 8, dtype=torch.int32), torch.tensor(lens)
        cu_seqlens_q = torch.arange(len(lens) + 1)

    ops.prefill_attention_fp8(torch.zeros(len(lens), 1, 128, dtype=torch.bfloat16), cache, cache, B, 1.0)
    assert ops.portions == [(3, 8), (1, 7), (2, 3), (1, 8)]
    assert ops.most == 2 * 8                             # keys and values


@pytest.mark.parametrize("budget,max_len,seqs,bs,pages", [
    (16384, 9000, 512, 256, 64 - 36),                    # the warm-up has one prompt of 9000 tokens, later portions up to 64 pages
    (16384, 4096, 512, 256, 0), (16384, 9000, 1, 256, 0),
    (16384, 40960, 512, 256, 160 - 64), (2048, 100, 512, 64, 32 - 32), (2048, 90, 3, 64, 0), (1000, 700, 512, 16, 62 - 44),
    (1000, 300, 512, 256, 3 - 2),                        # at most 3 pages together: one prompt of two in the warm-up, 300 and 200 tokens later
])
def test_the_cache_leaves_room_for_the_largest_portion_read_back(budget, max_len, seqs, bs, pages):
    """Beyond what the warm-up has read back: the most that any step of this configuration does."""
    from tinyllmforge_b200.engine.worker import warmup_lengths
    cfg = Config("x", hf_config=preset("tiny", max_position_embeddings=max_len), device="cpu", kvcache_block_size=bs, max_model_len=max_len,
                 max_num_batched_tokens=budget, max_num_seqs=seqs, chunked_prefill=True, kv_cache_dtype="fp8")
    model = _llm().worker.model
    warm = warmup_lengths(cfg)
    assert model.expansion_beyond(cfg, warm) == model.expansion_bytes(pages * bs)
    rng, cache = random.Random(0), Fp8KVCache.zeros(1, 1, bs, 128)

    def most(lens):
        ops = _prompt_ops(budget, bs)
        step = types.SimpleNamespace(num_seqs=len(lens), max_seqlen_q=1, key_lens=lens, block_tables=torch.zeros(len(lens), 1, dtype=torch.int32),
                                     context_lens=torch.tensor(lens), cu_seqlens_q=torch.arange(len(lens) + 1))
        ops.prefill_attention_fp8(torch.zeros(len(lens), 1, 128, dtype=torch.bfloat16), cache, cache, step, 1.0)
        return max(p for _, p in ops.portions)

    for _ in range(50):
        lens = [rng.choice((1, max_len, rng.randint(1, max_len))) for _ in range(rng.randint(1, min(seqs, 40)))]
        assert most(lens) <= most(warm) + pages
    model.fp8_cache = False
    assert model.expansion_beyond(cfg, warm) == 0


def test_the_rule_for_steps_from_the_raw_projection_refuses_heads_that_do_not_go_together():
    _C = pytest.importorskip("tinyllmforge_b200._C")
    from tinyllmforge_b200.ops.cuda import CudaOps
    ops = object.__new__(CudaOps)
    ops.C, ops.fused_qkv_max_batch, ops.decode_attention_mode = _C, 32, "auto"
    step = types.SimpleNamespace(padded_seqs=1, table_width=2)
    assert ops.decodes_from_projection(step, 16, Fp8KVCache.zeros(2, 8, 64, 128))
    for heads, kv_heads, block in ((4, 8, 64), (0, 1, 64), (7, 2, 64), (4, 0, 64), (-8, 8, 64), (8, 8, 24), (8, 8, 8)):
        with pytest.raises(RuntimeError, match="decode_fp8_qkv_pays"):
            ops.decodes_from_projection(step, heads, Fp8KVCache.zeros(2, kv_heads, block, 128))


@pytest.mark.parametrize("source", ["attn/fp8_cache.cu", "attn/decode_fp8.cu", "elt/norm_fp8.cu", "include/fp8_cache.cuh"])
def test_kernels_take_nothing_for_constant_that_the_kernel_before_them_writes(source):
    """They start beside their predecessor's end, and a pointer to const that is declared restrict lets the compiler load through it before the
    wait, or through a cache that is not kept up to date."""
    text = (pathlib.Path(__file__).parent.parent / "csrc" / source).read_text()
    code = re.sub(r"//[^\n]*", "", text)
    assert "__restrict__" not in code and "__ldg" not in code and "ld.global.nc" not in code


@pytest.mark.parametrize("ahead", [0, 1, 3])
def test_decode_steps_built_one_after_the_other_equal_rebuilt_ones(ahead):
    """Tables that grow as sequences do, with blocks reserved ahead at any time: equal in every word, but for entries behind the newest token's block."""
    from tinyllmforge_b200.engine.request import Request
    from tinyllmforge_b200.engine.step_batch import DecodeBuilder, build_decode
    rng, bs, width = random.Random(ahead), 8, 16
    reqs = [Request(list(range(n)), SamplingParams(temperature=0.5)) for n in (1, 7, 8, 9, 30)]
    free = iter(range(1000))
    builder = DecodeBuilder(bs)
    for step in range(60):
        for r in reqs:
            need = -(-len(r) // bs) + (rng.randint(0, ahead) if rng.random() < 0.3 else 0)
            r.block_table += [next(free) for _ in range(need - len(r.block_table))]
        got, want = builder.build(reqs, step, 5, 8, width), build_decode(reqs, bs, step, 5, 8, width)
        a, b = got.buf[:got.num_words].copy(), want.buf
        at, size = got.offsets["block_tables"]
        for i, r in enumerate(reqs):
            last = (len(r) - 1) // bs + 1                # entries that are read
            rows = [x[at + i * width:at + (i + 1) * width] for x in (a, b)]
            assert rows[0][:last].tolist() == rows[1][:last].tolist() == r.block_table[:last]
            for x in rows:
                if ahead:
                    x[last:] = -1
        assert (a == b).all()
        for r in reqs:
            r.append_token(rng.randrange(100))
