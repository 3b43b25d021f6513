"""The reference operator surface on torch CUDA tensors.

One function per reference launcher, same argument order and meaning
(Inference_gpt2/GEMV.cuh, GEMV_w8.cuh, attention_kvcache(_w8).cuh,
layernorm.cuh, encoder.cuh, sampler_gpu.cuh); the storage type is taken from
the tensors and the current length is a device tensor (``d_pos``) instead of
the reference's ``g_cur_len`` symbol.  Every call goes to libgpt2b.so and
raises :class:`Gpt2bError` on a non-zero status; torch only supplies device
memory and the current stream.  The operators for batches of requests over a
paged 4-bit cache and for drafted tokens, at the end, have no counterpart there.
"""
from __future__ import annotations

import ctypes

import torch

from . import Gpt2bError, check, lib


def _p(t):
    return None if t is None else t.data_ptr()


def _s(stream):
    return (stream if stream is not None else torch.cuda.current_stream()).cuda_stream


def _sfx(t):
    return {torch.float32: "f32", torch.bfloat16: "bf16"}[t.dtype]


def launch_GEMV6(out, W, x, M, K, stream=None):
    """out[M] (fp32) = W[M,K] . x  (GEMV.cuh:112)."""
    fn = getattr(lib(), f"gpt2b_launch_GEMV6_{_sfx(W)}")
    check(fn(_p(out), _p(W), _p(x), M, K, _s(stream)), "launch_GEMV6")


def launch_GEMV6_fused(out, pre_gelu, W, x, bias, M, K, do_gelu, stream=None):
    """out = gelu?(W.x + b), pre_gelu <- W.x + b  (GEMV.cuh:204)."""
    fn = getattr(lib(), f"gpt2b_launch_GEMV6_fused_{_sfx(W)}")
    check(fn(_p(out), _p(pre_gelu), _p(W), _p(x), _p(bias), M, K, int(bool(do_gelu)), _s(stream)),
          "launch_GEMV6_fused")


def launch_GEMV6_w8x2(out, pre_gelu, W, x, scale, bias, M, K, do_gelu, fmt="int8", stream=None):
    """8-bit weight-only GEMV (GEMV_w8.cuh:162); fp32 `out` selects the LM-head form."""
    sfx = "i8" if fmt == "int8" else "fp8"
    if out.dtype == torch.float32:
        fn = getattr(lib(), f"gpt2b_launch_GEMV6_w8x2_{sfx}_f32out")
        check(fn(_p(out), _p(W), _p(x), _p(scale), M, K, _s(stream)), "launch_GEMV6_w8x2")
    else:
        fn = getattr(lib(), f"gpt2b_launch_GEMV6_w8x2_{sfx}")
        check(fn(_p(out), _p(pre_gelu), _p(W), _p(x), _p(scale), _p(bias), M, K, int(bool(do_gelu)), _s(stream)),
              "launch_GEMV6_w8x2")


def dequant_wte(w8, scale, out, Vp, C, fmt="int8", stream=None):
    fn = getattr(lib(), "gpt2b_dequant_wte_" + ("i8" if fmt == "int8" else "fp8"))
    check(fn(_p(w8), _p(scale), _p(out), Vp, C, _s(stream)), "dequant_wte")


def quant_rows(W, W8, scale, M, K, fmt="int8", stream=None):
    fn = getattr(lib(), "gpt2b_quant_rows_" + ("i8" if fmt == "int8" else "fp8"))
    check(fn(_p(W), _p(W8), _p(scale), M, K, _s(stream)), "quant_rows")


def kv_cache_write(kv_cache, qkv, B, NH, hs, maxT, d_pos, kv_scale=None, fmt=None, stream=None):
    if kv_cache.dtype == torch.uint8:
        fn = getattr(lib(), "gpt2b_kv_cache_write_w8_" + ("i8" if fmt == "int8" else "fp8"))
        check(fn(_p(kv_cache), _p(kv_scale), _p(qkv), B, NH, hs, maxT, _p(d_pos), _s(stream)), "kv_cache_write_w8")
    else:
        fn = getattr(lib(), f"gpt2b_kv_cache_write_{_sfx(kv_cache)}")
        check(fn(_p(kv_cache), _p(qkv), B, NH, hs, maxT, _p(d_pos), _s(stream)), "kv_cache_write")


def attention_forward_kv_small(out, qkv, kv_cache, B, NH, hs, maxT, d_pos, kv_scale=None, fmt=None, stream=None):
    if kv_cache.dtype == torch.uint8:
        fn = getattr(lib(), "gpt2b_attention_forward_kv_small_w8_" + ("i8" if fmt == "int8" else "fp8"))
        check(fn(_p(out), _p(qkv), _p(kv_cache), _p(kv_scale), B, NH, hs, maxT, _p(d_pos), _s(stream)),
              "attention_forward_kv_small_w8")
    else:
        fn = getattr(lib(), f"gpt2b_attention_forward_kv_small_{_sfx(kv_cache)}")
        check(fn(_p(out), _p(qkv), _p(kv_cache), B, NH, hs, maxT, _p(d_pos), _s(stream)),
              "attention_forward_kv_small")


def attention_forward_kv_large(out, qkv, kv_cache, B, NH, hs, maxT, d_pos, part_out, part_lse, part_max, S,
                               kv_scale=None, fmt=None, stream=None):
    if kv_cache.dtype == torch.uint8:
        fn = getattr(lib(), "gpt2b_attention_forward_kv_large_w8_" + ("i8" if fmt == "int8" else "fp8"))
        check(fn(_p(out), _p(qkv), _p(kv_cache), _p(kv_scale), B, NH, hs, maxT, _p(d_pos), _s(stream),
                 _p(part_out), _p(part_lse), _p(part_max), S), "attention_forward_kv_large_w8")
    else:
        fn = getattr(lib(), f"gpt2b_attention_forward_kv_large_{_sfx(kv_cache)}")
        check(fn(_p(out), _p(qkv), _p(kv_cache), B, NH, hs, maxT, _p(d_pos), _s(stream), _p(part_out),
                 _p(part_lse), _p(part_max), S), "attention_forward_kv_large")


def attention_kv_split(part_out, part_lse, part_max, qkv, kv_cache, B, NH, hs, maxT, S, d_pos, kv_scale=None,
                       fmt=None, stream=None):
    """The split half alone (attention_kv_split_kernel(_w8), attention_kvcache.cuh:185, _w8.cuh:260)."""
    if kv_cache.dtype == torch.uint8:
        fn = getattr(lib(), "gpt2b_attention_kv_split_w8_" + ("i8" if fmt == "int8" else "fp8"))
        check(fn(_p(part_out), _p(part_lse), _p(part_max), _p(qkv), _p(kv_cache), _p(kv_scale), B, NH, hs, maxT, S,
                 _p(d_pos), _s(stream)), "attention_kv_split_w8")
    else:
        fn = getattr(lib(), f"gpt2b_attention_kv_split_{_sfx(kv_cache)}")
        check(fn(_p(part_out), _p(part_lse), _p(part_max), _p(qkv), _p(kv_cache), B, NH, hs, maxT, S, _p(d_pos),
                 _s(stream)), "attention_kv_split")


def attention_kv_merge(out, part_out, part_lse, part_max, B, NH, hs, S, w8=False, stream=None):
    """The merge half alone (attention_kv_merge_kernel(_w8), attention_kvcache.cuh:298, _w8.cuh:374)."""
    name = "gpt2b_attention_kv_merge_w8" if w8 else f"gpt2b_attention_kv_merge_{_sfx(out)}"
    check(getattr(lib(), name)(_p(out), _p(part_out), _p(part_lse), _p(part_max), B, NH, hs, S, _s(stream)),
          "attention_kv_merge")


def matmul_forward(out, inp, weight, bias, B, T, C, OC, pre_gelu=None, scale=None, fmt=None, stream=None):
    """out[B*T, OC] = inp . weight^T (+ bias), on the tensor cores
    (matmul_forward_cublaslt, matmul.cuh:141).  BF16 inp; weight BF16 or 8-bit
    codes (uint8 + per-row ``scale``, ``fmt`` "int8"/"fp8"); FP32 ``out``
    selects the LM-head form (no bias); ``pre_gelu`` fuses tanh-GELU."""
    w8 = weight.dtype == torch.uint8
    sfx = ("i8" if fmt == "int8" else "fp8") if w8 else None
    if out.dtype == torch.float32:
        if w8:
            rc = getattr(lib(), f"gpt2b_matmul_forward_w8_{sfx}_f32out")(_p(out), _p(inp), _p(weight), _p(scale), B, T,
                                                                          C, OC, _s(stream))
        else:
            rc = lib().gpt2b_matmul_forward_f32out_bf16(_p(out), _p(inp), _p(weight), B, T, C, OC, _s(stream))
    elif w8:
        rc = getattr(lib(), f"gpt2b_matmul_forward_w8_{sfx}")(_p(out), _p(inp), _p(weight), _p(scale), _p(bias), B, T,
                                                               C, OC, _p(pre_gelu), _s(stream))
    else:
        rc = lib().gpt2b_matmul_forward_bf16(_p(out), _p(inp), _p(weight), _p(bias), B, T, C, OC, _p(pre_gelu),
                                             _s(stream))
    check(rc, "matmul_forward")


def layernorm_forward(out, mean, rstd, inp, weight, bias, B, T, C, stream=None):
    fn = getattr(lib(), f"gpt2b_layernorm_forward_{_sfx(inp)}")
    check(fn(_p(out), _p(mean), _p(rstd), _p(inp), _p(weight), _p(bias), B, T, C, _s(stream)), "layernorm_forward")


def fused_residual_forward5(residual, normed, mean, rstd, inp1, inp2, weight, bias, N, C, stream=None):
    fn = getattr(lib(), f"gpt2b_fused_residual_forward5_{_sfx(inp1)}")
    check(fn(_p(residual), _p(normed), _p(mean), _p(rstd), _p(inp1), _p(inp2), _p(weight), _p(bias), N, C,
             _s(stream)), "fused_residual_forward5")


def encoder_forward_kv(out, inp, wte, wpe, d_pos, B, C, stream=None):
    fn = getattr(lib(), f"gpt2b_encoder_forward_kv_{_sfx(wte)}")
    check(fn(_p(out), _p(inp), _p(wte), _p(wpe), _p(d_pos), B, C, _s(stream)), "encoder_forward_kv")


def gpu_sample_softmax(d_token, logits, B, V, seed, step, stream=None):
    check(lib().gpt2b_gpu_sample_softmax(_p(d_token), _p(logits), B, V, seed, step, _s(stream)),
          "gpu_sample_softmax")


def gpu_argmax(d_token, logits, B, V, ld=None, stream=None):
    check(lib().gpt2b_gpu_argmax(_p(d_token), _p(logits), B, V, ld or V, _s(stream)), "gpu_argmax")


# ---------------------------------------------------------------------------
# batches of requests over a paged 4-bit KV cache, and drafted tokens
# ---------------------------------------------------------------------------
# These take their sizes from the tensors and check them (a wrong size would reach
# memory that is not theirs), run on the tensors' device whatever the current one
# is, and without ``stream`` on that device's current stream.  The checks and the
# call are compiled (csrc/bind.cpp): in Python they would cost more than the kernels.
_bind = None


def _b():
    global _bind
    if _bind is None:
        dll = lib()
        try:
            from . import _bind as module
        except ImportError as e:
            raise ImportError("the operators for batches need _bind.so, built against the torch and Python in use: "
                              "build it with `python -m cuda_gpt2_inference_b200.build`") from e
        module.init(Gpt2bError, {n: ctypes.cast(getattr(dll, n), ctypes.c_void_p).value for n in
                                 ("gpt2b_kv_block_tables", "gpt2b_kv_cache_write_w4", "gpt2b_kv_cache_read_w4",
                                  "gpt2b_attention_forward_paged_w4", "gpt2b_softmax_probs", "gpt2b_verify_draft_tokens")})
        _bind = module
    return _bind


def kv_block_tables(block_table, slot_map, positions, row_start, seq_lens, blocks_out, free_left, ctx_lens, new_lens,
                    blocks_have, free_list, free_count, block_size, stream=None):
    """Block tables, slot map and row offsets of one step from the requests'
    lengths (gpt2b_kv_block_tables).  int32, but ``slot_map`` int64; block_table
    [B, max_blocks], slot_map and positions [max_rows], row_start [B+1], free_list
    [any], free_left and free_count [1], the others [B]."""
    _b().kv_block_tables(block_table, slot_map, positions, row_start, seq_lens, blocks_out, free_left, ctx_lens, new_lens,
                         blocks_have, free_list, free_count, block_size, stream)


def kv_cache_write_w4(kv_cache, kv_scale, qkv, slot_map, NH, stream=None):
    """Append the K and V of packed qkv rows to the paged 4-bit cache at
    ``slot_map`` (gpt2b_kv_cache_write_w4).  kv_cache uint8 [blocks, 2, NKV,
    block_size, hs/2], kv_scale BF16 [blocks, 2, NKV, block_size, hs/64, 2], qkv BF16
    [rows, >= (NH + 2 NKV) hs], rows possibly further apart; slot_map int64 [rows],
    negative: skipped."""
    _b().kv_cache_write_w4(kv_cache, kv_scale, qkv, slot_map, NH, stream)


def kv_cache_read_w4(out, kv_cache, kv_scale, slot_map, stream=None):
    """Read rows of the paged 4-bit cache back as BF16 [rows, 2, NKV, hs]
    (gpt2b_kv_cache_read_w4); zeros for negative slots."""
    _b().kv_cache_read_w4(out, kv_cache, kv_scale, slot_map, stream)


def attention_paged_w4_workspace(NH, NKV, hs, max_q):
    """Bytes of the workspace of :func:`attention_forward_paged_w4` on the current device."""
    n = ctypes.c_size_t()
    check(lib().gpt2b_attention_paged_w4_workspace(NH, NKV, hs, max_q, ctypes.byref(n)), "attention_paged_w4_workspace")
    return n.value


def attention_forward_paged_w4(out, qkv, kv_cache, kv_scale, block_table, seq_lens, row_start, NH, max_q, workspace,
                               scale=None, stream=None):
    """Attention of packed rows over the paged 4-bit cache, causal among a
    request's rows (gpt2b_attention_forward_paged_w4).  out BF16 [rows, NH hs], cache
    and qkv as for :func:`kv_cache_write_w4`, block_table int32 [B, max_blocks], seq_lens
    [B], row_start [B+1]; ``max_q`` the most rows a request has (a hint);
    ``workspace`` uint8 of :func:`attention_paged_w4_workspace` bytes; ``scale``
    of the scores, default 1/sqrt(hs)."""
    _b().attention_forward_paged_w4(out, qkv, kv_cache, kv_scale, block_table, seq_lens, row_start, NH, max_q, workspace,
                                    scale, stream)


def softmax_probs(probs, logits, temperature=1.0, V=None, stream=None):
    """probs = softmax(logits / temperature) per row over the first ``V`` (default:
    all) columns; temperature 0: one-hot at the largest (gpt2b_softmax_probs).
    FP32 [rows, >= V]; ``probs`` may be ``logits``."""
    _b().softmax_probs(probs, logits, temperature, V, stream)


def verify_draft_tokens(out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample, stream=None):
    """Accept drafted tokens and draw the next one by rejection sampling from given
    random numbers (gpt2b_verify_draft_tokens).  out_tokens int32 [B, max_out],
    n_accepted [B], tokens int32 [rows] (packed: last token, then drafts),
    target_probs FP32 [rows, V], draft_probs the same or None (certain drafts),
    row_start int32 [B+1], u_accept FP32 [rows], u_sample [B]."""
    _b().verify_draft_tokens(out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample, stream)
