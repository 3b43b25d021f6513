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

import contextlib
import ctypes
import math

import torch

from . import ERR_INVALID_ARG, ERR_UNSUPPORTED, Gpt2bError, check, lib


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
# These take their sizes from the tensors and check them: a wrong size would
# reach memory that is not theirs.  They run on the tensors' device (whatever the
# current one) and, without ``stream``, on that device's current stream.
_NULL = contextlib.nullcontext()


def _fail(where, what, status=ERR_INVALID_ARG):
    raise Gpt2bError(status, f"{where}: {what}")


def _need(where, name, t, dtype, ndim, rows=False):
    """A tensor of that type and rank, contiguous (``rows``: only within its rows)."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != ndim:
        _fail(where, f"{name} must be a {ndim}-d {dtype} tensor")
    if not t.is_contiguous() and not (rows and ndim == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]):
        _fail(where, f"{name} must be contiguous")


def _one_device(where, *tensors):
    """The CUDA device that holds every tensor, as a context to call in."""
    dev = tensors[0].device
    if dev.type != "cuda" or any(t is not None and t.device != dev for t in tensors):
        _fail(where, "the tensors must be on one CUDA device")
    return dev, _NULL if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _stream_on(dev, stream):
    return (stream if stream is not None else torch.cuda.current_stream(dev)).cuda_stream


def _w4_cache(where, kv_cache, kv_scale):
    """(num_blocks, NKV, block_size, hs) of a 4-bit cache."""
    _need(where, "kv_cache", kv_cache, torch.uint8, 5)
    _need(where, "kv_scale", kv_scale, torch.bfloat16, 6)
    nb, two, NKV, bs, half = kv_cache.shape
    if two != 2 or tuple(kv_scale.shape) != (nb, 2, NKV, bs, half // 32, 2):
        _fail(where, "kv_cache is [blocks, 2, NKV, block_size, hs/2] and kv_scale [blocks, 2, NKV, block_size, hs/64, 2]")
    if half not in (32, 64) or bs % 16 or bs == 0:
        _fail(where, "head size 64 or 128, block size a multiple of 16", ERR_UNSUPPORTED)
    return nb, NKV, bs, 2 * half


def kv_block_tables(block_table, slot_map, positions, row_start, seq_lens, blocks_out, free_left, ctx_lens, new_lens,
                    blocks_have, free_list, free_count, block_size, stream=None):
    """Block tables, slot map and row offsets of one step from the requests'
    lengths (gpt2b_kv_block_tables).  int32, but ``slot_map`` int64; block_table
    [B, max_blocks], slot_map and positions [max_rows], row_start [B+1], free_list
    [any], free_left and free_count [1], the others [B]."""
    w, i32 = "kv_block_tables", torch.int32
    _need(w, "block_table", block_table, i32, 2)
    _need(w, "slot_map", slot_map, torch.int64, 1)
    B = block_table.shape[0]
    for name, t, n in (("positions", positions, slot_map.shape[0]), ("row_start", row_start, B + 1),
                       ("seq_lens", seq_lens, B), ("blocks_out", blocks_out, B), ("free_left", free_left, 1),
                       ("ctx_lens", ctx_lens, B), ("new_lens", new_lens, B), ("blocks_have", blocks_have, B),
                       ("free_list", free_list, None), ("free_count", free_count, 1)):
        _need(w, name, t, i32, 1)
        if n is not None and t.shape[0] != n:
            _fail(w, f"{name} must have {n} entries")
    dev, on = _one_device(w, block_table, slot_map, positions, row_start, seq_lens, blocks_out, free_left, ctx_lens, new_lens,
                          blocks_have, free_list, free_count)
    with on:
        check(lib().gpt2b_kv_block_tables(block_table.data_ptr(), slot_map.data_ptr(), positions.data_ptr(),
                                          row_start.data_ptr(), seq_lens.data_ptr(), blocks_out.data_ptr(),
                                          free_left.data_ptr(), ctx_lens.data_ptr(), new_lens.data_ptr(),
                                          blocks_have.data_ptr(), free_list.data_ptr(), free_count.data_ptr(), B,
                                          block_table.shape[1], block_size, slot_map.shape[0], free_list.shape[0],
                                          _stream_on(dev, stream)), w)


def kv_cache_write_w4(kv_cache, kv_scale, qkv, slot_map, NH, stream=None):
    """Append the K and V of packed qkv rows to the paged 4-bit cache at
    ``slot_map`` (gpt2b_kv_cache_write_w4).  qkv BF16 [rows, >= (NH + 2 NKV) hs],
    rows possibly further apart; slot_map int64 [rows], negative: skipped."""
    w = "kv_cache_write_w4"
    nb, NKV, bs, hs = _w4_cache(w, kv_cache, kv_scale)
    _need(w, "qkv", qkv, torch.bfloat16, 2, rows=True)
    _need(w, "slot_map", slot_map, torch.int64, 1)
    rows, ld = qkv.shape[0], _row_pitch(qkv)
    if slot_map.shape[0] != rows or qkv.shape[1] < (NH + 2 * NKV) * hs:
        _fail(w, "slot_map has one entry a row, a row Q, K and V of every head")
    dev, on = _one_device(w, kv_cache, kv_scale, qkv, slot_map)
    with on:
        check(lib().gpt2b_kv_cache_write_w4(kv_cache.data_ptr(), kv_scale.data_ptr(), qkv.data_ptr(), slot_map.data_ptr(), rows,
                                            NH, NKV, hs, ld, nb, bs, _stream_on(dev, stream)), w)


def kv_cache_read_w4(out, kv_cache, kv_scale, slot_map, stream=None):
    """Read rows of the paged 4-bit cache back as BF16 [rows, 2, NKV, hs]
    (gpt2b_kv_cache_read_w4); zeros for negative slots."""
    w = "kv_cache_read_w4"
    nb, NKV, bs, hs = _w4_cache(w, kv_cache, kv_scale)
    _need(w, "out", out, torch.bfloat16, 4)
    _need(w, "slot_map", slot_map, torch.int64, 1)
    if tuple(out.shape) != (slot_map.shape[0], 2, NKV, hs):
        _fail(w, "out is [rows, 2, NKV, hs]")
    dev, on = _one_device(w, out, kv_cache, kv_scale, slot_map)
    with on:
        check(lib().gpt2b_kv_cache_read_w4(out.data_ptr(), kv_cache.data_ptr(), kv_scale.data_ptr(), slot_map.data_ptr(),
                                           out.shape[0], NKV, hs, nb, bs, _stream_on(dev, stream)), w)


def attention_paged_w4_workspace(NH, NKV, hs, max_q):
    """Bytes of the workspace of :func:`attention_forward_paged_w4` on the current device."""
    n = ctypes.c_size_t()
    check(lib().gpt2b_attention_paged_w4_workspace(NH, NKV, hs, max_q, ctypes.byref(n)), "attention_paged_w4_workspace")
    return n.value


def attention_forward_paged_w4(out, qkv, kv_cache, kv_scale, block_table, seq_lens, row_start, NH, max_q, workspace,
                               scale=None, stream=None):
    """Attention of packed rows over the paged 4-bit cache, causal among a
    request's rows (gpt2b_attention_forward_paged_w4).  out BF16 [rows, NH hs], qkv
    as for :func:`kv_cache_write_w4`, block_table int32 [B, max_blocks], seq_lens
    [B], row_start [B+1]; ``max_q`` the most rows a request has (a hint);
    ``workspace`` uint8 of :func:`attention_paged_w4_workspace` bytes."""
    w, i32 = "attention_forward_paged_w4", torch.int32
    nb, NKV, bs, hs = _w4_cache(w, kv_cache, kv_scale)
    _need(w, "out", out, torch.bfloat16, 2)
    _need(w, "qkv", qkv, torch.bfloat16, 2, rows=True)
    _need(w, "block_table", block_table, i32, 2)
    _need(w, "seq_lens", seq_lens, i32, 1)
    _need(w, "row_start", row_start, i32, 1)
    _need(w, "workspace", workspace, torch.uint8, 1)
    (rows, width), B = qkv.shape, block_table.shape[0]
    if width < (NH + 2 * NKV) * hs or tuple(out.shape) != (rows, NH * hs):
        _fail(w, "qkv is [rows, >= (NH + 2 NKV) hs] and out [rows, NH hs]")
    if seq_lens.shape[0] != B or row_start.shape[0] != B + 1:
        _fail(w, "seq_lens has B entries and row_start B + 1")
    dev, on = _one_device(w, out, qkv, kv_cache, kv_scale, block_table, seq_lens, row_start, workspace)
    with on:
        check(lib().gpt2b_attention_forward_paged_w4(
            out.data_ptr(), qkv.data_ptr(), kv_cache.data_ptr(), kv_scale.data_ptr(), block_table.data_ptr(),
            seq_lens.data_ptr(), row_start.data_ptr(), B, rows, NH, NKV, hs, _row_pitch(qkv), nb, bs, block_table.shape[1],
            max_q, 1.0 / math.sqrt(hs) if scale is None else scale, workspace.data_ptr(), workspace.shape[0],
            _stream_on(dev, stream)), w)


def _row_pitch(t):
    """Elements between the rows of a 2-d tensor (its width where it has one row: the stride then says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def softmax_probs(probs, logits, temperature=1.0, V=None, stream=None):
    """probs = softmax(logits / temperature) per row over the first ``V`` (default:
    all) columns; temperature 0: one-hot at the largest (gpt2b_softmax_probs).
    FP32 [rows, >= V]; ``probs`` may be ``logits``."""
    w = "softmax_probs"
    _need(w, "probs", probs, torch.float32, 2, rows=True)
    _need(w, "logits", logits, torch.float32, 2, rows=True)
    V = logits.shape[1] if V is None else V
    if probs.shape[0] != logits.shape[0] or min(probs.shape[1], logits.shape[1]) < V:
        _fail(w, "probs and logits have the same rows, of at least V columns")
    dev, on = _one_device(w, probs, logits)
    with on:
        check(lib().gpt2b_softmax_probs(probs.data_ptr(), logits.data_ptr(), logits.shape[0], V, _row_pitch(logits),
                                        _row_pitch(probs), temperature, _stream_on(dev, stream)), w)


def verify_draft_tokens(out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample, stream=None):
    """Accept drafted tokens and draw the next one by rejection sampling from given
    random numbers (gpt2b_verify_draft_tokens).  out_tokens int32 [B, max_out],
    n_accepted [B], tokens int32 [rows] (packed: last token, then drafts),
    target_probs FP32 [rows, V], draft_probs the same or None (certain drafts),
    row_start int32 [B+1], u_accept FP32 [rows], u_sample [B]."""
    w, i32, f32 = "verify_draft_tokens", torch.int32, torch.float32
    _need(w, "out_tokens", out_tokens, i32, 2)
    _need(w, "n_accepted", n_accepted, i32, 1)
    _need(w, "tokens", tokens, i32, 1)
    _need(w, "target_probs", target_probs, f32, 2, rows=True)
    _need(w, "row_start", row_start, i32, 1)
    _need(w, "u_accept", u_accept, f32, 1)
    _need(w, "u_sample", u_sample, f32, 1)
    (B, max_out), (rows, V) = out_tokens.shape, target_probs.shape
    if n_accepted.shape[0] != B or row_start.shape[0] != B + 1 or u_sample.shape[0] != B:
        _fail(w, "n_accepted and u_sample have B entries, row_start B + 1")
    if tokens.shape[0] != rows or u_accept.shape[0] != rows:
        _fail(w, "tokens and u_accept have one entry a row")
    ld_q = V
    if draft_probs is not None:
        _need(w, "draft_probs", draft_probs, f32, 2, rows=True)
        if tuple(draft_probs.shape) != (rows, V):
            _fail(w, "draft_probs has target_probs' shape")
        ld_q = _row_pitch(draft_probs)
    dev, on = _one_device(w, out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample)
    with on:
        check(lib().gpt2b_verify_draft_tokens(out_tokens.data_ptr(), n_accepted.data_ptr(), tokens.data_ptr(),
                                              target_probs.data_ptr(), _p(draft_probs), row_start.data_ptr(),
                                              u_accept.data_ptr(), u_sample.data_ptr(), B, rows, V, _row_pitch(target_probs),
                                              ld_q, max_out, _stream_on(dev, stream)), w)
