// paged_attention.cu -- attention over the paged 4-bit KV cache.
//
// A row i of a request's n rows sees the positions [0, len - n + i]; query head h
// reads key/value head h / (NH/NKV).  Softmax statistics in FP32 (online).
#include "paged_kv.cuh"
#include "internal.h"

#include <float.h>
#include <limits.h>

namespace gpt2b {

GPT2B_DEFINE_ERROR_READER(paged_attention_device_error)

struct PagedAttnArgs {
    __nv_bfloat16* out;
    const __nv_bfloat16* qkv;
    const uint8_t* codes;
    const uint32_t* scales;
    const int *block_table, *seq_lens, *row_start;
    int B, rows, NH, NKV, ld, num_blocks, block_size, max_blocks;
    float scale;
};

constexpr int kPaThreads = 128;

// One CTA per (row, query head): its 4 warps take the positions in turn, a lane
// holds hs/32 channels, and the warps' states are merged at the end.
template <int HS>
__global__ void __launch_bounds__(kPaThreads) paged_attn_kernel(PagedAttnArgs a) {
    constexpr int CH = HS / 32, NG = HS / kW4Group;
    const int row = blockIdx.x / a.NH, head = blockIdx.x % a.NH, kvh = head / (a.NH / a.NKV);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int lo = 0, hi = a.B;  // first request that ends behind the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.row_start[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    if (lo >= a.B || a.row_start[lo] > row) return;
    int len = max(a.seq_lens[lo], 0);
    if (len > a.max_blocks * a.block_size) {
        len = a.max_blocks * a.block_size;
        report_device_error(GPT2B_DEVERR_BAD_POS);
    }
    if (a.row_start[lo + 1] > a.rows) report_device_error(GPT2B_DEVERR_BAD_POS);
    const int n = min(a.row_start[lo + 1], a.rows) - a.row_start[lo];
    const int seen = len - n + (row - a.row_start[lo]) + 1;
    float q[CH], o[CH], m = -FLT_MAX, l = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; k++) {
        q[k] = to_f(a.qkv[(size_t)row * a.ld + head * HS + lane * CH + k]) * a.scale;
        o[k] = 0.0f;
    }
    for (int p = w; p < seen; p += kPaThreads / 32) {
        const int blk = a.block_table[(size_t)lo * a.max_blocks + p / a.block_size];
        if (blk < 0 || blk >= a.num_blocks) {
            report_device_error(GPT2B_DEVERR_BAD_BLOCK);
            continue;
        }
        const size_t kl = (((size_t)blk * 2) * a.NKV + kvh) * a.block_size + p % a.block_size;
        const size_t vl = kl + (size_t)a.NKV * a.block_size;
        const int word = lane * CH / 8, sh = lane * CH % 8, g = lane * CH / kW4Group;
        const uint32_t kw = reinterpret_cast<const uint32_t*>(a.codes + kl * (HS / 2))[word] >> (4 * sh);
        const uint32_t vw = reinterpret_cast<const uint32_t*>(a.codes + vl * (HS / 2))[word] >> (4 * sh);
        const uint32_t km = a.scales[kl * NG + g], vm = a.scales[vl * NG + g];
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; k++) s += q[k] * w4_value(kw, km, k);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), f = __expf(m - mn), e = __expf(s - mn);
        m = mn;
        l = l * f + e;
#pragma unroll
        for (int k = 0; k < CH; k++) o[k] = o[k] * f + e * w4_value(vw, vm, k);
    }
    __shared__ float so[kPaThreads / 32][HS], sm[kPaThreads / 32], sl[kPaThreads / 32];
#pragma unroll
    for (int k = 0; k < CH; k++) so[w][lane * CH + k] = o[k];
    if (lane == 0) { sm[w] = m; sl[w] = l; }
    __syncthreads();
    float M = sm[0];
    for (int k = 1; k < kPaThreads / 32; k++) M = fmaxf(M, sm[k]);
    for (int d = threadIdx.x; d < HS; d += kPaThreads) {
        float num = 0.0f, den = 0.0f;
        for (int k = 0; k < kPaThreads / 32; k++) {
            const float f = __expf(sm[k] - M);
            num += f * so[k][d];
            den += f * sl[k];
        }
        a.out[(size_t)row * a.NH * HS + head * HS + d] = from_f<__nv_bfloat16>(den == 0.0f ? 0.0f : num / den);
    }
}

}  // namespace gpt2b

using namespace gpt2b;

extern "C" {

int gpt2b_attention_paged_w4_workspace(int NH, int NKV, int hs, int max_q, size_t* bytes) {
    if (NH <= 0 || NKV <= 0 || NH % NKV != 0 || max_q <= 0 || !bytes) return GPT2B_ERR_INVALID_ARG;
    if (hs != 64 && hs != 128) return GPT2B_ERR_UNSUPPORTED;
    *bytes = 16;
    return GPT2B_OK;
}

int gpt2b_attention_forward_paged_w4(uint16_t* out, const uint16_t* qkv, const uint8_t* kv_cache, const uint16_t* kv_scale,
                                     const int* block_table, const int* seq_lens, const int* row_start, int B, int rows,
                                     int NH, int NKV, int hs, int ld, int num_blocks, int block_size, int max_blocks,
                                     int max_q, float scale, void* workspace, size_t workspace_bytes,
                                     gpt2b_stream_t stream) {
    if (B <= 0 || rows < 0 || num_blocks <= 0 || block_size <= 0 || max_blocks <= 0 || !kv_cache || !kv_scale ||
        !block_table || !seq_lens || !row_start || !workspace || (rows > 0 && (!out || !qkv)))
        return GPT2B_ERR_INVALID_ARG;
    size_t need = 0;
    int rc = gpt2b_attention_paged_w4_workspace(NH, NKV, hs, max_q, &need);
    if (rc) return rc;
    if (workspace_bytes < need || ((long long)NH + 2ll * NKV) * hs > ld) return GPT2B_ERR_INVALID_ARG;
    if (block_size % kW4Tile != 0 || B > kTableMaxRequests || (long long)max_blocks * block_size > INT_MAX)
        return GPT2B_ERR_UNSUPPORTED;
    if (!aligned16(out) || !aligned16(qkv) || !aligned16(kv_cache) || !aligned16(kv_scale) || !aligned16(workspace) ||
        ld % 8 != 0)
        return GPT2B_ERR_ALIGNMENT;
    if (rows == 0) return GPT2B_OK;
    if ((long long)rows * NH > INT_MAX) return GPT2B_ERR_UNSUPPORTED;
    PagedAttnArgs a{(__nv_bfloat16*)out, (const __nv_bfloat16*)qkv, kv_cache, (const uint32_t*)kv_scale, block_table, seq_lens,
                    row_start, B, rows, NH, NKV, ld, num_blocks, block_size, max_blocks, scale};
    return status_from(hs == 64 ? launch_k(paged_attn_kernel<64>, dim3(rows * NH), dim3(kPaThreads), 0, (cudaStream_t)stream, false, a)
                                : launch_k(paged_attn_kernel<128>, dim3(rows * NH), dim3(kPaThreads), 0, (cudaStream_t)stream, false, a));
}

}  // extern "C"
