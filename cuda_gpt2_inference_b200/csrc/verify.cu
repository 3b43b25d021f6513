// verify.cu -- logits to probabilities, and verification of drafted tokens.
#include "common.cuh"
#include "internal.h"

#include <float.h>
#include <limits.h>

namespace gpt2b {

GPT2B_DEFINE_ERROR_READER(verify_device_error)

// e^x to about 2 ulp for x <= 0: x log2(e) is split into a rounded product and its
// remainder, so that the error does not grow with |x| as that of a single product does.
__device__ __forceinline__ float exp_neg(float x) {
    x = fmaxf(x, -200.0f);  // e^-200 is 0 in FP32; keeps the remainder of -infinity from being NaN
    const float t = x * 1.4426950408889634f;
    const float r = fmaf(x, 1.4426950408889634f, -t) + x * 1.92596299e-8f;  // log2(e) - fp32(log2(e))
    return exp2f(t) * fmaf(r, 0.693147181f, 1.0f);
}

constexpr int kProbThreads = 1024;

__global__ void __launch_bounds__(kProbThreads)
    softmax_probs_kernel(float* probs, const float* logits, int V, int ld_in, int ld_out, float temperature) {
    __shared__ float sv[32];
    __shared__ int si[32];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const float* row = logits + (size_t)blockIdx.x * ld_in;
    float* out = probs + (size_t)blockIdx.x * ld_out;
    float mx = -INFINITY;
    int at = INT_MAX;
    for (int i = tid; i < V; i += kProbThreads) {
        const float v = row[i];
        if (v > mx) { mx = v; at = i; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, mx, o);
        const int oi = __shfl_xor_sync(0xffffffffu, at, o);
        if (ov > mx || (ov == mx && oi < at)) { mx = ov; at = oi; }
    }
    if (lane == 0) { sv[w] = mx; si[w] = at; }
    __syncthreads();
    for (int k = 0; k < 32; k++)
        if (sv[k] > mx || (sv[k] == mx && si[k] < at)) { mx = sv[k]; at = si[k]; }
    __syncthreads();
    if (temperature == 0.0f) {
        for (int i = tid; i < V; i += kProbThreads) out[i] = i == at ? 1.0f : 0.0f;
        return;
    }
    const float inv = __frcp_rn(temperature);
    bool nan = mx == INFINITY;
    float s = 0.0f;
    for (int i = tid; i < V; i += kProbThreads) {
        const float v = row[i];
        nan = nan || v != v;
        if (mx > -INFINITY) s += exp_neg((v - mx) * inv);
    }
    nan = __syncthreads_or(nan);
    s = block_sum(s, sv);
    for (int i = tid; i < V; i += kProbThreads) {
        float p = 0.0f;
        if (mx > -INFINITY) p = __fdiv_rn(exp_neg((row[i] - mx) * inv), s);
        out[i] = nan ? NAN : p;
    }
}

// ---------------------------------------------------------------------------
// verification
// ---------------------------------------------------------------------------
struct VerifyArgs {
    int *out_tokens, *n_accepted;
    const int* tokens;
    const float *p, *q;
    const int* row_start;
    const float *u_accept, *u_sample;
    int B, rows, V, ld_p, ld_q, max_out;
};

constexpr int kVerThreads = 1024;

// Weight of token k: 0 unless positive, so NaN counts as nothing.
struct Weights {
    const float *p, *q;
    int drop;
    __device__ __forceinline__ double operator()(int k) const {
        double v = (double)p[k];
        if (q) v -= (double)q[k];
        return v > 0.0 && k != drop ? v : 0.0;
    }
};

__global__ void __launch_bounds__(kVerThreads) verify_kernel(VerifyArgs a) {
    __shared__ int s_first, s_last, s_pick;
    __shared__ double seg[kVerThreads / 32];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int raw0 = a.row_start[b], raw1 = a.row_start[b + 1];
    const int r0 = min(max(raw0, 0), a.rows), r1 = min(max(raw1, r0), a.rows);
    if (tid == 0 && (r0 != raw0 || r1 != raw1)) report_device_error(GPT2B_DEVERR_BAD_POS);
    int* out = a.out_tokens + (size_t)b * a.max_out;
    if (r0 == r1) {
        for (int i = tid; i < a.max_out; i += kVerThreads) out[i] = -1;
        if (tid == 0) a.n_accepted[b] = 0;
        return;
    }
    const int n = min(r1 - r0 - 1, a.max_out - 1);
    if (tid == 0) { s_first = n; s_last = -1; s_pick = INT_MAX; }
    __syncthreads();
    for (int i = tid; i < n; i += kVerThreads) {
        const int x = a.tokens[r0 + i + 1];
        bool ok = x >= 0 && x < a.V;
        if (ok) {
            const double q = a.q ? (double)a.q[(size_t)(r0 + i) * a.ld_q + x] : 1.0;
            ok = (double)a.u_accept[r0 + i] * q < (double)a.p[(size_t)(r0 + i) * a.ld_p + x];
        }
        if (!ok) atomicMin(&s_first, i);
    }
    __syncthreads();
    const int taken = s_first, r = r0 + taken;
    const int x = taken < n ? a.tokens[r + 1] : -1;
    const bool refused = x >= 0 && x < a.V;
    const int chunk = (a.V + kVerThreads / 32 - 1) / (kVerThreads / 32);
    const int lo = min(w * chunk, a.V), hi = min(lo + chunk, a.V);
    Weights wt{a.p + (size_t)r * a.ld_p, refused && a.q ? a.q + (size_t)r * a.ld_q : nullptr, refused && !a.q ? x : -1};
    double total = 0.0;
    for (int pass = 0; pass < 2; pass++) {
        double s = 0.0;
        int last = -1;
        for (int k = lo + lane; k < hi; k += 32) {
            const double v = wt(k);
            s += v;
            if (v > 0.0) last = k;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) seg[w] = s;
        if (last >= 0) atomicMax(&s_last, last);
        __syncthreads();
        total = 0.0;
        for (int k = 0; k < kVerThreads / 32; k++) total += seg[k];
        if (total > 0.0 || !refused) break;
        wt = Weights{wt.p, nullptr, -1};  // nothing left of the target: the target itself
        __syncthreads();
    }
    const double t = (double)a.u_sample[b] * total;
    double run = 0.0;
    for (int k = 0; k < w; k++) run += seg[k];
    if (run + seg[w] > t) {  // candidates of later warps lose in the minimum
        for (int base = lo; base < hi; base += 32) {
            const int k = base + lane;
            double v = k < hi ? wt(k) : 0.0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += up;
            }
            const unsigned over = __ballot_sync(0xffffffffu, run + v > t);
            if (over) {
                if (lane == 0) atomicMin(&s_pick, base + __ffs(over) - 1);
                break;
            }
            run += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    const int pick = s_pick < a.V ? s_pick : s_last;
    for (int i = tid; i < a.max_out; i += kVerThreads)
        out[i] = i < taken ? a.tokens[r0 + 1 + i] : i == taken ? pick : -1;
    if (tid == 0) a.n_accepted[b] = taken;
}

}  // namespace gpt2b

using namespace gpt2b;

extern "C" {

int gpt2b_softmax_probs(float* probs, const float* logits, int rows, int V, int ld_logits, int ld_probs, float temperature,
                        gpt2b_stream_t stream) {
    if (rows < 0 || V <= 0 || ld_logits < V || ld_probs < V || !(temperature == 0.0f || (temperature >= 1e-30f && temperature <= FLT_MAX)) ||
        (rows > 0 && (!probs || !logits)))
        return GPT2B_ERR_INVALID_ARG;
    if (probs == logits && ld_logits != ld_probs) return GPT2B_ERR_INVALID_ARG;
    if (rows == 0) return GPT2B_OK;
    return status_from(launch_k(softmax_probs_kernel, dim3(rows), dim3(kProbThreads), 0, (cudaStream_t)stream, false, probs,
                                logits, V, ld_logits, ld_probs, temperature));
}

int gpt2b_verify_draft_tokens(int* out_tokens, int* n_accepted, const int* tokens, const float* target_probs,
                              const float* draft_probs, const int* row_start, const float* u_accept, const float* u_sample,
                              int B, int rows, int V, int ld_target, int ld_draft, int max_out, gpt2b_stream_t stream) {
    if (B <= 0 || rows < 0 || V <= 0 || ld_target < V || max_out <= 0 || !out_tokens || !n_accepted || !row_start || !u_sample)
        return GPT2B_ERR_INVALID_ARG;
    if (rows > 0 && (!tokens || !target_probs || !u_accept)) return GPT2B_ERR_INVALID_ARG;
    if (draft_probs && ld_draft < V) return GPT2B_ERR_INVALID_ARG;
    VerifyArgs a{out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample,
                 B, rows, V, ld_target, ld_draft, max_out};
    return status_from(launch_k(verify_kernel, dim3(B), dim3(kVerThreads), 0, (cudaStream_t)stream, false, a));
}

}  // extern "C"
