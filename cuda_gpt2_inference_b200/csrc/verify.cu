// verify.cu -- logits to probabilities, and verification of drafted tokens.
//
// Both work on rows of a vocabulary (50257 logits: 200 KB) of which there are few: one to a
// few hundred.  A row is therefore spread over a cluster of CTAs that exchange their partial
// results through distributed shared memory: one launch, each row read once, no atomics.
#include "common.cuh"
#include "internal.h"

#include <cooperative_groups.h>
#include <float.h>
#include <limits.h>

namespace cg = cooperative_groups;

namespace gpt2b {

GPT2B_DEFINE_ERROR_READER(verify_device_error)

// The exchange: arrive at the start, wait before the first store to another CTA (which has then begun), store
// the own part into every CTA, arrive and wait again; afterwards each CTA reads its own shared memory only and
// may leave.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// CTAs of a row: a power of two up to 8 (the portable cluster size), so that each takes about `share` entries.
static int row_cluster(int V, int share) {
    int c = 1;
    while (c < 8 && (long long)c * share < V) c *= 2;
    return c;
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_cluster(void (*kernel)(KArgs...), unsigned rows, unsigned cluster, unsigned threads, cudaStream_t st,
                                  Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * cluster);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// e^x to about 2 ulp for x <= 0: x log2(e) is split into a rounded product and its
// remainder, so that the error does not grow with |x| as that of a single product does.
__device__ __forceinline__ float exp_neg(float x) {
    x = fmaxf(x, -200.0f);  // e^-200 is 0 in FP32; keeps the remainder of -infinity from being NaN
    const float t = x * 1.4426950408889634f;
    const float r = fmaf(x, 1.4426950408889634f, -t) + x * 1.92596299e-8f;  // log2(e) - fp32(log2(e))
    return exp2f(t) * fmaf(r, 0.693147181f, 1.0f);
}

// One CTA of a row's cluster takes a contiguous part of it, R entries a thread in registers (entries beyond
// cluster * 512 * R are read twice more).  Each CTA sums e^(x - m) about its own maximum m; the pairs
// (m, sum) are exchanged once, and what a CTA wrote off about m is put right by one factor, e^(m - M) / total.
// 320 x 50257: 8 bytes an entry from and to HBM bound it; 5 rows: the chain launch - load - exchange - store.
constexpr int kProbThreads = 512;

struct ProbPart {
    float m, s;
    int at, nan;
};

template <int R>
__global__ void __launch_bounds__(kProbThreads, R == 4 ? 4 : R == 16 ? 3 : 2)
    softmax_probs_kernel(float* probs, const float* logits, int V, long long ld_in, long long ld_out, float temperature) {
    __shared__ ProbPart parts[kProbThreads / 32], all[8];
    cluster_arrive();
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const long long row = blockIdx.x / C;
    const int share = (V + C - 1) / C, lo = min(rank * share, V), n = min(share, V - lo);
    const float* x = logits + row * ld_in + lo;
    float* out = probs + row * ld_out + lo;

    float v[R], m = -INFINITY;
    int at = INT_MAX;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int i = tid + k * kProbThreads;
        v[k] = i < n ? x[i] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < R; k++) {
        if (v[k] > m) { m = v[k]; at = lo + tid + k * kProbThreads; }
        nan = nan || v[k] != v[k];
    }
    for (int i = tid + R * kProbThreads; i < n; i += kProbThreads) {
        const float y = x[i];
        if (y > m) { m = y; at = lo + i; }
        nan = nan || y != y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > m || (om == m && oa < at)) { m = om; at = oa; }
    }
    nan = __any_sync(0xffffffffu, nan);
    if (lane == 0) parts[w] = ProbPart{m, 0.0f, at, nan};
    __syncthreads();
    for (int k = 0; k < kProbThreads / 32; k++) {
        const ProbPart p = parts[k];
        if (p.m > m || (p.m == m && p.at < at)) { m = p.m; at = p.at; }
        nan = nan || p.nan;
    }
    const bool greedy = temperature == 0.0f;
    const float inv = greedy ? 1.0f : __frcp_rn(temperature);
    float s = 0.0f;
    if (!greedy && m > -INFINITY) {
#pragma unroll
        for (int k = 0; k < R; k++) {
            v[k] = exp_neg((v[k] - m) * inv);
            if (tid + k * kProbThreads < n) s += v[k];
        }
        for (int i = tid + R * kProbThreads; i < n; i += kProbThreads) s += exp_neg((x[i] - m) * inv);
    }
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) parts[w].s = s;
    __syncthreads();
    cluster_wait();
    if (tid < C) {
        s = 0.0f;
        for (int k = 0; k < kProbThreads / 32; k++) s += parts[k].s;
        *cl.map_shared_rank(&all[rank], tid) = ProbPart{m, s, at, nan || m == INFINITY};
    }
    cluster_arrive();
    cluster_wait();
    ProbPart p{-INFINITY, 0.0f, INT_MAX, 0};
    if (lane < C) p = all[lane];
    float M = p.m;
    int best = p.at;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, M, o);
        const int oa = __shfl_xor_sync(0xffffffffu, best, o);
        if (om > M || (om == M && oa < best)) { M = om; best = oa; }
    }
    M = __shfl_sync(0xffffffffu, M, 0);
    best = __shfl_sync(0xffffffffu, best, 0);
    if (greedy) {
        for (int i = tid; i < n; i += kProbThreads) out[i] = lo + i == best ? 1.0f : 0.0f;
        return;
    }
    const bool any = __any_sync(0xffffffffu, p.nan);
    // this CTA's factor; 0 where the row (or its part) has nothing above -infinity
    const float total = warp_sum(p.m > -INFINITY ? p.s * exp_neg((p.m - M) * inv) : 0.0f);
    float f = m > -INFINITY ? __fdiv_rn(exp_neg((m - M) * inv), total) : 0.0f;
    if (any) f = NAN;
    if (!(m > -INFINITY)) {
#pragma unroll
        for (int k = 0; k < R; k++) v[k] = 0.0f;  // f is 0 or NaN
    }
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int i = tid + k * kProbThreads;
        if (i < n) out[i] = v[k] * f;
    }
    for (int i = tid + R * kProbThreads; i < n; i += kProbThreads)
        out[i] = m > -INFINITY ? exp_neg((x[i] - m) * inv) * f : f;
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

constexpr int kVerThreads = 512, kVerWarps = kVerThreads / 32;

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

struct VerPart {
    double sum;
    int last;  // last token of positive weight, -1 without
};

// A cluster of CTAs a request.  Each CTA finds the first refused draft for itself (one gathered entry of
// each distribution a draft) and then sums the weights of its part of that one row, a warp a contiguous
// piece; the sums are exchanged, and in the CTA in whose part the cumulative weight passes u * total the warp
// in whose piece it does scans that piece again, and the CTA writes the request's results.  64-bit sums: with 32 bits the border of one token in 200 of a 50257-token vocabulary
// would be off by more than a random number's own step.
__global__ void __launch_bounds__(kVerThreads) verify_kernel(VerifyArgs a) {
    __shared__ double seg[kVerWarps];
    __shared__ int s_first, s_last, s_pick;
    __shared__ VerPart all[2][8];
    cluster_arrive();
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int raw0 = a.row_start[b], raw1 = a.row_start[b + 1];
    const int r0 = min(max(raw0, 0), a.rows), r1 = min(max(raw1, r0), a.rows);
    if (tid == 0 && rank == 0 && (r0 != raw0 || r1 != raw1)) report_device_error(GPT2B_DEVERR_BAD_POS);
    int* out = a.out_tokens + (size_t)b * a.max_out;
    if (r0 == r1) {  // the whole cluster leaves
        cluster_wait();
        if (rank == 0) {
            for (int i = tid; i < a.max_out; i += kVerThreads) out[i] = -1;
            if (tid == 0) a.n_accepted[b] = 0;
        }
        return;
    }
    const float u = a.u_sample[b];
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

    const int share = (a.V + C - 1) / C, end = min((rank + 1) * share, a.V);
    const int piece = (share + kVerWarps - 1) / kVerWarps, lo = min(rank * share + w * piece, end), hi = min(lo + piece, end);
    Weights wt{a.p + (size_t)r * a.ld_p, refused && a.q ? a.q + (size_t)r * a.ld_q : nullptr, refused && !a.q ? x : -1};
    double total = 0.0;
    int last_all = -1, done = 0;
    for (int pass = 0; pass < 2; pass++) {
        done = pass;
        double s = 0.0;
        int last = -1;
#pragma unroll 8
        for (int k = lo + lane; k < hi; k += 32) {
            const double v = wt(k);
            s += v;
            if (v > 0.0) last = k;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) {
            seg[w] = s;
            if (last >= 0) atomicMax(&s_last, last);
        }
        __syncthreads();
        cluster_wait();
        if (tid < C) {
            s = 0.0;
            for (int k = 0; k < kVerWarps; k++) s += seg[k];
            *cl.map_shared_rank(&all[pass][rank], tid) = VerPart{s, s_last};
        }
        cluster_arrive();
        cluster_wait();
        last_all = -1;
        total = 0.0;
        for (int k = 0; k < C; k++) {
            total += all[pass][k].sum;
            last_all = max(last_all, all[pass][k].last);
        }
        if (total > 0.0 || !refused) break;
        wt = Weights{wt.p, nullptr, -1};  // nothing left of the target: the target itself
        cluster_arrive();
    }
    // the CTA in whose part the cumulative weight passes t, the same in every CTA; none (t at or beyond the
    // total, or NaN): the first CTA writes the last token of positive weight
    const double t = (double)u * total;
    int owner = -1;
    double upto = 0.0, before = 0.0;
    for (int k = 0; k < C && owner < 0; k++) {
        before = upto;
        upto += all[done][k].sum;
        if (upto > t) owner = k;
    }
    if (rank != max(owner, 0)) return;
    double run = before;
    for (int k = 0; k < w; k++) run += seg[k];
    if (owner >= 0 && run + seg[w] > t) {  // candidates of later pieces lose in the minimum
        constexpr int kAhead = 8;  // 32-entry rows whose loads are in flight together
        bool found = false;
        for (int base = lo; base < hi && !found; base += 32 * kAhead) {
            double v[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) v[j] = base + 32 * j + lane < hi ? wt(base + 32 * j + lane) : 0.0;
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                if (found) break;
                double c = v[j];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, c, o);
                    if (lane >= o) c += up;
                }
                // rounding alone never picks a token without weight
                const unsigned over = __ballot_sync(0xffffffffu, run + c > t && (v[j] > 0.0 || t < 0.0));
                if (over) {
                    if (lane == 0) atomicMin(&s_pick, base + 32 * j + __ffs(over) - 1);
                    found = true;
                }
                run += __shfl_sync(0xffffffffu, c, 31);
            }
        }
    }
    __syncthreads();
    // rounding can leave the scan of the owner's part without a token: its last one then
    const int pick = s_pick < a.V ? s_pick : owner >= 0 && all[done][rank].last >= 0 ? all[done][rank].last : last_all;
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
    if (V > 1 << 30) return GPT2B_ERR_UNSUPPORTED;
    if (rows == 0) return GPT2B_OK;
    const int c = row_cluster(V, 16 * kProbThreads);
    if ((long long)rows * c > INT_MAX) return GPT2B_ERR_UNSUPPORTED;
    const int each = ((V + c - 1) / c + kProbThreads - 1) / kProbThreads;  // entries a thread
    const cudaStream_t st = (cudaStream_t)stream;
    const long long li = ld_logits, lo = ld_probs;
    if (each <= 4) return status_from(launch_cluster(softmax_probs_kernel<4>, rows, c, kProbThreads, st, probs, logits, V, li, lo, temperature));
    if (each <= 16) return status_from(launch_cluster(softmax_probs_kernel<16>, rows, c, kProbThreads, st, probs, logits, V, li, lo, temperature));
    return status_from(launch_cluster(softmax_probs_kernel<32>, rows, c, kProbThreads, st, probs, logits, V, li, lo, temperature));
}

int gpt2b_verify_draft_tokens(int* out_tokens, int* n_accepted, const int* tokens, const float* target_probs,
                              const float* draft_probs, const int* row_start, const float* u_accept, const float* u_sample,
                              int B, int rows, int V, int ld_target, int ld_draft, int max_out, gpt2b_stream_t stream) {
    if (B <= 0 || rows < 0 || V <= 0 || ld_target < V || max_out <= 0 || !out_tokens || !n_accepted || !row_start || !u_sample)
        return GPT2B_ERR_INVALID_ARG;
    if (rows > 0 && (!tokens || !target_probs || !u_accept)) return GPT2B_ERR_INVALID_ARG;
    if (draft_probs && ld_draft < V) return GPT2B_ERR_INVALID_ARG;
    if (V > 1 << 30) return GPT2B_ERR_UNSUPPORTED;
    VerifyArgs a{out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample,
                 B, rows, V, ld_target, ld_draft, max_out};
    // up to 8 CTAs a request, fewer where the requests alone fill the SMs (4 CTAs each)
    int c = row_cluster(V, 8 * kVerThreads);
    while (c > 1 && (long long)B * c > 4ll * sm_count()) c /= 2;
    if ((long long)B * c > INT_MAX) return GPT2B_ERR_UNSUPPORTED;
    return status_from(launch_cluster(verify_kernel, B, c, kVerThreads, (cudaStream_t)stream, a));
}

}  // extern "C"
