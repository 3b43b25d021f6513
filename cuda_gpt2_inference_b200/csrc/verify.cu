// verify.cu -- logits to probabilities, and verification of drafted tokens.
//
// Both work on rows of a vocabulary (50257 logits: 200 KB) of which there are few: one to a
// few hundred.  A row is therefore spread over a cluster of CTAs that exchange their partial
// results through distributed shared memory: one launch, each row read from HBM once (and a second time from L1 or L2
// where a result needs the whole row first), no atomics.
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
__device__ __forceinline__ void cluster_begin() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
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
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// e^(d/T) to about 2 ulp for d <= 0, with c = log2(e)/T as hi + lo: d * c is taken as a rounded product and its
// remainder, so that the error does not grow with |d| as that of a single product does.  d below `least` is
// taken as that (2^-200, which is 0 in FP32): the remainder of -infinity would be NaN.
struct ExpScale {
    float hi, lo, least;
};
static ExpScale exp_scale(float temperature) {
    const double c = 1.4426950408889634 / (double)temperature;
    const float hi = (float)c;
    return {hi, (float)(c - (double)hi), (float)(-200.0 / c)};
}
__device__ __forceinline__ float exp_neg(float d, const ExpScale& c) {
    d = fmaxf(d, c.least);
    const float t = d * c.hi, r = fmaf(d, c.lo, fmaf(d, c.hi, -t));
    return exp2f(t) * fmaf(r, 0.693147181f, 1.0f);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// One CTA of a row's cluster takes a contiguous part of it.  A thread keeps a running maximum and a sum about it,
// a warp joins its threads', and the pairs (m, sum) of all the cluster's warps are exchanged behind its one
// barrier.  Then each thread reads its entries again, from L1 or L2 (unless one batch of loads was all), and writes
// e^((x - M)/T) / total.  Nothing is kept in between, so 6 CTAs of 256 threads fit an SM and their loads, exchanges
// and stores overlap: 320 x 50257 takes 35 us (3.6 TB/s), against 38 with the entries kept in registers (3 CTAs of
// 512 an SM) and 53 with those and the next row's.  HBM, 8 bytes an entry, would take 19.7; what keeps it from that
// is the chain load - exchange - store of each row.  Few rows: 512 threads with all loads in flight at once; there
// launch and chain are all (5 rows: 3.7 us on the device).
struct ProbPart {
    float m, s;
};

template <int U, int T>
__global__ void __launch_bounds__(T, T == 256 ? 6 : 2)
    softmax_probs_kernel(float* probs, const float* logits, int V, long long ld_in, long long ld_out, ExpScale c) {
    __shared__ ProbPart all[8 * (T / 32)];
    cluster_begin();
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int share = (V + C - 1) / C, lo = min(rank * share, V);
    const int left = min(share, V - lo) - (int)threadIdx.x;  // entry k is there while k T < left
    const float* x = logits + (long long)(blockIdx.x / C) * ld_in + lo + threadIdx.x;
    float* out = probs + (long long)(blockIdx.x / C) * ld_out + lo + threadIdx.x;

    pdl_wait();
    // NaN goes through the maximum.  In the sum a single product serves as exponent: its error grows with the
    // distance from the maximum, but the terms fall faster (2^-22 of the sum at a spread of 10; against 64 bits the
    // result is off by 1.1e-7 on 5 rows of 50257, a plain 32-bit form by 0.6e-7).
    float v[U], m = -INFINITY, s = 0.0f;
    for (int i = 0; i < left; i += U * T) {
        float top = m;
#pragma unroll
        for (int k = 0; k < U; k++) v[k] = i + k * T < left ? x[i + k * T] : -INFINITY;
#pragma unroll
        for (int k = 0; k < U; k++) top = max_nan(top, v[k]);
        const float about = top > -INFINITY ? top : 0.0f;
        s *= exp2f((m - about) * c.hi);
#pragma unroll
        for (int k = 0; k < U; k++) s += exp2f((v[k] - about) * c.hi);
        m = top;
    }
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, o));
    s = warp_sum(m > -INFINITY ? s * exp_neg(m - M, c) : 0.0f);
    cluster_wait();
    if (lane < C) *cl.map_shared_rank(&all[rank * (T / 32) + w], lane) = ProbPart{M, s};
    cluster_arrive();
    cluster_wait();
    M = -INFINITY;
    for (int k = lane; k < C * (T / 32); k += 32) M = max_nan(M, all[k].m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, o));
    s = 0.0f;
    for (int k = lane; k < C * (T / 32); k += 32)
        if (all[k].m > -INFINITY) s += all[k].s * exp_neg(all[k].m - M, c);
    s = warp_sum(s);
    // zeros where the row has nothing above -infinity, NaN where it has a NaN or +infinity
    float inv = M > -INFINITY ? __frcp_rn(s) : 0.0f;
    if (!(M < INFINITY)) inv = NAN;
    const float about = M > -INFINITY ? M : 0.0f;
    for (int i = 0; i < left; i += U * T) {
        if (share > U * T) {
#pragma unroll
            for (int k = 0; k < U; k++)
                if (i + k * T < left) v[k] = x[i + k * T];
        }
#pragma unroll
        for (int k = 0; k < U; k++)
            if (i + k * T < left) out[i + k * T] = exp_neg(v[k] - about, c) * inv;
    }
}

// Temperature 0: 1 at the first largest, NaN left out.  320 x 50257: 43 us, 5 rows 3.8 us.
struct FirstMax {
    float m;
    int at;
};
// a > b where the build's fast comparison takes subnormals as 0
__device__ __forceinline__ bool above(float a, float b) {
    int r;
    asm("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %1, %2;\n\tselp.s32 %0, 1, 0, p;\n\t}" : "=r"(r) : "f"(a), "f"(b));
    return r;
}
// whether b comes before a: larger, or as large and earlier (neither is NaN)
__device__ __forceinline__ bool before(FirstMax a, FirstMax b) { return above(b.m, a.m) || (!above(a.m, b.m) && b.at < a.at); }
__device__ __forceinline__ FirstMax first_max(FirstMax a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const FirstMax b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.at, o)};
        if (before(a, b)) a = b;
    }
    return a;
}
constexpr int kProbThreads = 512, kProbWarps = kProbThreads / 32;

__global__ void __launch_bounds__(kProbThreads)
    greedy_probs_kernel(float* probs, const float* logits, int V, long long ld_in, long long ld_out) {
    __shared__ FirstMax all[8 * kProbWarps];
    cluster_begin();
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int share = (V + C - 1) / C, lo = min(rank * share, V), hi = min(lo + share, V);
    const float* x = logits + (long long)(blockIdx.x / C) * ld_in;
    float* out = probs + (long long)(blockIdx.x / C) * ld_out;
    pdl_wait();
    FirstMax a{-INFINITY, INT_MAX};
#pragma unroll 8
    for (int i = lo + tid; i < hi; i += kProbThreads) {
        const float y = x[i];
        if (above(y, a.m)) a = {y, i};
    }
    a = first_max(a);
    cluster_wait();
    if (lane < C) *cl.map_shared_rank(&all[rank * kProbWarps + w], lane) = a;
    cluster_arrive();
    cluster_wait();
    a = {-INFINITY, INT_MAX};
    for (int k = lane; k < C * kProbWarps; k += 32)
        if (before(a, all[k])) a = all[k];
    a = first_max(a);
    for (int i = lo + tid; i < hi; i += kProbThreads) out[i] = i == a.at ? 1.0f : 0.0f;
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

// FP32 to 64 bits with subnormals, which the build's fast arithmetic takes as 0: they are weights like others.
__device__ __forceinline__ double widen(float x) {
    double r;
    asm("cvt.f64.f32 %0, %1;" : "=d"(r) : "f"(x));
    return r;
}

constexpr int kVerThreads = 512, kVerWarps = kVerThreads / 32;

// Weight of token k: 0 unless positive, so NaN counts as nothing.
struct Weights {
    const float *p, *q;
    int drop;
    __device__ __forceinline__ double operator()(int k) const {
        double v = widen(p[k]);
        if (q) v -= widen(q[k]);
        return v > 0.0 && k != drop ? v : 0.0;
    }
};

struct VerPart {
    double sum;
    int last, pad;  // last token of positive weight, -1 without
};

// A cluster of CTAs a request.  Each warp finds the first refused draft for itself (one gathered entry of each
// distribution a draft; a few lanes' work repeated by every warp costs less than a block barrier) and sums the
// weights of its contiguous piece of that one row.  The CTAs' sums are exchanged behind the cluster's one
// barrier; every warp then knows in whose piece the cumulative weight passes u * total, and that warp scans its
// piece again (from L1) and writes the request's results.  64-bit sums: with 32 bits the border of one token in
// 200 of a 50257-token vocabulary would be off by more than a random number's own step.
// Bound by the chain launch - offsets - drafts - row - exchange - scan: 6.7 us for one request of a 50257-token
// vocabulary, 9.9 us for 64, whose two rows each (26 MB) take HBM 4 us.
__global__ void __launch_bounds__(kVerThreads, 2) verify_kernel(VerifyArgs a) {
    __shared__ VerPart all[2][8], seg[kVerWarps];
    cluster_begin();
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int b = blockIdx.x / C, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    pdl_wait();
    const int raw0 = a.row_start[b], raw1 = a.row_start[b + 1];
    const float u = a.u_sample[b];
    const int r0 = min(max(raw0, 0), a.rows), r1 = min(max(raw1, r0), a.rows);
    if (threadIdx.x == 0 && rank == 0 && (r0 != raw0 || r1 != raw1)) report_device_error(GPT2B_DEVERR_BAD_POS);
    int* out = a.out_tokens + (size_t)b * a.max_out;
    if (r0 == r1) {  // the whole cluster leaves
        cluster_wait();
        if (rank == 0 && w == 0) {
            for (int i = lane; i < a.max_out; i += 32) out[i] = -1;
            if (lane == 0) a.n_accepted[b] = 0;
        }
        return;
    }
    const int n = min(r1 - r0 - 1, a.max_out - 1);
    int taken = n, x = -1;  // accepted drafts, and the draft behind them
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane, d = i < n ? a.tokens[r0 + i + 1] : -1;
        bool ok = i >= n;
        if (d >= 0 && d < a.V) {
            const double q = a.q ? widen(a.q[(size_t)(r0 + i) * a.ld_q + d]) : 1.0;
            ok = widen(a.u_accept[r0 + i]) * q < widen(a.p[(size_t)(r0 + i) * a.ld_p + d]);
        }
        const unsigned no = __ballot_sync(0xffffffffu, !ok);
        if (no) {
            taken = i0 + __ffs(no) - 1;
            x = __shfl_sync(0xffffffffu, d, __ffs(no) - 1);
            break;
        }
    }
    const int r = r0 + taken;
    const bool refused = x >= 0 && x < a.V;

    const int share = (a.V + C - 1) / C, end = min((rank + 1) * share, a.V);
    const int piece = (share + kVerWarps - 1) / kVerWarps, lo = min(rank * share + w * piece, end), hi = min(lo + piece, end);
    Weights wt{a.p + (size_t)r * a.ld_p, refused && a.q ? a.q + (size_t)r * a.ld_q : nullptr, refused && !a.q ? x : -1};
    double total = 0.0;
    int done = 0;
    for (int pass = 0; pass < 2; pass++) {
        done = pass;
        constexpr int kAhead = 14;  // loads in flight a lane and distribution
        double sum = 0.0;
        int last = -1;
        for (int k0 = lo + lane; k0 < hi; k0 += 32 * kAhead) {
            float p[kAhead], q[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const bool in = k0 + 32 * j < hi;
                p[j] = in ? wt.p[k0 + 32 * j] : 0.0f;
                q[j] = in && wt.q ? wt.q[k0 + 32 * j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const int k = k0 + 32 * j;
                const double v = widen(p[j]) - widen(q[j]);
                if (v > 0.0 && k != wt.drop) {
                    sum += v;
                    last = k;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) seg[w] = VerPart{sum, last, 0};
        __syncthreads();
        cluster_wait();
        if (threadIdx.x < C) {
            sum = 0.0;
            for (int k = 0; k < kVerWarps; k++) {
                sum += seg[k].sum;
                last = max(last, seg[k].last);
            }
            *cl.map_shared_rank(&all[pass][rank], threadIdx.x) = VerPart{sum, last, 0};
        }
        cluster_arrive();
        cluster_wait();
        total = 0.0;
        for (int k = 0; k < C; k++) total += all[pass][k].sum;
        if (total > 0.0 || !refused) break;
        wt = Weights{wt.p, nullptr, -1};  // nothing left of the target: the target itself
        cluster_begin();
    }
    // The CTA and then the warp in whose part the cumulative weight passes t, the same in every warp.  Where none
    // does (t at or beyond the total, or NaN) the last token of positive weight is drawn, by the first warp.
    const double t = widen(u) * total;
    int cta = -1, owner = -1, last_all = -1;
    double upto = 0.0, run = 0.0;
    for (int k = 0; k < C; k++) {
        if (cta < 0 && upto + all[done][k].sum > t) { cta = k; run = upto; }
        upto += all[done][k].sum;
        last_all = max(last_all, all[done][k].last);
    }
    if (rank != max(cta, 0)) return;
    if (cta >= 0) {
        upto = run;
        for (int k = 0; k < kVerWarps; k++) {
            if (owner < 0 && upto + seg[k].sum > t) { owner = k; run = upto; }
            upto += seg[k].sum;
        }
        if (owner < 0) {
            // the CTA's sum, added in another order, passed t by a rounding: its last warp with weight
            double before = upto = run;
            for (int k = 0; k < kVerWarps; k++) {
                if (seg[k].sum > 0.0) { owner = k; before = upto; }
                upto += seg[k].sum;
            }
            run = before;
        }
    }
    if (w != max(owner, 0)) return;
    int pick = last_all;
    if (owner >= 0) {
        // a contiguous run of entries a lane: their sums, a scan over the lanes, and the run that passes t
        const int each = (hi - lo + 31) / 32, from = min(lo + lane * each, hi), to = min(from + each, hi);
        double sum = 0.0;
#pragma unroll 8
        for (int k = from; k < to; k++) sum += wt(k);
        double c = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += up;
        }
        double before = __shfl_up_sync(0xffffffffu, c, 1);
        if (lane == 0) before = 0.0;
        // a run without weight is passed over, and so is an entry without (unless t is negative): rounding alone
        // never picks one
        const unsigned over = __ballot_sync(0xffffffffu, run + c > t && (sum > 0.0 || t < 0.0));
        const unsigned some = __ballot_sync(0xffffffffu, sum > 0.0);
        const int src = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
        if (src >= 0) {
            // that run's entries, a lane each
            run += __shfl_sync(0xffffffffu, before, src);
            const int begin = __shfl_sync(0xffffffffu, from, src), stop = __shfl_sync(0xffffffffu, to, src);
            int found = -1, last = -1;
            for (int k0 = begin; k0 < stop && found < 0; k0 += 32) {
                const double v = k0 + lane < stop ? wt(k0 + lane) : 0.0;
                double sofar = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, sofar, o);
                    if (lane >= o) sofar += up;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, run + sofar > t && (v > 0.0 || t < 0.0));
                const unsigned any = __ballot_sync(0xffffffffu, v > 0.0);
                if (hit) found = k0 + __ffs(hit) - 1;
                if (any) last = k0 + 31 - __clz(any);
                run += __shfl_sync(0xffffffffu, sofar, 31);
            }
            pick = found >= 0 ? found : last;
        }
    }
    for (int i = lane; i < a.max_out; i += 32) out[i] = i < taken ? a.tokens[r0 + 1 + i] : i == taken ? pick : -1;
    if (lane == 0) a.n_accepted[b] = taken;
}

}  // namespace gpt2b

using namespace gpt2b;

extern "C" {

int gpt2b_softmax_probs(float* probs, const float* logits, int rows, int V, int ld_logits, int ld_probs, float temperature,
                        gpt2b_stream_t stream) {
    if (rows < 0 || V <= 0 || ld_logits < V || ld_probs < V || !(temperature == 0.0f || (temperature >= 1e-30f && temperature <= 1e30f)) ||
        (rows > 0 && (!probs || !logits)))
        return GPT2B_ERR_INVALID_ARG;
    if (rows > 0 && ranges_overlap(probs, ((size_t)(rows - 1) * ld_probs + V) * 4, logits, ((size_t)(rows - 1) * ld_logits + V) * 4)) {
        // the same rows, or columns side by side in one buffer
        const long long apart = ((long long)((intptr_t)probs - (intptr_t)logits) / 4 % ld_probs + ld_probs) % ld_probs;
        const bool beside = apart >= V && apart + V <= ld_probs;
        if (ld_probs != ld_logits || !(probs == logits || beside)) return GPT2B_ERR_INVALID_ARG;
    }
    if (V > 1 << 30) return GPT2B_ERR_UNSUPPORTED;
    if (rows == 0) return GPT2B_OK;
    const int cluster = row_cluster(V, 16 * kProbThreads);
    if ((long long)rows * cluster > INT_MAX) return GPT2B_ERR_UNSUPPORTED;
    const cudaStream_t st = (cudaStream_t)stream;
    const long long li = ld_logits, lo = ld_probs;
    if (temperature == 0.0f)
        return status_from(launch_cluster(greedy_probs_kernel, rows, cluster, kProbThreads, st, probs, logits, V, li, lo));
    const ExpScale c = exp_scale(temperature);
    if ((long long)rows * cluster <= 2ll * sm_count())
        return status_from(launch_cluster(softmax_probs_kernel<16, 512>, rows, cluster, 512, st, probs, logits, V, li, lo, c));
    return status_from(launch_cluster(softmax_probs_kernel<16, 256>, rows, cluster, 256, st, probs, logits, V, li, lo, c));
}

int gpt2b_verify_draft_tokens(int* out_tokens, int* n_accepted, const int* tokens, const float* target_probs,
                              const float* draft_probs, const int* row_start, const float* u_accept, const float* u_sample,
                              int B, int rows, int V, int ld_target, int ld_draft, int max_out, gpt2b_stream_t stream) {
    if (B <= 0 || rows < 0 || V <= 0 || ld_target < V || max_out <= 0 || !out_tokens || !n_accepted || !row_start || !u_sample)
        return GPT2B_ERR_INVALID_ARG;
    if (rows > 0 && (!tokens || !target_probs || !u_accept)) return GPT2B_ERR_INVALID_ARG;
    if (draft_probs && ld_draft < V) return GPT2B_ERR_INVALID_ARG;
    // a request's results may be written before another's inputs are read
    const size_t b4 = 4 * (size_t)B, r4 = 4 * (size_t)rows;
    auto row_bytes = [&](int ld) { return rows > 0 ? 4 * ((size_t)(rows - 1) * ld + V) : 0; };
    if (outputs_overlap({{out_tokens, b4 * max_out}, {n_accepted, b4}},
                        {{tokens, r4}, {target_probs, row_bytes(ld_target)}, {draft_probs, row_bytes(ld_draft)},
                         {row_start, b4 + 4}, {u_accept, r4}, {u_sample, b4}}))
        return GPT2B_ERR_INVALID_ARG;
    if (V > 1 << 30) return GPT2B_ERR_UNSUPPORTED;
    VerifyArgs a{out_tokens, n_accepted, tokens, target_probs, draft_probs, row_start, u_accept, u_sample,
                 B, rows, V, ld_target, ld_draft, max_out};
    // up to 8 CTAs a request, fewer where the requests fill the SMs (2 CTAs each) in one wave without
    int c = row_cluster(V, 8 * kVerThreads);
    while (c > 1 && (long long)B * c > 2ll * sm_count()) c /= 2;
    if ((long long)B * c > INT_MAX) return GPT2B_ERR_UNSUPPORTED;
    return status_from(launch_cluster(verify_kernel, B, c, kVerThreads, (cudaStream_t)stream, a));
}

}  // extern "C"
