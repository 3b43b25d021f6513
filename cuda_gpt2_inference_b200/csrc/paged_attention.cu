// paged_attention.cu -- attention over the paged 4-bit KV cache.
//
// A row i of a request's n rows sees the positions [0, len - n + i]; query head h
// reads key/value head h / (NH/NKV).  The (row, head) pairs that share a key/value
// head are the columns of one tile, so its codes are read and decoded once for all
// of them:
//   S[pos][col] = s_pos (codes_K[pos] . q[col]) + lo_pos sum(q[col])
//   out[ch][col] = sum_pos codes_V[pos][ch] (P[pos][col] s_pos) + sum_pos P lo_pos
// Step and low end are factors of a whole position, so the products take the codes
// themselves (0..15) as FP16 operands of mma.sync m16n8k16, positions (K) or
// channels (V) in its 16 rows, 8 columns in its N.
//
// Codes as FP16.  A nibble masked in place in bits 0..3 or 4..7 of a 16-bit half is
// the FP16 subnormal code * 2^-24 or code * 2^-20: one AND a pair, no conversion and
// no offset to take off again (0.6 instructions a code).  The tensor cores multiply
// subnormals exactly; the powers of two are put right in q (K: even nibbles carry a
// factor of 16) and in the final scaling (V).
//
// Why mma.sync and not tcgen05: an operand of tcgen05.mma has 64 rows or more and
// lies in shared or tensor memory, so every decoded code would be written and read
// there again; here a tile has 1..16 columns, and the codes go from a register to
// the tensor core that multiplies them.
//
// What bounds it: the latency of a warp's own arithmetic.  A step of 32 positions of 128
// channels takes a warp about 540 instructions, half of them on the ALU pipe (decode, steps,
// maxima).  Registers leave 3 warps a scheduler with 8 columns and 2 with 16, which issue in
// 55 and 52 % of the cycles and wait longest for results of their own instructions; nothing is
// full (ALU 54 and 42 %, tensor pipe 26 and 39 %).  Measured, of the 6.54 TB/s of a copy:
// 32 x 16384 positions of 8 heads of 128, one row of 4 query heads each: 125 us, 74 %; 4 rows,
// 16 columns: 175 us, 53 %; 32 x 8192 of 25 heads of 64, one row: 105 us, 69 %.  One request of
// 1001 positions and 12 heads: 6 us, a chain of launch, lengths, table, codes, join.
//
// Weights times V's steps are the products' other operand, in FP16: 2^-11 of each, where BF16 would
// be 2^-8 and FP32 operands have no such product.  Against 64 bits the result is off by 1.71e-3 to
// 1.77e-3 (root mean square, relative), a 32-bit form rounded once to BF16 by 1.66e-3 to 1.68e-3.
#include "paged_kv.cuh"
#include "internal.h"

#include <float.h>
#include <limits.h>

#include <type_traits>

namespace gpt2b {

GPT2B_DEFINE_ERROR_READER(paged_attention_device_error)

struct PagedAttnArgs {
    __nv_bfloat16* out;
    const __nv_bfloat16* qkv;
    const uint8_t* codes;
    const uint32_t* scales;
    const int *block_table, *seq_lens, *row_start;
    int B, rows, NH, NKV, ld, num_blocks, block_size, max_blocks;
    int unit_blocks, unit_rest;  // kPaUnit in whole blocks and positions
    float scale_log2;       // softmax scale * log2(e)
    float* ws;
};

constexpr int kPaWarps = 4, kPaThreads = 32 * kPaWarps;
constexpr int kPaStep = 32;                  // positions a warp takes at a time
constexpr int kPaUnit = kPaStep * kPaWarps;  // positions of a unit of the work partition
constexpr int kPaExtra = 2;                  // what a segment costs beside its units, in units
// Weights are 2^(score - running maximum - kBias): their sums, up to 2^8 a position, then reach 2^24 positions before
// a product with a value of FP32's whole range overflows, and a weight underflows only 2^-100 below the largest.
constexpr float kBias = 24.0f;

// NG groups of 64 channels, NT tiles of 8 columns.
template <int NG, int NT> struct PaShape {
    static constexpr int kHS = NG * kW4Group, kCols = 8 * NT;
    static constexpr int kStages = NG == 1 ? 3 : 2;  // steps in flight a warp
    static constexpr int kCodeBytes = kPaStep * 32 * NG, kMetaBytes = kPaStep * 4 * NG;
    static constexpr int kStageBytes = 2 * (kCodeBytes + kMetaBytes);
    static constexpr int kRing = kPaWarps * kStages * kStageBytes;
    static constexpr int kPitch = kHS + 1;  // floats between the columns of a warp's slab
    static constexpr int kMerge = (kPaWarps * kCols * kPitch + 2 * kPaWarps * kCols) * 4;
    static constexpr int kJoin = ((kRing > kMerge ? kRing : kMerge) + 15) & ~15;
    // query fragments: in registers, or where those run out in shared memory, one copy for all warps
    static constexpr bool kQShared = NG * NT >= 4;
    static constexpr int kQBytes = kQShared ? NT * NG * 4 * 32 * 8 : 0;
    static constexpr int kSmem = kJoin + kQBytes;
    // Resident CTAs an SM.  More registers a thread (more products in flight) beat more warps: hs 128 with 8
    // columns (32 x 16384 positions) 3 CTAs 131 us, 4 139; hs 64 with 16 columns 3 CTAs 157, 4 172; hs 128 with 16
    // columns 2 CTAs 183, 3 191; hs 64 with 8 columns the same for long requests, and 4 better for short ones
    // (18.5 against 19.4 us at 16 x 1024).
    static constexpr int kCtas = NG * NT == 1 ? 4 : NG * NT == 2 ? 3 : 2;
    static constexpr int kSlot = kCols * (kHS + 2);                 // floats of a partial result
    // Scores and low ends two columns an instruction (us at the sizes above): hs 128 with 8 columns 129 -> 125,
    // hs 64 with 16 columns 153 -> 150, with 8 the same; hs 128 with 16 columns 174 -> 183, so not there.
    static constexpr bool kPacked = NG * NT <= 2;
};

// ---------------------------------------------------------------------------
// work partition
// ---------------------------------------------------------------------------
// A segment is a (request, key/value head, tile of columns); it has ceil(len/128)
// units, and before them kPaExtra that stand for what it takes to begin and to end one.
// The units of all segments are numbered in one row and dealt out in equal contiguous
// runs to the resident CTAs, whatever the lengths are: a long request is split over
// many CTAs, short ones share one.  A CTA writes a finished segment to `out`, and the
// piece of a segment that it shares with its neighbours to one of its two slots (0: the
// segment began before its run, 1: it goes on behind it).
struct PaRequest {
    int r0, n, len, chunks, units;  // units with the extra ones
};
__device__ __forceinline__ PaRequest pa_request(const PagedAttnArgs& a, int b, int cols, bool report) {
    PaRequest r;
    const int s0 = a.row_start[b], s1 = a.row_start[b + 1], l0 = a.seq_lens[b];
    r.r0 = min(max(s0, 0), a.rows);
    const int r1 = min(max(s1, r.r0), a.rows);
    r.n = r1 - r.r0;
    r.len = min(max(l0, 0), a.max_blocks * a.block_size);
    if (report && (r.r0 != s0 || r1 != s1 || l0 > r.len)) report_device_error(GPT2B_DEVERR_BAD_POS);
    r.chunks = (r.n * (a.NH / a.NKV) + cols - 1) / cols;
    r.units = kPaExtra + max(1, (r.len + kPaUnit - 1) / kPaUnit);  // a request that sees nothing still gets its zeros
    return r;
}

// head, tile of columns and unit of the v-th unit of a request; 32-bit divisions where they do
struct PaPlace {
    int kvh, chunk, unit;
};
__device__ __forceinline__ PaPlace pa_place(const PaRequest& r, long long v) {
    const long long per_head = (long long)r.chunks * r.units;
    if ((v | per_head) >> 32) {
        const long long in = v % per_head;
        return {(int)(v / per_head), (int)(in / r.units), (int)(in % r.units)};
    }
    const unsigned q = (unsigned)v / (unsigned)per_head, in = (unsigned)v - q * (unsigned)per_head;
    const unsigned c = in / (unsigned)r.units;
    return {(int)q, (int)c, (int)(in - c * (unsigned)r.units)};
}

// pre[b] = units of the requests before b, pre[B] = all; every thread of the CTA calls it.
__device__ __forceinline__ void pa_scan(const PagedAttnArgs& a, int cols, long long* pre, long long* wsum, bool report) {
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    long long base = 0;
    if (tid == 0) pre[0] = 0;
    for (int b0 = 0; b0 < a.B; b0 += kPaThreads) {
        const int b = b0 + tid;
        long long v = 0;
        if (b < a.B) {
            const PaRequest r = pa_request(a, b, cols, report);
            v = (long long)a.NKV * r.chunks * r.units;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) wsum[w] = v;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int k = 0; k < kPaWarps; k++) {
            if (k < w) v += wsum[k];
            all += wsum[k];
        }
        if (b < a.B) pre[b + 1] = base + v;
        base += all;
        __syncthreads();
    }
}
// where the run of CTA i of G begins: total * i / G, in 32 bits where that does (a 64-bit division takes longer than
// the loads around it)
__device__ __forceinline__ long long pa_run(long long total, int i, int G) {
    return total < (1 << 20) && G < 4096 ? (long long)((unsigned)total * (unsigned)i / (unsigned)G) : total * i / G;
}
// the request that holds unit u
__device__ __forceinline__ int pa_find(const long long* pre, int B, long long u) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid + 1] > u) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// ---------------------------------------------------------------------------
// PTX
// ---------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t mov_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
// two FP32 operations an instruction
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.ftz.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1) {
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "add.rn.ftz.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(a0), "f"(a1));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
// step and low end of each group of a position
template <int NG> __device__ __forceinline__ void lds_meta(uint32_t addr, uint32_t* meta) {
    if constexpr (NG == 1) {
        meta[0] = lds32(addr);
    } else {
        const uint2 v = lds64(addr);
        meta[0] = v.x;
        meta[1] = v.y;
    }
}
__device__ __forceinline__ float meta_step(uint32_t m) { return __uint_as_float(m << 16); }
__device__ __forceinline__ float meta_low(uint32_t m) { return __uint_as_float(m & 0xffff0000u); }
__device__ __forceinline__ float pow2_field(int field) { return __uint_as_float((uint32_t)field << 23); }

__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;  // nibbles as code * 2^-24 / code * 2^-20

// Tile row r of 8 holds the position r ^ (r >> 2): then the 8 rows of a K load (8 bytes a lane) and
// the 4 even or odd rows of a V load (4 bytes a lane) each fall in distinct banks.
__device__ __forceinline__ int tile_pos(int r) { return r ^ ((r >> 2) & 1); }

// PAIR: the block size is a multiple of 32, so a step's two tiles lie in one block, one behind the other.  That
// leaves one block to look up and one address to work out a step: 32 x 8192 positions of 25 heads of 64 take 106
// us against 113, 32 x 16384 of 8 heads of 128 with 16 columns 169 against 177.
template <int NG, int NT, bool PAIR>
__global__ void __launch_bounds__(kPaThreads, PaShape<NG, NT>::kCtas) paged_attn_kernel(PagedAttnArgs a) {
    using Sh = PaShape<NG, NT>;
    constexpr int HS = Sh::kHS, COLS = Sh::kCols, STAGES = Sh::kStages;
    extern __shared__ __align__(16) unsigned char smem[];
    long long* pre = reinterpret_cast<long long*>(smem + Sh::kSmem);
    __shared__ long long wsum[kPaWarps];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int ratio = a.NH / a.NKV;

    pdl_wait();
    pdl_trigger();  // the joining launch may wait on the SMs as they become free
    pa_scan(a, COLS, pre, wsum, blockIdx.x == 0);
    const long long total = pre[a.B];
    const int G = (int)min((long long)gridDim.x, total);
    if ((int)blockIdx.x >= G) return;
    long long u = pa_run(total, blockIdx.x, G);
    const long long u_end = pa_run(total, blockIdx.x + 1, G);
    int b = pa_find(pre, a.B, u);

    // this lane's places in a stage
    const uint32_t q_lane = smem_addr(smem) + Sh::kJoin + lane * 8;
    const uint32_t ring = smem_addr(smem) + w * (STAGES * Sh::kStageBytes);
    const uint32_t k_off = tile_pos(g) * 32 + 8 * t;           // K codes, rows g and (+ 256) g + 8
    const uint32_t m_off = tile_pos(g) * 4 * NG;               // steps of the same rows
    const uint32_t va_off = tile_pos(2 * t) * 32 + 4 * g;      // V codes of the row pairs (2t, 2t + 1)
    const uint32_t vb_off = tile_pos(2 * t + 1) * 32 + 4 * g;

    while (u < u_end) {
        while (pre[b + 1] <= u) b++;
        const PaRequest rq = pa_request(a, b, COLS, false);
        const PaPlace pl = pa_place(rq, u - pre[b]);
        const int kvh = pl.kvh, chunk = pl.chunk, v1 = (int)min((long long)rq.units, pl.unit + (u_end - u));
        u += v1 - pl.unit;
        const int t0 = max(pl.unit - kPaExtra, 0), t1 = v1 - kPaExtra;
        if (t1 <= 0) continue;  // the next CTA begins this one
        const int ncol = min(COLS, rq.n * ratio - chunk * COLS);
        const int last = rq.len - rq.n;  // row i sees positions <= last + i
        const int row_lo = chunk * COLS / ratio, row_hi = (chunk * COLS + ncol - 1) / ratio;
        const int seen_all = last + row_lo;                               // seen by every column
        const int p_end = min(min(rq.len, last + row_hi + 1), t1 * kPaUnit);  // behind the last position seen

        // ---- queries, on their way while the first blocks are looked up: column g of each tile, channels
        // 16t .. 16t + 15 of each group
        uint4 raw[NT][NG][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int col = nt * 8 + g, gc = chunk * COLS + col;
            const __nv_bfloat16* src =
                a.qkv + (size_t)(rq.r0 + gc / ratio) * a.ld + (size_t)(kvh * ratio + gc % ratio) * HS + 16 * t;
#pragma unroll
            for (int ng = 0; ng < NG; ng++)
#pragma unroll
                for (int k = 0; k < 2; k++)
                    raw[nt][ng][k] = col < ncol ? *reinterpret_cast<const uint4*>(src + ng * kW4Group + 8 * k) : make_uint4(0, 0, 0, 0);
        }

        // ---- this warp's steps: positions first, first + kPaUnit, ..
        const int first = t0 * kPaUnit + w * kPaStep;
        const int steps = first < p_end ? (p_end - first + kPaUnit - 1) / kPaUnit : 0;
        const int* table = a.block_table + (size_t)b * a.max_blocks;
        const uint32_t head_rows = (uint32_t)a.NKV * a.block_size;  // positions of one K or V part of a block
        const uint32_t page = head_rows * HS, meta_page = head_rows * (2 * 4 * NG);
        const uint8_t* k_src = a.codes + (size_t)kvh * a.block_size * (HS / 2) + lane * 16;
        const bool v_meta = lane & (4 * NG);  // lanes: [tile][K|V][16-byte piece of the tile's steps]
        const uint8_t* m_src = reinterpret_cast<const uint8_t*>(a.scales) +
                               ((size_t)kvh * a.block_size + (v_meta ? head_rows : 0)) * (4 * NG) + lane % (4 * NG) * 16;
        uint32_t bad = 0;  // two bits a stage: tiles whose block lies outside the cache

        // a step on its way: its two tiles' blocks and positions in them
        struct Step {
            int blk0, blk1, off0, off1;
        };
        int f_pos = first, f_idx = first / a.block_size, f_off = first % a.block_size;  // of the next one to be looked up
        auto fetch = [&]() {
            Step f{0, 0, 0, 0};
            if (f_pos < p_end) {
                f.off0 = f_off;
                f.blk0 = f.blk1 = table[f_idx];
                if constexpr (!PAIR) {
                    const bool next = f_off + 16 >= a.block_size, two = f_pos + 16 < p_end;
                    f.off1 = two ? (next ? 0 : f_off + 16) : f_off;  // behind the end: the first tile again
                    f.blk1 = table[f_idx + (two && next)];
                }
                f_pos += kPaUnit;
                f_idx += a.unit_blocks;
                f_off += a.unit_rest;
                if (f_off >= a.block_size) {
                    f_off -= a.block_size;
                    f_idx++;
                }
            }
            return f;
        };
        auto issue = [&](Step f, int it, int stage) {
            if (it < steps) {
                const uint32_t base = ring + stage * Sh::kStageBytes;
                const bool bad0 = (unsigned)f.blk0 >= (unsigned)a.num_blocks;
                const bool bad1 = PAIR ? bad0 : (unsigned)f.blk1 >= (unsigned)a.num_blocks;
                bad &= ~(3u << (2 * stage));
                if (bad0 || bad1) {  // left out: block 0 is read in its place and masked
                    bad |= (bad0 ? 1u : 0u) << (2 * stage) | (bad1 ? 2u : 0u) << (2 * stage);
                    if (bad0) f.blk0 = 0;
                    if (bad1) f.blk1 = 0;
                    if (lane == 0) report_device_error(GPT2B_DEVERR_BAD_BLOCK);
                }
                const uint8_t* src0 = k_src + ((size_t)(uint32_t)f.blk0 * page + (uint32_t)f.off0 * (HS / 2));
                const uint8_t* src[2] = {src0, PAIR ? src0 + 16 * (HS / 2)
                                                    : k_src + ((size_t)(uint32_t)f.blk1 * page + (uint32_t)f.off1 * (HS / 2))};
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < NG; k++) {
                        const int i = lane + 32 * k, row = i / (2 * NG), c = i % (2 * NG);
                        const uint32_t dst = base + (c >> 1) * (kPaStep * 32) + (16 * j + row) * 32 + (c & 1) * 16;
                        cp_async16(dst, src[j] + k * 512);
                        cp_async16(dst + Sh::kCodeBytes, src[j] + head_rows * (HS / 2) + k * 512);
                    }
                const bool hi = lane >= 8 * NG;
                if (lane < 16 * NG)
                    cp_async16(base + 2 * Sh::kCodeBytes + (v_meta ? Sh::kMetaBytes : 0) + (hi ? 64 * NG : 0) + lane % (4 * NG) * 16,
                               PAIR ? m_src + (hi ? 64 * NG : 0) + ((size_t)(uint32_t)f.blk0 * meta_page + (uint32_t)f.off0 * (4 * NG))
                                    : m_src + ((size_t)(uint32_t)(hi ? f.blk1 : f.blk0) * meta_page +
                                               (uint32_t)(hi ? f.off1 : f.off0) * (4 * NG)));
            }
            cp_async_commit();
        };

        // the first steps' blocks are looked up together, not one behind the other's copies
        Step ahead[STAGES];
#pragma unroll
        for (int k = 0; k < STAGES; k++) ahead[k] = fetch();
#pragma unroll
        for (int k = 0; k < STAGES - 1; k++) issue(ahead[k], k, k);
        Step pending = ahead[STAGES - 1];

        // ---- queries as the B operand, scaled to [2^10, 2^11) at a column's largest
        uint32_t q[Sh::kQShared ? 1 : NT][NG][4][2];
        if constexpr (Sh::kQShared) __syncthreads();  // the piece before has been read
        float cf[NT][2], qs[NT][NG][2];
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            uint32_t u[NG][8];
            float mx = 0.0f;
#pragma unroll
            for (int ng = 0; ng < NG; ng++) {
                const uint4 x = raw[nt][ng][0], y = raw[nt][ng][1];
                u[ng][0] = x.x; u[ng][1] = x.y; u[ng][2] = x.z; u[ng][3] = x.w;
                u[ng][4] = y.x; u[ng][5] = y.y; u[ng][6] = y.z; u[ng][7] = y.w;
#pragma unroll
                for (int k = 0; k < 8; k++) mx = fmaxf(mx, fmaxf(fabsf(bf16lo(u[ng][k])), fabsf(bf16hi(u[ng][k]))));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int field = min(264 - (int)(__float_as_uint(mx) >> 23), 254);
            // the sign of the softmax scale goes to q, so that scores grow with S
            const float f = copysignf(pow2_field(field), a.scale_log2);
            // D is in units of 2^-20 / f; never 0 or infinite, so that a masked -infinity and a 0 stay ones
            const float c = fminf(fmaxf(fabsf(a.scale_log2) * 1048576.0f * pow2_field(254 - field), 0x1p-120f), FLT_MAX);
            cf[nt][0] = __shfl_sync(0xffffffffu, c, 8 * t);
            cf[nt][1] = __shfl_sync(0xffffffffu, c, 8 * t + 4);
#pragma unroll
            for (int ng = 0; ng < NG; ng++) {
                float v[16], s = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    v[2 * k] = bf16lo(u[ng][k]) * f;
                    v[2 * k + 1] = bf16hi(u[ng][k]) * f;
                    s += v[2 * k] + v[2 * k + 1];
                }
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                s *= 9.5367431640625e-7f;  // 2^-20
                qs[nt][ng][0] = __shfl_sync(0xffffffffu, s, 8 * t);
                qs[nt][ng][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float* z = v + 8 * e + 2 * h;
                        const uint32_t q0 = f16x2(z[0] * 16.0f, z[4] * 16.0f), q1 = f16x2(z[1], z[5]);
                        if constexpr (Sh::kQShared) {
                            if (w == 2 * e + h) sts64(q_lane + ((nt * NG + ng) * 4 + 2 * e + h) * 256, q0, q1);
                        } else {
                            q[nt][ng][2 * e + h][0] = q0;
                            q[nt][ng][2 * e + h][1] = q1;
                        }
                    }
            }
#pragma unroll
            for (int c2 = 0; c2 < 2; c2++) {
                const int cc = nt * 8 + 2 * t + c2;
                lim[nt][c2] = cc < ncol ? last + (chunk * COLS + cc) / ratio : rq.len - 1;
            }
        }

        if constexpr (Sh::kQShared) __syncthreads();

        float m[NT][2], l[NT][2], az[NT][NG][2], acc[NT][NG][4][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -FLT_MAX;  // nothing seen
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int ng = 0; ng < NG; ng++) {
                az[nt][ng][0] = az[nt][ng][1] = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[nt][ng][i][k] = 0.0f;
            }
        }
        // A column's acc carries its `vscale`, a power of two that brings the V steps that the column sees below
        // 2^31: with the weights, at most 2^(8 - kBias), they stay below 2^15, in FP16's range.  Steps that it does
        // not see have no part in it, or a later row's outlier would take bits from an earlier row.  Only masked steps
        // make columns differ, and what follows a step that some columns do not see is masked too, so unmasked ones
        // find the same vscale everywhere.  l and az have no factor: low ends have a range of their own.
        float vscale[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) vscale[nt][0] = vscale[nt][1] = 0x1p124f;

        auto step = [&](auto mask_tag, int p0, uint32_t base, uint32_t badbits) {
            constexpr bool MASKED = decltype(mask_tag)::value;
            const uint32_t mbase = base + 2 * Sh::kCodeBytes + m_off;

            // ---- scores
            float S[2][NT][4];
            uint32_t km[2][2][NG];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int k = 0; k < 2; k++) lds_meta<NG>(mbase + j * (64 * NG) + k * (32 * NG), km[j][k]);
#pragma unroll
            for (int ng = 0; ng < NG; ng++) {
                float D[2][NT][4];
                uint2 x[2], y[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t addr = base + ng * (kPaStep * 32) + j * 512 + k_off;
                    x[j] = lds64(addr);
                    y[j] = lds64(addr + 256);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int k = 0; k < 4; k++) D[j][nt][k] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint2 qf[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if constexpr (Sh::kQShared) qf[nt] = lds64(q_lane + ((nt * NG + ng) * 4 + 2 * e + h) * 256);
                            else qf[nt] = make_uint2(q[nt][ng][2 * e + h][0], q[nt][ng][2 * e + h][1]);
                        }
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t xx = (e ? x[j].y : x[j].x) >> (8 * h), yy = (e ? y[j].y : y[j].x) >> (8 * h);
                            const uint32_t a0 = xx & kEven, a1 = yy & kEven, a2 = xx & kOdd, a3 = yy & kOdd;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma_f16(D[j][nt], a0, a1, a2, a3, qf[nt].x, qf[nt].y);
                        }
                    }
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float ks = meta_step(km[j][k][ng]), kz = meta_low(km[j][k][ng]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if constexpr (Sh::kPacked) {
                                float z0, z1;
                                if (ng == 0) {
                                    z0 = kz * qs[nt][0][0];
                                    z1 = kz * qs[nt][0][1];
                                } else {
                                    fma2(z0, z1, kz, kz, qs[nt][ng][0], qs[nt][ng][1], S[j][nt][2 * k], S[j][nt][2 * k + 1]);
                                }
                                fma2(S[j][nt][2 * k], S[j][nt][2 * k + 1], ks, ks, D[j][nt][2 * k], D[j][nt][2 * k + 1], z0, z1);
                            } else {
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    const float z = ng == 0 ? kz * qs[nt][0][c] : fmaf(kz, qs[nt][ng][c], S[j][nt][2 * k + c]);
                                    S[j][nt][2 * k + c] = fmaf(ks, D[j][nt][2 * k + c], z);
                                }
                            }
                        }
                    }
            }
            uint32_t hidden = 0;  // a bit a score: positions that a column does not see
            if constexpr (MASKED) {
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int p = p0 + 16 * j + tile_pos(g) + (k >> 1) * 8;
                            if (p > lim[nt][k & 1] || ((badbits >> j) & 1u)) {
                                S[j][nt][k] = -INFINITY;
                                hidden |= 1u << ((j * NT + nt) * 4 + k);
                            }
                        }
            }
            // ---- running maximum: raised only where a score passes it by 2^8, so weights stay below 2^8
            bool grow = false;
            float top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    top[nt][c] = fmaxf(fmaxf(S[0][nt][c], S[0][nt][c + 2]), fmaxf(S[1][nt][c], S[1][nt][c + 2])) * cf[nt][c];
                    grow = grow || top[nt][c] > m[nt][c] + 8.0f;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float x = top[nt][c];
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                        // a column's own scores decide, so that its bits do not depend on another's
                        const float mn = x > m[nt][c] + 8.0f ? x : m[nt][c];
                        const float f = mn == m[nt][c] ? 1.0f : ex2(m[nt][c] - mn);
                        m[nt][c] = mn;
                        l[nt][c] *= f;
#pragma unroll
                        for (int ng = 0; ng < NG; ng++) {
                            az[nt][ng][c] *= f;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                acc[nt][ng][i][c] *= f;
                                acc[nt][ng][i][c + 2] *= f;
                            }
                        }
                    }
            }
            // ---- V steps; a column's largest where it passes what the column's factor allows
            uint32_t vm[2][2][NG];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int k = 0; k < 2; k++) lds_meta<NG>(mbase + Sh::kMetaBytes + j * (64 * NG) + k * (32 * NG), vm[j][k]);
            auto largest = [&](int nt, int c, bool finite) {  // of this lane's positions that the column sees
                float big = 0.0f;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int ng = 0; ng < NG; ng++) {
                            const float x = fabsf(meta_step(vm[j][k][ng]));
                            if (!(hidden >> ((j * NT + nt) * 4 + 2 * k + c) & 1u) && (!finite || x < INFINITY)) big = fmaxf(big, x);
                        }
                return big;
            };
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < (MASKED ? NT : 1); nt++)
#pragma unroll
                for (int c = 0; c < (MASKED ? 2 : 1); c++) over = over || largest(nt, c, false) * vscale[nt][c] >= 0x1p31f;
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float big = largest(nt, c, true);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                        if (big * vscale[nt][c] >= 0x1p31f) {
                            // largest step -> [2^28, 2^29), with room for two exponents of growth
                            const float next = pow2_field(282 - (int)(__float_as_uint(big) >> 23));
                            const float f = next * pow2_inverse(vscale[nt][c]);
                            vscale[nt][c] = next;
#pragma unroll
                            for (int ng = 0; ng < NG; ng++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    acc[nt][ng][i][c] *= f;
                                    acc[nt][ng][i][c + 2] *= f;
                                }
                        }
                    }
            }
            // ---- weights (FP32 statistics, FP16 operands) and out += codes_V^T . weights
            float off[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) off[nt][c] = -kBias - m[nt][c];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint32_t wb[NT][NG][2];
                float vt[NG][2];
#pragma unroll
                for (int ng = 0; ng < NG; ng++)
#pragma unroll
                    for (int k = 0; k < 2; k++) vt[ng][k] = meta_step(vm[j][k][ng]) * (MASKED ? 1.0f : vscale[0][0]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        fma2(p[k], p[k + 1], S[j][nt][k], S[j][nt][k + 1], cf[nt][0], cf[nt][1], off[nt][0], off[nt][1]);
                        p[k] = ex2(p[k]);
                        p[k + 1] = ex2(p[k + 1]);
                        add2(l[nt][0], l[nt][1], p[k], p[k + 1]);
                    }
#pragma unroll
                    for (int ng = 0; ng < NG; ng++) {
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const float vz = meta_low(vm[j][k][ng]);
                            float x[2];
                            if constexpr (!MASKED && Sh::kPacked) {
                                x[0] = p[2 * k] * vt[ng][k];
                                x[1] = p[2 * k + 1] * vt[ng][k];
                                fma2(az[nt][ng][0], az[nt][ng][1], p[2 * k], p[2 * k + 1], vz, vz, az[nt][ng][0], az[nt][ng][1]);
                            } else {
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    // a position that this column does not see may hold NaN, and 0 * NaN is not 0
                                    const bool none = MASKED && (hidden >> ((j * NT + nt) * 4 + 2 * k + c) & 1u);
                                    x[c] = none ? 0.0f : p[2 * k + c] * (MASKED ? vt[ng][k] * vscale[nt][c] : vt[ng][k]);
                                    az[nt][ng][c] = none ? az[nt][ng][c] : fmaf(p[2 * k + c], vz, az[nt][ng][c]);
                                }
                            }
                            wb[nt][ng][k] = mov_trans(f16x2(x[0], x[1]));
                        }
                    }
                }
#pragma unroll
                for (int ng = 0; ng < NG; ng++) {
                    const uint32_t vaddr = base + Sh::kCodeBytes + ng * (kPaStep * 32) + j * 512;
                    const uint32_t x0 = lds32(vaddr + va_off), x1 = lds32(vaddr + vb_off);
                    const uint32_t y0 = lds32(vaddr + 256 + va_off), y1 = lds32(vaddr + 256 + vb_off);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t sel = i < 2 ? 0x5410u : 0x7632u;
                        const uint32_t x = __byte_perm(x0, x1, sel) >> (8 * (i & 1)), y = __byte_perm(y0, y1, sel) >> (8 * (i & 1));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            mma_f16(acc[nt][ng][i], x & kEven, x & kOdd, y & kEven, y & kOdd, wb[nt][ng][0], wb[nt][ng][1]);
                    }
                }
            }
        };
        int stage = 0;
        for (int it = 0; it < steps; it++) {
            __syncwarp();  // every lane has read the stage that is filled next
            issue(pending, it + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
            pending = fetch();
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            const int p0 = first + it * kPaUnit;
            const uint32_t badbits = (bad >> (2 * stage)) & 3u;
            if (badbits == 0 && p0 + kPaStep - 1 <= seen_all)
                step(std::false_type{}, p0, ring + stage * Sh::kStageBytes, 0u);
            else
                step(std::true_type{}, p0, ring + stage * Sh::kStageBytes, badbits);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }

        // ---- join the four warps
        float* slab = reinterpret_cast<float*>(smem);
        float* s_m = slab + kPaWarps * COLS * Sh::kPitch;
        float* s_l = s_m + kPaWarps * COLS;
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
#pragma unroll
                    for (int ng = 0; ng < NG; ng++) az[nt][ng][c] += __shfl_xor_sync(0xffffffffu, az[nt][ng][c], o);
                }
                if (g == 0) s_m[w * COLS + nt * 8 + 2 * t + c] = m[nt][c];
            }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int col = nt * 8 + 2 * t + c;
                const float even = 16777216.0f * pow2_inverse(vscale[nt][c]), odd = 0.0625f * even;
                float M = s_m[col];
                for (int k = 1; k < kPaWarps; k++) M = fmaxf(M, s_m[k * COLS + col]);
                const float f = ex2(m[nt][c] - M);  // 1 where nothing was seen: zeros (or NaN) are joined
                if (g == 0) s_l[w * COLS + col] = l[nt][c] * f;
                float* dst = slab + (w * COLS + col) * Sh::kPitch;
#pragma unroll
                for (int ng = 0; ng < NG; ng++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int ch = ng * kW4Group + 8 * g + 2 * i;
                        dst[ch] = fmaf(acc[nt][ng][i][c], even, az[nt][ng][c]) * f;
                        dst[ch + 1] = fmaf(acc[nt][ng][i][c + 2], odd, az[nt][ng][c]) * f;
                    }
            }
        __syncthreads();
        const bool whole = t0 == 0 && v1 == rq.units;
        float* slot = a.ws + ((size_t)blockIdx.x * 2 + (t0 > 0 ? 0 : 1)) * Sh::kSlot;
        for (int i = tid; i < ncol * (HS / 2); i += kPaThreads) {
            const int col = i / (HS / 2), ch = 2 * (i % (HS / 2));
            float x = 0.0f, y = 0.0f, sum = 0.0f;
            for (int k = 0; k < kPaWarps; k++) {
                x += slab[(k * COLS + col) * Sh::kPitch + ch];
                y += slab[(k * COLS + col) * Sh::kPitch + ch + 1];
                sum += s_l[k * COLS + col];
            }
            if (whole) {
                const int gc = chunk * COLS + col;
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                __nv_bfloat16* o = a.out + (size_t)(rq.r0 + gc / ratio) * a.NH * HS + (size_t)(kvh * ratio + gc % ratio) * HS + ch;
                *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(x * inv, y * inv);
            } else {
                slot[col * HS + ch] = x;
                slot[col * HS + ch + 1] = y;
                if (ch == 0) {
                    float M = s_m[col];
                    for (int k = 1; k < kPaWarps; k++) M = fmaxf(M, s_m[k * COLS + col]);
                    slot[COLS * HS + col] = M;
                    slot[COLS * HS + COLS + col] = sum;
                }
            }
        }
        __syncthreads();
    }
}

// Joins the pieces of the segments that several CTAs shared: block i takes the segment that the border between
// the runs of CTAs i and i + 1 cuts, if that is the segment's first border.  A thread holds two channels of a
// column; pieces are added in the order of their CTAs.  Launched early: its CTAs find their
// segments while the last of the main ones still run.
template <int NG, int NT>
__global__ void __launch_bounds__(kPaThreads) paged_attn_join_kernel(PagedAttnArgs a, int main_grid) {
    using Sh = PaShape<NG, NT>;
    constexpr int HS = Sh::kHS, COLS = Sh::kCols;
    extern __shared__ __align__(16) unsigned char smem[];
    long long* pre = reinterpret_cast<long long*>(smem);
    __shared__ long long wsum[kPaWarps];
    // Lengths and offsets are read ahead of pdl_wait: the main launch lets this one start only behind its own wait,
    // when whatever wrote them has ended, and does not write them itself.
    pa_scan(a, COLS, pre, wsum, false);
    const long long total = pre[a.B];
    const int G = (int)min((long long)main_grid, total), i0 = blockIdx.x;
    const int ratio = a.NH / a.NKV;
    bool mine = false;
    int b = 0, kvh = 0, chunk = 0, pieces = 0;
    PaRequest rq{};
    if (i0 + 1 < G) {
        const long long u = pa_run(total, i0 + 1, G);
        b = pa_find(pre, a.B, u);
        rq = pa_request(a, b, COLS, false);
        const PaPlace pl = pa_place(rq, u - pre[b]);
        kvh = pl.kvh;
        chunk = pl.chunk;
        const long long begin = u - pl.unit + kPaExtra, end = u - pl.unit + rq.units;
        // CTA of a unit x: the last one whose run begins at or before it
        mine = u > begin && ((begin + 1) * G - 1) / total == i0;
        pieces = (int)((end * G - 1) / total - i0) + 1;
    }
    const int i = (int)blockIdx.y * kPaThreads + (int)threadIdx.x;
    const int col = i / (HS / 2), ch = 2 * (i % (HS / 2));
    mine = mine && col < min(COLS, rq.n * ratio - chunk * COLS);
    pdl_wait();
    if (!mine) return;
    // piece k > 0 is slot 0 of CTA i0 + k, the first slot 1 of CTA i0
    const float* first = a.ws + ((size_t)i0 * 2 + 1) * Sh::kSlot;
    auto slot = [&](int k) { return k == 0 ? first : first + (2 * (size_t)k - 1) * Sh::kSlot; };
    constexpr int kAhead = 16;  // pieces whose results are on their way together
    float M = -FLT_MAX, x = 0.0f, y = 0.0f, sum = 0.0f;
    for (int k0 = 0; k0 < pieces; k0 += kAhead) {
        float m[kAhead], l[kAhead];
        float2 o[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            m[k] = -FLT_MAX;
            l[k] = 0.0f;
            o[k] = make_float2(0.0f, 0.0f);
            if (k0 + k < pieces) {
                const float* s = slot(k0 + k);
                m[k] = s[COLS * HS + col];
                l[k] = s[COLS * HS + COLS + col];
                o[k] = *reinterpret_cast<const float2*>(s + col * HS + ch);
            }
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < kAhead; k++) top = fmaxf(top, m[k]);
        const float f = ex2(M - top);
        x *= f;
        y *= f;
        sum *= f;
        M = top;
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const float fk = ex2(m[k] - M);
            x = fmaf(o[k].x, fk, x);
            y = fmaf(o[k].y, fk, y);
            sum = fmaf(l[k], fk, sum);
        }
    }
    const int gc = chunk * COLS + col;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    __nv_bfloat16* o = a.out + (size_t)(rq.r0 + gc / ratio) * a.NH * HS + (size_t)(kvh * ratio + gc % ratio) * HS + ch;
    *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(x * inv, y * inv);
}

// Two tiles of 8 columns where a request's rows and shared heads give more than 8.
static int pa_tiles(int NH, int NKV, int max_q) { return (long long)(NH / NKV) * max_q <= 8 ? 1 : 2; }

template <int NG, int NT> static size_t pa_workspace() {
    return (size_t)sm_count() * PaShape<NG, NT>::kCtas * 2 * PaShape<NG, NT>::kSlot * sizeof(float);
}

template <int NG, int NT, bool PAIR> static cudaError_t pa_launch(const PagedAttnArgs& a, cudaStream_t st) {
    using Sh = PaShape<NG, NT>;
    static unsigned long long mask = 0, mask2 = 0;
    cudaError_t e = ensure_smem_limit(paged_attn_kernel<NG, NT, PAIR>, &mask);
    if (e == cudaSuccess) e = ensure_smem_limit(paged_attn_join_kernel<NG, NT>, &mask2);
    if (e != cudaSuccess) return e;
    const size_t pre = sizeof(long long) * ((size_t)a.B + 1);
    // one wave: no more CTAs than fit an SM's 228 KB of shared memory (1 KB of each is the system's)
    const int fit = (int)(228 * 1024 / (Sh::kSmem + pre + 1024 + 512));
    const int grid = sm_count() * (fit < Sh::kCtas ? fit : Sh::kCtas);
    e = launch_k(paged_attn_kernel<NG, NT, PAIR>, dim3(grid), dim3(kPaThreads), Sh::kSmem + pre, st, true, a);
    if (e != cudaSuccess) return e;
    // a thread two channels of a column
    const unsigned parts = Sh::kCols * (Sh::kHS / 2) / kPaThreads;
    return launch_k(paged_attn_join_kernel<NG, NT>, dim3(grid - 1, parts), dim3(kPaThreads), pre, st, true, a, grid);
}

template <int NG, int NT> static cudaError_t pa_launch(const PagedAttnArgs& a, cudaStream_t st) {
    return a.block_size % kPaStep == 0 ? pa_launch<NG, NT, true>(a, st) : pa_launch<NG, NT, false>(a, st);
}

}  // namespace gpt2b

using namespace gpt2b;

extern "C" {

int gpt2b_attention_paged_w4_workspace(int NH, int NKV, int hs, int max_q, size_t* bytes) {
    if (NH <= 0 || NKV <= 0 || NH % NKV != 0 || max_q <= 0 || !bytes) return GPT2B_ERR_INVALID_ARG;
    if (hs != 64 && hs != 128) return GPT2B_ERR_UNSUPPORTED;
    const int nt = pa_tiles(NH, NKV, max_q);
    *bytes = hs == 64 ? (nt == 1 ? pa_workspace<1, 1>() : pa_workspace<1, 2>())
                      : (nt == 1 ? pa_workspace<2, 1>() : pa_workspace<2, 2>());
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
    if (!(scale >= -1e30f && scale <= 1e30f)) return GPT2B_ERR_INVALID_ARG;
    // (positions are counted a few units past the end in 32 bits)
    if (block_size % kW4Tile != 0 || B > kTableMaxRequests || (long long)max_blocks * block_size > 1 << 30)
        return GPT2B_ERR_UNSUPPORTED;
    if (!aligned16(out) || !aligned16(qkv) || !aligned16(kv_cache) || !aligned16(kv_scale) || !aligned16(workspace) ||
        ld % 8 != 0)
        return GPT2B_ERR_ALIGNMENT;
    if (rows == 0) return GPT2B_OK;
    if ((long long)rows * NH > INT_MAX - 64) return GPT2B_ERR_UNSUPPORTED;
    if ((long long)NKV * block_size * hs > INT_MAX) return GPT2B_ERR_UNSUPPORTED;  // bytes of a block
    const size_t codes = (size_t)NKV * block_size * hs * num_blocks, b4 = 4 * (size_t)B;
    if (outputs_overlap({{out, 2 * (size_t)rows * NH * hs}, {workspace, need}},
                        {{qkv, 2 * ((size_t)(rows - 1) * ld + ((size_t)NH + 2 * (size_t)NKV) * hs)}, {kv_cache, codes},
                         {kv_scale, codes / 8}, {block_table, b4 * max_blocks}, {seq_lens, b4}, {row_start, b4 + 4}}))
        return GPT2B_ERR_INVALID_ARG;
    const PagedAttnArgs a{(__nv_bfloat16*)out, (const __nv_bfloat16*)qkv, kv_cache, (const uint32_t*)kv_scale, block_table,
                          seq_lens, row_start, B, rows, NH, NKV, ld, num_blocks, block_size, max_blocks,
                          kPaUnit / block_size, kPaUnit % block_size,
                          scale * 1.4426950408889634f, (float*)workspace};
    const cudaStream_t st = (cudaStream_t)stream;
    if (pa_tiles(NH, NKV, max_q) == 1)
        return status_from(hs == 64 ? pa_launch<1, 1>(a, st) : pa_launch<2, 1>(a, st));
    return status_from(hs == 64 ? pa_launch<1, 2>(a, st) : pa_launch<2, 2>(a, st));
}

}  // extern "C"
