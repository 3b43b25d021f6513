// paged_kv.cu -- a paged KV cache held in 4 bits: block tables and slot maps
// from request lengths, append and read-back.
//
// Cache of one layer: codes u8 [num_blocks][K|V][NKV][block_size][hs/2] (byte i
// of a row: channel 2i in the low nibble, 2i+1 in the high one) and steps
// [num_blocks][K|V][NKV][block_size][hs/64][2] BF16 (step s, low end lo of each
// group of 64 channels).  value = code * s + lo.  4.5 bits a value.
#include "common.cuh"
#include "internal.h"
#include "paged_kv.cuh"

#include <limits.h>

namespace gpt2b {

GPT2B_DEFINE_ERROR_READER(paged_kv_device_error)

// ---------------------------------------------------------------------------
// block tables and slot maps
// ---------------------------------------------------------------------------
// Every CTA computes the two exclusive prefix sums over the requests (rows, and
// blocks to be taken from the free list) for itself and then writes its share of
// the rows and of the table entries, so one launch does without a grid barrier:
// 12 bytes a request from L2 against a second launch.  Nothing that a CTA reads
// is written by another: a row's block is either one that the request held
// (below have, which no CTA writes) or comes from the free list directly.
// Bound by its launch and the chain lengths - scan - block - store: 2.7 us for 8
// requests of one row, 3.7 us for 256 with 64000 rows (a row a thread; with four rows
// a thread in a quarter of the CTAs 5.9 us).
constexpr int kTabThreads = 256;

struct TableArgs {
    int* block_table;
    long long* slot_map;
    int *positions, *row_start, *seq_lens, *blocks_out, *free_left;
    const int *ctx_lens, *new_lens, *blocks_have, *free_list, *free_count;
    int B, max_blocks, block_size, max_rows, free_cap;
};

struct Request {
    long long end;  // context + new rows
    int n, ctx, have;
};
__device__ __forceinline__ Request load_request(const TableArgs& a, int b) {
    Request r;
    r.ctx = max(a.ctx_lens[b], 0);
    r.n = max(a.new_lens[b], 0);
    r.have = min(max(a.blocks_have[b], 0), a.max_blocks);
    r.end = (long long)r.ctx + r.n;
    return r;
}

__global__ void __launch_bounds__(kTabThreads) block_tables_kernel(TableArgs a) {
    extern __shared__ int tab_smem[];
    int* row_end = tab_smem;        // [B] inclusive prefix of rows, at most max_rows
    int* excl = tab_smem + a.B;     // [B] exclusive prefix of blocks asked for, at most INT_MAX
    int* need = tab_smem + 2 * a.B; // [B] blocks asked for, or -1 where the request is not served
    __shared__ long long w_rows[kTabThreads / 32], w_need[kTabThreads / 32];
    __shared__ int s_take;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    pdl_wait();
    const int F = min(max(*a.free_count, 0), a.free_cap);
    const long long most = (long long)a.max_blocks * a.block_size;
    if (tid == 0) s_take = 0;
    long long rows0 = 0, need0 = 0;  // totals of the requests before this pass
    for (int base = 0; base < a.B; base += kTabThreads) {
        const int b = base + tid;
        Request r{};
        if (b < a.B) r = load_request(a, b);
        // a refused request asks for no block; whether its rows fit is known after the first scan
        long long rows = r.n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, rows, o);
            if (lane >= o) rows += v;
        }
        if (lane == 31) w_rows[w] = rows;
        __syncthreads();
        long long before = rows0, all_rows = 0;
        for (int k = 0; k < kTabThreads / 32; k++) {
            if (k < w) before += w_rows[k];
            all_rows += w_rows[k];
        }
        rows += before;
        const bool fits = b < a.B && r.end <= most && rows <= a.max_rows;
        const long long blocks = (r.end + a.block_size - 1) / a.block_size;
        const int nd = fits && blocks > r.have ? (int)(blocks - r.have) : 0;
        long long upto = nd;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) w_need[w] = upto;
        __syncthreads();
        long long nbefore = need0, all_need = 0;
        for (int k = 0; k < kTabThreads / 32; k++) {
            if (k < w) nbefore += w_need[k];
            all_need += w_need[k];
        }
        upto += nbefore;
        if (b < a.B) {
            const bool served = fits && (nd == 0 || upto <= F);
            row_end[b] = (int)min(rows, (long long)a.max_rows);
            excl[b] = (int)min(upto - nd, (long long)INT_MAX);
            need[b] = served ? nd : -1;
            if (served && nd) atomicMax(&s_take, (int)upto);
            if (blockIdx.x == 0) {
                a.row_start[b + 1] = row_end[b];
                a.seq_lens[b] = served ? (int)r.end : 0;
                a.blocks_out[b] = r.have + (served ? nd : 0);
            }
        }
        rows0 += all_rows;
        need0 += all_need;
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) {
        a.row_start[0] = 0;
        *a.free_left = F - s_take;
    }
    // table entries of the new blocks: a warp per request
    for (int b = blockIdx.x * (kTabThreads / 32) + w; b < a.B; b += gridDim.x * (kTabThreads / 32)) {
        const int nd = need[b];
        if (nd <= 0) continue;
        const int have = min(max(a.blocks_have[b], 0), a.max_blocks);
        for (int j = lane; j < nd; j += 32)
            a.block_table[(size_t)b * a.max_blocks + have + j] = a.free_list[F - 1 - excl[b] - j];
    }
    // rows
    for (long long i = (long long)blockIdx.x * kTabThreads + tid; i < a.max_rows; i += (long long)gridDim.x * kTabThreads) {
        const int r = (int)i;
        int lo = 0, hi = a.B;  // first request whose rows end behind r
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (row_end[mid] > r) hi = mid; else lo = mid + 1;
        }
        long long slot = -1;
        int pos = 0;
        if (lo < a.B && need[lo] >= 0) {
            const Request q = load_request(a, lo);
            // a served request's rows are not cut, so it begins n rows before its end
            pos = q.ctx + (r - (row_end[lo] - q.n));
            const int j = pos / a.block_size;
            const int blk = j < q.have ? a.block_table[(size_t)lo * a.max_blocks + j]
                                       : a.free_list[F - 1 - excl[lo] - (j - q.have)];
            slot = blk < 0 ? -1 : (long long)blk * a.block_size + pos % a.block_size;
        }
        a.slot_map[r] = slot;
        a.positions[r] = pos;
    }
}

// ---------------------------------------------------------------------------
// append and read-back
// ---------------------------------------------------------------------------
// Appending, a thread holds 16 channels (two 16-byte loads of BF16, one 8-byte store of codes), 4 threads a group
// of 64; reading back 8 (one 4-byte load of codes, one 16-byte store: with 32 bytes a thread the stores of a warp
// left gaps, 24 us against 19).  A CTA's threads cover whole rows, so a thread's head and channels are worked out
// once.  The 8 lanes that share a row (at least) work out the places of their next 8 rows together, one each, and
// hand them round as numbers of 32-byte groups of codes (a step to each, in the same order).  Several rows' loads
// are in flight.  16384 rows of 2 * 8 * 128: 22 us to append and 19 to read back, of 13 each that HBM takes.  Neither
// is full of anything (issue slots 69 and 68 %, ALU pipe 45 and 57 %): with 7 warps a scheduler the batches of loads
// that a thread works through one behind the other, the places of the next rows among them, are most of the wait
// (4.0 and 3.8 of 10.2 cycles an instruction).
constexpr int kRwThreads = 256, kWriteChannels = 16, kReadChannels = 8, kWriteAhead = 2, kReadAhead = 4;
constexpr uint32_t kNoRow = 0xffffffffu;

struct RowPlace {
    int row, col;    // row of the CTA's pass, channel in the row
    uint32_t group;  // this thread's group of codes in a block, at offset 0
    bool active;
};
__device__ __forceinline__ RowPlace row_place(int channels, int hs, int block_size, int per_row, int part, int parts, int rows_per_cta) {
    RowPlace r;
    const int i = part * kRwThreads + threadIdx.x;  // thread of the row pass, over all parts of a wide row
    r.row = parts > 1 ? 0 : i / per_row;
    r.col = (i - r.row * per_row) * channels;
    r.active = parts > 1 ? i < per_row : r.row < rows_per_cta;
    const int head = r.col / hs, d = r.col - head * hs;  // head of [K | V]
    r.group = (uint32_t)head * block_size * (hs / kW4Group) + d / kW4Group;
    return r;
}
// Group of codes where head 0 of the slot's row begins; page: groups of a block.
__device__ __forceinline__ uint32_t slot_group(long long slot, long long slots, int block_size, int per_pos, uint32_t page) {
    if (slot < 0) return kNoRow;
    if (slot >= slots) {
        report_device_error(GPT2B_DEVERR_BAD_BLOCK);
        return kNoRow;
    }
    const unsigned b = (unsigned)slot / (unsigned)block_size;  // slots < 2^32: a slot has groups of its own
    return b * page + ((unsigned)slot - b * (unsigned)block_size) * per_pos;
}

// Bound by the latencies above for many rows (HBM: rows * 2 * NKV * hs * 2.56 bytes), by its launch for few.
__global__ void __launch_bounds__(kRwThreads)
    kv_write_w4_kernel(uint8_t* codes, uint32_t* scales, const __nv_bfloat16* qkv, const long long* slot_map, int rows,
                       int NH, int NKV, int hs, int ld, long long slots, int block_size, int parts, int rows_per_cta) {
    const int per_row = 2 * NKV * hs / kWriteChannels, part = blockIdx.x % parts;
    const RowPlace me = row_place(kWriteChannels, hs, block_size, per_row, part, parts, rows_per_cta);
    pdl_wait();
    if (!me.active) return;  // per_row is a multiple of 8: the 8 lanes of a row leave together
    const uint32_t page = (uint32_t)(2 * NKV) * block_size * (hs / kW4Group);
    const long long step = (long long)(gridDim.x / parts) * rows_per_cta;
    const __nv_bfloat16* src = qkv + (size_t)NH * hs + me.col;
    uint8_t* my_codes = codes + (size_t)me.group * (kW4Group / 2) + (me.col & (kW4Group - 1)) / 2;
    uint32_t* my_scales = scales + me.group;
    const unsigned eight = 0xffu << (threadIdx.x & 24);
    const bool first = (me.col & (kW4Group - 1)) == 0;
    for (long long base = (long long)(blockIdx.x / parts) * rows_per_cta + me.row; base < rows; base += 8 * step) {
        const long long ahead = base + (threadIdx.x & 7) * step;
        const uint32_t place =
            ahead < rows ? slot_group(slot_map[ahead], slots, block_size, hs / kW4Group, page) : kNoRow;
        const __nv_bfloat16* row = src + base * ld;
        const int n = (int)min(8ll, (rows - base + step - 1) / step);
        for (int k0 = 0; k0 < n; k0 += kWriteAhead) {
            uint4 v[kWriteAhead][2];
            uint32_t at[kWriteAhead];
#pragma unroll
            for (int k = 0; k < kWriteAhead; k++) {
                at[k] = __shfl_sync(eight, place, k0 + k, 8);
                if (at[k] != kNoRow) {
                    v[k][0] = reinterpret_cast<const uint4*>(row)[0];
                    v[k][1] = reinterpret_cast<const uint4*>(row)[1];
                }
                row += step * ld;
            }
#pragma unroll
            for (int k = 0; k < kWriteAhead; k++) {
                if (at[k] == kNoRow) continue;
                const uint32_t u[8] = {v[k][0].x, v[k][0].y, v[k][0].z, v[k][0].w, v[k][1].x, v[k][1].y, v[k][1].z, v[k][1].w};
                // ends of the group as (min, -max): pairs, then the two halves, then 4 threads
                uint32_t mn = u[0], mx = u[0];
#pragma unroll
                for (int i = 1; i < 8; i++) {
                    mn = bf16x2_min_nan(mn, u[i]);
                    mx = bf16x2_max_nan(mx, u[i]);
                }
                mx ^= 0x80008000u;
                uint32_t e = bf16x2_min_nan(__byte_perm(mn, mx, 0x5410), __byte_perm(mn, mx, 0x7632));
#pragma unroll
                for (int o = 2; o > 0; o >>= 1) e = bf16x2_min_nan(e, __shfl_xor_sync(eight, e, o));
                uint32_t meta;
                *reinterpret_cast<uint2*>(my_codes + (size_t)at[k] * (kW4Group / 2)) =
                    w4_encode16(u, bf16lo(e), bf16hi(e), meta);
                if (first) my_scales[at[k]] = meta;
            }
        }
    }
}

__global__ void __launch_bounds__(kRwThreads)
    kv_read_w4_kernel(__nv_bfloat16* out, const uint8_t* codes, const uint32_t* scales, const long long* slot_map, int rows,
                      int NKV, int hs, long long slots, int block_size, int parts, int rows_per_cta) {
    const int per_row = 2 * NKV * hs / kReadChannels, part = blockIdx.x % parts;
    const RowPlace me = row_place(kReadChannels, hs, block_size, per_row, part, parts, rows_per_cta);
    pdl_wait();
    if (!me.active) return;
    const uint32_t page = (uint32_t)(2 * NKV) * block_size * (hs / kW4Group);
    const long long step = (long long)(gridDim.x / parts) * rows_per_cta, ld = (long long)per_row * kReadChannels;
    const uint8_t* my_codes = codes + (size_t)me.group * (kW4Group / 2) + (me.col & (kW4Group - 1)) / 2;
    const uint32_t* my_scales = scales + me.group;
    const unsigned eight = 0xffu << (threadIdx.x & 24);
    for (long long base = (long long)(blockIdx.x / parts) * rows_per_cta + me.row; base < rows; base += 8 * step) {
        const long long ahead = base + (threadIdx.x & 7) * step;
        const uint32_t place =
            ahead < rows ? slot_group(slot_map[ahead], slots, block_size, hs / kW4Group, page) : kNoRow;
        __nv_bfloat16* row = out + base * ld + me.col;
        const int n = (int)min(8ll, (rows - base + step - 1) / step);
        for (int k0 = 0; k0 < n; k0 += kReadAhead) {
            uint32_t word[kReadAhead], meta[kReadAhead];
#pragma unroll
            for (int k = 0; k < kReadAhead; k++) {
                const uint32_t at = __shfl_sync(eight, place, k0 + k, 8);
                word[k] = meta[k] = 0u;  // code 0, step 0, low end 0: zeros
                if (at != kNoRow) {
                    word[k] = *reinterpret_cast<const uint32_t*>(my_codes + (size_t)at * (kW4Group / 2));
                    meta[k] = my_scales[at];
                }
            }
#pragma unroll
            for (int k = 0; k < kReadAhead; k++) {
                if (k0 + k < n) {
                    float x[8];
                    w4_values(word[k], meta[k], x);
                    uint32_t r[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                        r[i] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    *reinterpret_cast<uint4*>(row) = make_uint4(r[0], r[1], r[2], r[3]);
                }
                row += step * ld;
            }
        }
    }
}

// CTAs of a row pass: `parts` CTAs share a wide row, or a CTA takes `rows_per_cta` narrow ones; as many passes at
// once as the rows give `ahead` each, at most 4 CTAs an SM (what the append's registers allow: one wave; with 8
// append and read-back of 16384 rows took 42.9 us together, with 4 41.3).
struct RowGrid {
    int parts, rows_per_cta, grid;
};
static RowGrid row_grid(int rows, int NKV, int hs, int channels, int ahead) {
    const int per_row = 2 * NKV * hs / channels;
    RowGrid g;
    g.parts = (per_row + kRwThreads - 1) / kRwThreads;
    g.rows_per_cta = g.parts > 1 ? 1 : kRwThreads / per_row;
    // few rows: a pass each, so that all of them are on their way at once
    long long passes = (rows + g.rows_per_cta - 1) / g.rows_per_cta;
    const long long most = (long long)sm_count() * 4 / g.parts;
    if (passes > most) passes = (passes + ahead - 1) / ahead;
    if (passes > most) passes = most;
    if (passes < 1) passes = 1;
    g.grid = (int)(passes * g.parts);
    return g;
}

}  // namespace gpt2b

using namespace gpt2b;

extern "C" {

int gpt2b_kv_block_tables(int* block_table, long long* slot_map, int* positions, int* row_start, int* seq_lens,
                          int* blocks_out, int* free_left, const int* ctx_lens, const int* new_lens,
                          const int* blocks_have, const int* free_list, const int* free_count, int B, int max_blocks,
                          int block_size, int max_rows, int free_cap, gpt2b_stream_t stream) {
    if (B <= 0 || max_blocks <= 0 || block_size <= 0 || max_rows < 0 || free_cap < 0) return GPT2B_ERR_INVALID_ARG;
    if (!block_table || !row_start || !seq_lens || !blocks_out || !free_left || !ctx_lens || !new_lens || !blocks_have ||
        !free_count)
        return GPT2B_ERR_INVALID_ARG;
    if ((max_rows > 0 && (!slot_map || !positions)) || (free_cap > 0 && !free_list)) return GPT2B_ERR_INVALID_ARG;
    if (B > kTableMaxRequests || (long long)max_blocks * block_size > INT_MAX) return GPT2B_ERR_UNSUPPORTED;
    // every CTA reads the inputs while others write
    const size_t b4 = 4 * (size_t)B, r = (size_t)max_rows;
    if (outputs_overlap({{block_table, b4 * max_blocks}, {slot_map, 8 * r}, {positions, 4 * r}, {row_start, b4 + 4},
                         {seq_lens, b4}, {blocks_out, b4}, {free_left, 4}},
                        {{ctx_lens, b4}, {new_lens, b4}, {blocks_have, b4}, {free_list, 4 * (size_t)free_cap}, {free_count, 4}}))
        return GPT2B_ERR_INVALID_ARG;
    TableArgs a{block_table, slot_map, positions, row_start, seq_lens, blocks_out, free_left, ctx_lens, new_lens,
                blocks_have, free_list, free_count, B, max_blocks, block_size, max_rows, free_cap};
    static unsigned long long mask = 0;  // 4096 requests take 48 KB
    if (const cudaError_t e = ensure_smem_limit(block_tables_kernel, &mask)) return status_from(e);
    long long grid = ((long long)max_rows + kTabThreads - 1) / kTabThreads;  // a row a thread, up to 2 CTAs an SM
    if (grid < 1) grid = 1;
    if (grid > 2 * sm_count()) grid = 2 * sm_count();
    return status_from(launch_k(block_tables_kernel, dim3((unsigned)grid), dim3(kTabThreads), 3 * sizeof(int) * (size_t)B,
                                (cudaStream_t)stream, true, a));
}

static int w4_check(const void* codes, const void* scales, int NKV, int hs, int num_blocks, int block_size) {
    if (NKV <= 0 || num_blocks <= 0 || block_size <= 0 || !codes || !scales) return GPT2B_ERR_INVALID_ARG;
    if ((hs != 64 && hs != 128) || block_size % kW4Tile != 0) return GPT2B_ERR_UNSUPPORTED;
    if (!aligned16(codes) || !aligned16(scales)) return GPT2B_ERR_ALIGNMENT;
    return GPT2B_OK;
}

// a block's bytes and the cache's groups of 64 channels are counted in 32 bits
static bool w4_too_large(int NKV, int hs, int num_blocks, int block_size) {
    const long long block = (long long)NKV * block_size * hs;
    return block > INT_MAX || block / (kW4Group / 2) * num_blocks >= (long long)kNoRow;
}

// bytes of a cache's codes; its steps take an eighth
static size_t w4_code_bytes(int NKV, int hs, int num_blocks, int block_size) {
    return (size_t)NKV * block_size * hs * num_blocks;
}

int gpt2b_kv_cache_write_w4(uint8_t* kv_cache, uint16_t* kv_scale, const uint16_t* qkv, const long long* slot_map, int rows,
                            int NH, int NKV, int hs, int ld, int num_blocks, int block_size, gpt2b_stream_t stream) {
    int rc = w4_check(kv_cache, kv_scale, NKV, hs, num_blocks, block_size);
    if (rc) return rc;
    if (rows < 0 || NH <= 0 || (rows > 0 && (!qkv || !slot_map))) return GPT2B_ERR_INVALID_ARG;
    if (((long long)NH + 2ll * NKV) * hs > ld) return GPT2B_ERR_INVALID_ARG;
    if (w4_too_large(NKV, hs, num_blocks, block_size)) return GPT2B_ERR_UNSUPPORTED;
    if (!aligned16(qkv) || ld % 8 != 0) return GPT2B_ERR_ALIGNMENT;
    if (rows == 0) return GPT2B_OK;
    const size_t bytes = w4_code_bytes(NKV, hs, num_blocks, block_size);
    if (outputs_overlap({{kv_cache, bytes}, {kv_scale, bytes / 8}},
                        {{qkv, 2 * ((size_t)(rows - 1) * ld + ((size_t)NH + 2 * (size_t)NKV) * hs)}, {slot_map, 8 * (size_t)rows}}))
        return GPT2B_ERR_INVALID_ARG;
    const RowGrid g = row_grid(rows, NKV, hs, kWriteChannels, kWriteAhead);
    return status_from(launch_k(kv_write_w4_kernel, dim3(g.grid), dim3(kRwThreads), 0, (cudaStream_t)stream, true, kv_cache,
                                (uint32_t*)kv_scale, (const __nv_bfloat16*)qkv, slot_map, rows, NH, NKV, hs, ld,
                                (long long)num_blocks * block_size, block_size, g.parts, g.rows_per_cta));
}

int gpt2b_kv_cache_read_w4(uint16_t* out, const uint8_t* kv_cache, const uint16_t* kv_scale, const long long* slot_map,
                           int rows, int NKV, int hs, int num_blocks, int block_size, gpt2b_stream_t stream) {
    int rc = w4_check(kv_cache, kv_scale, NKV, hs, num_blocks, block_size);
    if (rc) return rc;
    if (rows < 0 || (rows > 0 && (!out || !slot_map))) return GPT2B_ERR_INVALID_ARG;
    if (w4_too_large(NKV, hs, num_blocks, block_size)) return GPT2B_ERR_UNSUPPORTED;
    if (!aligned16(out)) return GPT2B_ERR_ALIGNMENT;
    if (rows == 0) return GPT2B_OK;
    const size_t bytes = w4_code_bytes(NKV, hs, num_blocks, block_size);
    if (outputs_overlap({{out, 4 * (size_t)rows * NKV * hs}},
                        {{kv_cache, bytes}, {kv_scale, bytes / 8}, {slot_map, 8 * (size_t)rows}}))
        return GPT2B_ERR_INVALID_ARG;
    const RowGrid g = row_grid(rows, NKV, hs, kReadChannels, kReadAhead);
    return status_from(launch_k(kv_read_w4_kernel, dim3(g.grid), dim3(kRwThreads), 0, (cudaStream_t)stream, true,
                                (__nv_bfloat16*)out, kv_cache, (const uint32_t*)kv_scale, slot_map, rows, NKV, hs,
                                (long long)num_blocks * block_size, block_size, g.parts, g.rows_per_cta));
}

}  // extern "C"
