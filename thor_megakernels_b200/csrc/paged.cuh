// Paged KV cache: what the append and attention kernels share - the description of
// a cache and of a ragged batch of sequences on it, and the arithmetic that deals
// attention work out to CTAs.  The latter is plain integer code for host and device.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200_megakernel.h"
#include "batched_ops.cuh"
#include "mk_device.cuh"

namespace mk {
namespace paged {

constexpr int kErrorWait = 1;    // a bounded wait ran out
constexpr int kErrorIndex = 2;   // a page id, position, length or row offset was outside its tensor

// Sequences of a call.  `cu` (optional) holds seqs + 1 row offsets into the token rows; without
// it every sequence has `per_seq` rows.
struct Batch {
    const int *table;     // [seqs, table_stride] page ids; negative: no page
    long long table_stride;
    const int *where;     // append: first position of the new rows (negative: idle); attention: length with the new rows
    const int *cu;
    int seqs, tokens, per_seq;
    int max_pages;        // columns of the table
    int num_pages;
    int page_shift;       // log2 of the page size
    int where_offset;     // attention: added to `where` (a caller that has the position of the last row but one keeps no second array)
    int *error;
};

__host__ __device__ inline int clamp_int(long long v, int low, int high) {
    return v < low ? low : v > high ? high : (int)v;
}

// Rows of sequence b: [first, first + count).  Offsets come from device memory and are held inside the tensor.
__device__ __forceinline__ void rows_of(const Batch &bt, int b, int &first, int &count) {
    if (bt.cu == nullptr) {
        first = b * bt.per_seq;
        count = bt.per_seq;
        return;
    }
    const int lo = __ldg(bt.cu + b), hi = __ldg(bt.cu + b + 1);
    first = clamp_int(lo, 0, bt.tokens);
    count = clamp_int(hi, first, bt.tokens) - first;
    if (first != lo || first + count != hi) atomicOr(bt.error, kErrorIndex);
}

// Most positions of a sequence that attention counts: the position behind any tile that is looked ahead to is an int.
constexpr int kMostPositions = 0x7fff0000;

__host__ __device__ inline int held_length(long long length, int max_pages, int page_shift) {
    return clamp_int(length, 0, clamp_int((long long)max_pages << page_shift, 0, kMostPositions));
}

// Cached length of sequence b, held inside its page table.
__device__ __forceinline__ int length_of(const Batch &bt, int b) {
    const long long len = (long long)__ldg(bt.where + b) + bt.where_offset;
    const int held = held_length(len, bt.max_pages, bt.page_shift);
    if (len > held) atomicOr(bt.error, kErrorIndex);
    return held;
}

// ---------------------------------------------------------------------------
// attention work
// ---------------------------------------------------------------------------
// A row block is `rows` consecutive (query token, query head of the group) pairs of one
// sequence and KV head: pair r is token r / group, head r % group.  It attends the positions
// its last token sees, tile by tile.  CTAs take equal consecutive ranges of units (tiles, and
// a few for every row block's fixed cost), so that sequences of any lengths finish together
// without the host knowing the lengths.

// Division of numbers below 2^31 by one that a launch knows: q = (mulhi(x, mul) + x) >> shift.
struct FastDiv {
    int d;
    uint32_t mul, shift;
};
inline FastDiv fast_div(int d) {
    FastDiv f = {d, 0, 0};
    while ((1ll << f.shift) < d) ++f.shift;
    f.mul = (uint32_t)((((1ull << f.shift) - (uint64_t)d) << 32) / (uint64_t)d + 1);
    return f;
}
__host__ __device__ inline int div(int x, const FastDiv &f) {
#ifdef __CUDA_ARCH__
    const uint32_t high = __umulhi((uint32_t)x, f.mul);
#else
    const uint32_t high = (uint32_t)(((uint64_t)(uint32_t)x * f.mul) >> 32);
#endif
    return (int)((high + (uint32_t)x) >> f.shift);
}

// Positions that query token i of `count` sees in a cache of `length` positions (the new tokens are its last ones).
__host__ __device__ inline int visible(int length, int count, int i) {
    const int v = length - count + i + 1;
    return v < 0 ? 0 : v > length ? length : v;
}

__host__ __device__ inline int block_count(int count, int group, int rows) { return (count * group + rows - 1) / rows; }

// Tiles that row block rb has to look at: those its last token sees.
__host__ __device__ inline int block_tiles(int length, int count, const FastDiv &group, int rows, int rb, int tile) {
    int last = div((rb + 1) * rows - 1, group);
    if (last > count - 1) last = count - 1;
    return (visible(length, count, last) + tile - 1) / tile;
}

// How a kernel cuts its work: rows per row block, positions per tile, and what a segment costs besides its
// tiles (queries, the first copies' latency, the merge), in tiles.
struct Cut {
    int rows, tile, extra;
};

// Units of one (row block, KV head): its tiles behind `extra` units that stand for the fixed cost.  A block
// that sees nothing still counts one tile: its output rows have to be written.
__host__ __device__ inline int block_units(int length, int count, const FastDiv &group, const Cut &cut, int rb) {
    const int t = block_tiles(length, count, group, cut.rows, rb, cut.tile);
    return (t > 0 ? t : 1) + cut.extra;
}

__host__ __device__ inline int sequence_units(int length, int count, const FastDiv &group, const Cut &cut, int kv_heads) {
    const int blocks = block_count(count, group.d, cut.rows);
    long long total = 0;
    for (int rb = 0; rb < blocks; ++rb) total += block_units(length, count, group, cut, rb);
    total *= kv_heads;
    return total > 0x7fffffff ? 0x7fffffff : (int)total;
}

// The CTAs that get work: never more than there are units, so that the owners of a segment's units are
// consecutive.
__host__ __device__ inline int working_ctas(int ctas, int units) { return ctas < units ? ctas : units; }
// CTA c of `ctas` working ones takes units [first_unit(c), first_unit(c + 1)); unit u belongs to CTA owner(u).
__host__ __device__ inline int first_unit(int c, int ctas, int units) { return (int)((long long)c * units / ctas); }
__host__ __device__ inline int owner(int u, int ctas, int units) { return (int)((((long long)u + 1) * ctas - 1) / units); }

// Where unit u lies in a sequence: row block, head and offset in their units.  `rb` and `base` (the row block's
// first unit) start at a row block at or before it and are left at its own.
struct Place {
    int head, offset, units;
};
__host__ __device__ inline Place place_of(int u, int &rb, int &base, int length, int count, const FastDiv &group, const Cut &cut, int kv_heads) {
    Place p;
    while (true) {
        p.units = block_units(length, count, group, cut, rb);
        if (u - base < p.units * kv_heads) break;
        base += p.units * kv_heads;
        ++rb;
    }
    p.head = (u - base) / p.units;
    p.offset = (u - base) - p.head * p.units;
    return p;
}

// A CTA's share of one (row block, KV head).  Segments that several CTAs share are joined by another kernel:
// a CTA leaves what begins in its range but does not end there in its part 1, what it continues in its part 0,
// and the CTA a segment begins in describes it (its parts are that CTA's part 1 and the part 0 of the next ones).
struct Segment {
    int b, first, count, length;   // sequence, its rows, its cached positions
    int rb, head, rows;            // row block, KV head, rows of the block
    int tile0, tile1;              // tiles of this share
    bool begins, ends;
    int parts;                     // CTAs that share the segment (where it begins here)
};

// One for each CTA of the grid: a segment that begins in its range and ends in a later one's.
struct __align__(16) JoinEntry {
    int parts;       // 0: none
    int row;         // first token row of the sequence
    int pair;        // first (token, head of the group) pair of the row block
    int head_rows;   // KV head << 16 | rows
};

struct Walk {
    const int *prefix;   // units of the sequences before each one
    int u, u_end, ctas, units;
    int b, rb, base;     // the last segment's sequence and row block, and the row block's first unit
    int first, count, length;   // of that sequence
};

// The CTA's next segment; false at the end of its range.
__device__ __forceinline__ bool next_segment(const Batch &bt, int kv_heads, const FastDiv &group, const Cut &cut, Walk &w, Segment &s) {
    while (w.u < w.u_end) {
        int lo = max(w.b, 0), hi = bt.seqs - 1;   // the last sequence that starts at or before u
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (w.prefix[mid] <= w.u) lo = mid;
            else hi = mid - 1;
        }
        if (lo != w.b) {
            w.b = lo;
            w.rb = 0;
            w.base = w.prefix[lo];
            rows_of(bt, lo, w.first, w.count);
            w.length = length_of(bt, lo);
        }
        s.first = w.first;
        s.count = w.count;
        s.length = w.length;
        const Place p = place_of(w.u, w.rb, w.base, s.length, s.count, group, cut, kv_heads);
        const int take = p.units - p.offset < w.u_end - w.u ? p.units - p.offset : w.u_end - w.u;
        const int end = w.u - p.offset + p.units;   // of the segment's units
        w.u += take;
        s.tile0 = max(p.offset - cut.extra, 0);
        s.tile1 = max(p.offset + take - cut.extra, 0);
        if (s.tile1 == s.tile0) continue;           // only of the fixed cost: the next CTA begins the segment
        s.b = lo;
        s.rb = w.rb;
        s.head = p.head;
        s.rows = min(cut.rows, s.count * group.d - w.rb * cut.rows);
        s.begins = s.tile0 == 0;
        s.ends = w.u == end;
        s.parts = s.begins && !s.ends ? owner(end - 1, w.ctas, w.units) - (int)blockIdx.x + 1 : 1;
        return true;
    }
    return false;
}

// Sum of two counts, held at the largest int.
__device__ __forceinline__ int add_held(int a, int b) { return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu); }

// Fills prefix [seqs + 1] in shared memory with the units before each sequence of those that have between
// min_count and max_count new rows, and sets up the CTA's walk.  All THREADS threads call it.
template <int THREADS>
__device__ __forceinline__ void plan_walk(const Batch &bt, int kv_heads, const FastDiv &group, const Cut &cut, int min_count, int max_count, int *prefix,
                                          int *scan, Walk &w) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (bt.seqs + THREADS - 1) / THREADS;
    const int b0 = min((int)threadIdx.x * per, bt.seqs), b1 = min(b0 + per, bt.seqs);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
        int first, count;
        rows_of(bt, b, first, count);
        const int length = length_of(bt, b);
        const int n = count < min_count || count > max_count ? 0 : sequence_units(length, count, group, cut, kv_heads);
        prefix[b + 1] = n;
        sum = add_held(sum, n);
    }
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl = add_held(incl, v);
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int before = incl - sum, total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        if (i == warp) before += total;
        total = add_held(total, scan[i]);
    }
    // Row offsets that do not grow can give rows to many sequences at once, more than the host counted on: no work then.
    const bool refused = total == 0x7fffffff;
    if (refused && threadIdx.x == 0) atomicOr(bt.error, kErrorIndex);
    for (int b = b0; b < b1; ++b) {
        before += prefix[b + 1];
        prefix[b + 1] = refused ? 0 : before;
    }
    if (threadIdx.x == 0) prefix[0] = 0;
    __syncthreads();
    w.prefix = prefix;
    w.b = -1;
    w.units = prefix[bt.seqs];
    w.ctas = working_ctas(gridDim.x, w.units);
    const bool works = (int)blockIdx.x < w.ctas;
    w.u = works ? first_unit(blockIdx.x, w.ctas, w.units) : 0;
    w.u_end = works ? first_unit(blockIdx.x + 1, w.ctas, w.units) : 0;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

// Lets `kernel` use as much shared memory as a device has (once per device and kernel: `done` is the kernel's own).
inline cudaError_t allow_smem(const void *kernel, bool (&done)[64]) {
    int device = 0, most = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && done[device])) return e;
    e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)attr.sharedSizeBytes);
    if (e == cudaSuccess && device < 64) done[device] = true;
    return e;
}

// The small kernels of this family (append, the joins) do not let the next kernel start early.  The attention
// kernels fill an SM's registers exactly; a CTA that finds even one small neighbour there leaves a gap that the last
// CTA of the SM does not fit into, and that CTA then runs after all the others: 128 sequences of up to 4096
// positions took 154 us instead of 111.

struct Pool {
    void *k, *v;
    float *k_scales, *v_scales;                          // [num_pages, kv_heads]; null for a bf16 cache
    long long page_stride, head_stride, slot_stride;     // elements
    int num_pages, page_size, kv_heads, head_dim;
    bool fp8;
};

struct Rows {                           // bf16 rows [token][head][dim] at any token and head pitch (elements)
    const bf16 *p;
    long long token, head;
};

struct AppendParams {
    Batch bt;
    Rows q, k, v;
    bo::LinOut lin;                     // instead of q, k, v: one linear's result [tokens, (Hq + 2 Hkv) D], split-K sums not added yet
    bool from_linear;
    bf16 *q_out;                        // [tokens, Hq, D]
    const float *rope_cos, *rope_sin;   // [positions, rot] or null (no rotation)
    int rot, positions, half;
    Pool pool;
    int hq;
    FastDiv slots, per_seq;             // page slots and tokens per sequence (without cu)
    FastDiv kv_heads, q_groups;         // groups of query heads per token
    int kv_blocks;                      // CTAs that store keys and values; the rest rotate queries
};
cudaError_t launch_append(AppendParams p, cudaStream_t st);

struct AttentionParams {
    Batch bt;                           // where: cached length of a sequence, its new tokens included
    const bf16 *q;                      // [tokens, Hq, D] at any token and head pitch
    long long q_token, q_head;
    bf16 *out;                          // [tokens, Hq, D]
    const float *k_scales, *v_scales;   // [pages, Hkv] (8-bit cache)
    int hq, hkv;
    FastDiv group;                      // query heads per KV head
    int max_count;                      // sequences with more new tokens than this are another kernel's
    float scale_log2e;                  // score scale times log2 e
    float *partial;                     // workspace: 2 parts per CTA
    JoinEntry *entries;                 // workspace: one per CTA
};
// Pool and batch of a call from the public structs, or an error code (and its text) where they do not fit together.
int read_cache(const MkPagedCache &c, const MkPagedBatch &b, int max_seqs, Pool &pool, Batch &bt, const char *who);
// bytes of workspace; negative: more work than the kernels count
long long attention_workspace(const Batch &bt, const Pool &pool, int hq, int sms);
// fills the workspace pointers and max_count of p
int launch_attention(AttentionParams p, const Pool &pool, void *workspace, int sms, cudaStream_t st);

}  // namespace paged
}  // namespace mk
