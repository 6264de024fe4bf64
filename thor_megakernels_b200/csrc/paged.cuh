// Paged KV cache: what the append and attention kernels share - the description of
// a cache and of a ragged batch of sequences on it, and the arithmetic that deals
// attention work out to CTAs.  The latter is plain integer code for host and device.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

// Cached length of sequence b, held inside its page table.
__device__ __forceinline__ int length_of(const Batch &bt, int b) {
    const int len = __ldg(bt.where + b);
    const int held = clamp_int(len, 0, clamp_int((long long)bt.max_pages << bt.page_shift, 0, 0x7fffffff));
    if (len > held) atomicOr(bt.error, kErrorIndex);
    return held;
}

// ---------------------------------------------------------------------------
// attention work
// ---------------------------------------------------------------------------
// A row block is `rows` consecutive (query token, query head of the group) pairs of one
// sequence and KV head: pair r is token r / group, head r % group.  It attends the positions
// its last token sees.  A unit is one tile of `tile` cache positions of one (row block, KV head).

// Positions that query token i of `count` sees in a cache of `length` positions (the new tokens are its last ones).
__host__ __device__ inline int visible(int length, int count, int i) {
    const int v = length - count + i + 1;
    return v < 0 ? 0 : v > length ? length : v;
}

__host__ __device__ inline int block_count(int count, int group, int rows) { return (count * group + rows - 1) / rows; }

// Tiles that row block rb has to look at: those its last token sees.
__host__ __device__ inline int block_tiles(int length, int count, int group, int rows, int rb, int tile) {
    int last = ((rb + 1) * rows - 1) / group;
    if (last > count - 1) last = count - 1;
    return (visible(length, count, last) + tile - 1) / tile;
}

// Units of one sequence.  A block that sees nothing still counts one tile: its output rows have to be written.
__host__ __device__ inline int sequence_units(int length, int count, int group, int rows, int tile, int kv_heads) {
    const int blocks = block_count(count, group, rows);
    long long total = 0;
    for (int rb = 0; rb < blocks; ++rb) {
        const int t = block_tiles(length, count, group, rows, rb, tile);
        total += t > 0 ? t : 1;
    }
    total *= kv_heads;
    return total > 0x7fffffff ? 0x7fffffff : (int)total;
}

// The CTAs that get work: never more than there are units, so that each has one and the owners of a
// segment's units are consecutive.
__host__ __device__ inline int working_ctas(int ctas, int units) { return ctas < units ? ctas : units; }
// CTA c of `ctas` working ones takes units [first_unit(c), first_unit(c + 1)); unit u belongs to CTA owner(u).
__host__ __device__ inline int first_unit(int c, int ctas, int units) { return (int)((long long)c * units / ctas); }
__host__ __device__ inline int owner(int u, int ctas, int units) { return (int)((((long long)u + 1) * ctas - 1) / units); }

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

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
    int slots;                          // page slots per sequence (without cu)
    int kv_blocks;                      // CTAs that store keys and values; the rest rotate queries
};
cudaError_t launch_append(AppendParams p, cudaStream_t st);

struct AttentionParams {
    Batch bt;                           // where: cached length of a sequence, its new tokens included
    const bf16 *q;                      // [tokens, Hq, D] at any token and head pitch
    long long q_token, q_head;
    bf16 *out;                          // [tokens, Hq, D]
    const float *k_scales, *v_scales;   // [pages, Hkv] (8-bit cache)
    int hq, hkv, group;
    int max_count;                      // sequences with more new tokens than this are another kernel's
    float scale_log2e;                  // score scale times log2 e
    float *partial;                     // workspace: 2 parts per CTA of [rows, D + 2]
    int *prefix_out;                    // workspace: [seqs + 1] units before each sequence
};
// bytes of workspace; negative: more work than the kernels count
long long attention_workspace(const Batch &bt, const Pool &pool, int hq, int sms);
// fills the workspace pointers and max_count of p
int launch_attention(AttentionParams p, const Pool &pool, void *workspace, int sms, cudaStream_t st);

}  // namespace paged
}  // namespace mk
