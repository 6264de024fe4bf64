// Rotary embedding of new query and key rows, and the append of keys and values to a
// paged cache (bf16, or E4M3 with one scale per page and KV head).
//
// Rotation: element d of a head, d < rot, becomes x[d] c[d] -+ x[pair(d)] s[d] in fp32 with
// separately rounded products; the pair of d is d ^ 1 ("interleaved") or d +- rot / 2
// ("half").  Elements from rot on pass unchanged.  One rounding at the store.
//
// The 8-bit cache.  A page's codes of one head share a scale 2^e with the smallest e that
// brings the largest finite magnitude of the page's rows under 448, E4M3's largest value
// (e is kept in [-64, 120]; what is larger saturates, infinities with it, NaN stays NaN).
// E4M3 is a floating format, so a coarser scale costs no significant bits, and a power of
// two lets a page's scale grow as rows arrive without a second rounding of the rows it holds:
// their codes are multiplied by a power of two, which is exact down to E4M3's subnormals.  A
// scale only grows while its page holds rows; the first row of a page starts afresh.
//
// Work split.  One CTA owns the rows that a call adds to one (page, KV head): its first half
// takes keys, its second values, 16 bytes of bf16 per thread and row, every row in registers
// between the magnitude's reduction and the store, so that each input is read once.  Pages of
// one sequence belong to nobody else, hence no atomics.  Query rows need no such grouping:
// a thread keeps the table's elements of its 8 columns and walks over heads of one token.

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "batched_ops.cuh"
#include "paged.cuh"

namespace mk {
namespace paged {

constexpr int kQueryHeads = 8;        // query heads of one token that a thread rotates with the same table elements
constexpr int kScaleMin = -64, kScaleMax = 120;

__device__ __forceinline__ uint4 pack_bf16(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 consecutive bf16 elements of a row (a linear's result is rounded to bf16: nothing is lost by keeping it so)
template <bool LIN>
__device__ __forceinline__ uint4 load8(const AppendParams &p, const Rows &r, int lin_col, int t, int head, int d) {
    if constexpr (LIN) {
        const int col = lin_col + head * p.pool.head_dim + d;
        const float4 a = bo::lin_value4(p.lin, t, col), b = bo::lin_value4(p.lin, t, col + 4);
        const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        return pack_bf16(x);
    } else {
        return __ldg(reinterpret_cast<const uint4 *>(r.p + t * r.token + head * r.head + d));
    }
}

__device__ __forceinline__ void load_table(const float *table, long long at, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(table + at)), b = __ldg(reinterpret_cast<const float4 *>(table + at) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// Rotates the 8 elements at column 8 * chunk.  `lane_chunk0`: lane of the row's first chunk.  All lanes of a warp call it.
__device__ __forceinline__ void rotate8(float (&x)[8], const float (&c)[8], const float (&s)[8], int chunk, int lane_chunk0, int rot,
                                        int half) {
    const bool inside = 8 * chunk < rot;
    if (half) {
        const int away = rot / 16;   // chunks between the two elements of a pair
        const bool second = chunk >= away;
        const int partner = lane_chunk0 + (inside ? (second ? chunk - away : chunk + away) : chunk);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_sync(0xffffffffu, x[i], partner);
            if (inside) x[i] = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(second ? other : -other, s[i]));
        }
    } else if (inside) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float a = x[i], b = x[i + 1];
            x[i] = __fadd_rn(__fmul_rn(a, c[i]), __fmul_rn(-b, s[i]));
            x[i + 1] = __fadd_rn(__fmul_rn(b, c[i + 1]), __fmul_rn(a, s[i + 1]));
        }
    }
}

__device__ __forceinline__ uint2 pack_e4m3(const float (&x)[8], float factor) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * factor, x[2 * i + 1] * factor), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

__device__ __forceinline__ uint2 recode_e4m3(uint2 codes, float factor) {
    float x[8];
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i % 2))), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
    return pack_e4m3(x, factor);
}

// Exponent of the smallest power of two that brings amax to 448 = 1.75 * 2^8 or less.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < kScaleMin ? kScaleMin : e > kScaleMax ? kScaleMax : e;
}

// The last sequence b of a ragged call with key(cu[b], b) <= x (keys grow with b).  One warp narrows 32
// intervals per step.
template <typename Key>
__device__ __forceinline__ int find_sequence(const Batch &bt, int x, Key key) {
    const int lane = threadIdx.x & 31;
    int lo = 0, size = bt.seqs;
    while (size > 1) {
        const int step = (size + 31) / 32, at = min(lo + lane * step, bt.seqs);
        const bool below = lane * step < size && key(clamp_int(__ldg(bt.cu + at), 0, bt.tokens), at) <= x;
        const int n = max(__popc(__ballot_sync(0xffffffffu, below)), 1) - 1;
        lo += n * step;
        size = min(step, size - n * step);
    }
    return lo;
}

// First page slot of a sequence of a ragged call whose rows begin at `first`: from one sequence to the next there
// are enough for every page its rows can touch, wherever in a page they start.
__device__ __forceinline__ int first_slot(const Batch &bt, int first, int b) { return (first >> bt.page_shift) + 2 * b; }

// D: head dimension.  ITERS: rows of one page that a thread may hold.
template <int D, int THREADS, int ITERS, bool FP8, bool LIN>
__global__ void __launch_bounds__(THREADS, 768 / THREADS)   // 80 registers: 64 spill (7 prompts 74 us instead of 65), 128 leave too few threads (77)
append_kernel(const AppendParams p) {
    pdl_wait();   // and no early start for the next kernel: see paged.cuh
    constexpr int kLanes = D / 8;                          // threads per row
    constexpr int kHalf = THREADS / 2, kHalfWarps = kHalf / 32;
    constexpr int kRows = kHalf / kLanes;                  // rows per pass of half a CTA
    __shared__ float amax_s[2 * kHalfWarps];
    const Batch &bt = p.bt;
    const int lane = threadIdx.x & 31, chunk = threadIdx.x % kLanes, lane0 = lane - chunk;
    const bool rope = p.rope_cos != nullptr;
    // table elements of a position for this thread's columns
    auto tables = [&](long long want, bool live, float (&c)[8], float (&s)[8]) {
        const int pos = clamp_int(want, 0, p.positions - 1);
        if (live && pos != want) atomicOr(bt.error, kErrorIndex);
        if (8 * chunk < p.rot) {
            load_table(p.rope_cos, (long long)pos * p.rot + 8 * chunk, c);
            load_table(p.rope_sin, (long long)pos * p.rot + 8 * chunk, s);
        }
    };

    if ((int)blockIdx.x >= p.kv_blocks) {                  // query rows: one token, kQueryHeads heads per thread
        constexpr int kUnits = THREADS / kLanes;           // (token, group of heads) pairs per CTA
        const int groups = (p.hq + kQueryHeads - 1) / kQueryHeads;
        const long long unit0 = (long long)((int)blockIdx.x - p.kv_blocks) * kUnits, unit = unit0 + threadIdx.x / kLanes;
        int t = (int)(unit / groups);
        const int head0 = (int)(unit % groups) * kQueryHeads;
        bool live = t < bt.tokens;
        t = min(t, bt.tokens - 1);
        uint4 raw[kQueryHeads];
#pragma unroll
        for (int i = 0; i < kQueryHeads; ++i) raw[i] = head0 + i < p.hq ? load8<LIN>(p, p.q, 0, t, head0 + i, 8 * chunk) : make_uint4(0u, 0u, 0u, 0u);
        int b;
        if (bt.cu) {
            b = find_sequence(bt, (int)(unit0 / groups), [](int first, int) { return first; });
            while (b + 1 < bt.seqs && __ldg(bt.cu + b + 1) <= t) ++b;
        } else {
            b = t / bt.per_seq;
        }
        int first, count;
        rows_of(bt, b, first, count);
        const int start = __ldg(bt.where + b);
        live = live && start >= 0 && t >= first && t < first + count;   // idle sequences' rows stay as they were
        float c[8] = {}, s[8] = {};
        if (rope) tables((long long)start + (t - first), live, c, s);
#pragma unroll
        for (int i = 0; i < kQueryHeads; ++i) {
            float x[8];
            unpack8(raw[i], x);
            if (rope) rotate8(x, c, s, chunk, lane0, p.rot, p.half);
            if (live && head0 + i < p.hq)
                *reinterpret_cast<uint4 *>(p.q_out + ((long long)t * p.hq + head0 + i) * D + 8 * chunk) = pack_bf16(x);
        }
        return;
    }

    // keys and values of one (page, KV head)
    const int hkv = p.pool.kv_heads, page_size = 1 << bt.page_shift;
    const int slot = blockIdx.x / hkv, head = blockIdx.x % hkv;
    const bool is_v = threadIdx.x >= kHalf;
    const int row_in_pass = (threadIdx.x % kHalf) / kLanes;
    int b, ordinal;
    if (bt.cu) {
        b = find_sequence(bt, slot, [&](int first, int at) { return first_slot(bt, first, at); });
        ordinal = slot - first_slot(bt, clamp_int(__ldg(bt.cu + b), 0, bt.tokens), b);
    } else {
        b = slot / p.slots;
        ordinal = slot % p.slots;
    }
    int first, count;
    rows_of(bt, b, first, count);
    const int start = __ldg(bt.where + b);
    if (start < 0) return;                                 // idle sequence
    const long long column = (long long)(start >> bt.page_shift) + ordinal;
    const long long page_begin = column << bt.page_shift;
    if (page_begin >= (long long)start + count) return;    // the sequence's rows end before this slot's page
    if (column >= bt.max_pages) {
        if (threadIdx.x == 0) atomicOr(bt.error, kErrorIndex);
        return;
    }
    const int held = page_begin < start ? (int)(start - page_begin) : 0;   // rows in the page before this call
    const int end = (int)min((long long)page_size, (long long)start + count - page_begin);
    const int added = end - held;
    const int t0 = first + (int)(page_begin + held - start);               // token row of the page's first new row

    const int page = __ldg(bt.table + b * bt.table_stride + column);
    uint4 raw[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        if (it * kRows < added) {
            const int t = t0 + min(it * kRows + row_in_pass, added - 1);   // repeated rows change nothing
            raw[it] = is_v ? load8<LIN>(p, p.v, (p.hq + hkv) * D, t, head, 8 * chunk) : load8<LIN>(p, p.k, p.hq * D, t, head, 8 * chunk);
        }
    }
    if (page < 0) return;                                  // no page: nothing is kept
    if (page >= bt.num_pages) {
        if (threadIdx.x == 0) atomicOr(bt.error, kErrorIndex);
        return;
    }
    // row `it` of this thread in fp32, keys rotated
    auto value = [&](int it, float (&x)[8]) {
        unpack8(raw[it], x);
        if (rope && !is_v) {
            float c[8] = {}, s[8] = {};
            tables(page_begin + held + min(it * kRows + row_in_pass, added - 1), true, c, s);
            rotate8(x, c, s, chunk, lane0, p.rot, p.half);
        }
    };
    const long long base = page * p.pool.page_stride + head * p.pool.head_stride + 8 * chunk;
    if constexpr (!FP8) {
        bf16 *dst = reinterpret_cast<bf16 *>(is_v ? p.pool.v : p.pool.k) + base;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            if (it * kRows < added) {
                const int i = it * kRows + row_in_pass;
                float x[8];
                value(it, x);
                if (i < added) *reinterpret_cast<uint4 *>(dst + (held + i) * p.pool.slot_stride) = pack_bf16(x);
            }
        }
    } else {
        // The rotation is done twice, for the magnitude and for the store, where a thread holds many rows: their fp32
        // values would cost twice the registers, and the tables' elements are in L1 by then.
        constexpr bool kKeep = ITERS <= 2;
        float kept[kKeep ? ITERS : 1][8];
        float amax = 0.f;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            if (it * kRows < added) {
                float (&x)[8] = kept[kKeep ? it : 0];
                value(it, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float a = fabsf(x[j]);
                    if (a < INFINITY) amax = fmaxf(amax, a);
                }
            }
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        if (lane == 0) amax_s[threadIdx.x >> 5] = amax;
        float *scales = (is_v ? p.pool.v_scales : p.pool.k_scales) + (long long)page * hkv + head;
        const float old = held > 0 ? *scales : 0.f;
        __syncthreads();                                       // after every thread's read of the scale, too
        amax = 0.f;
#pragma unroll
        for (int w = 0; w < kHalfWarps; ++w) amax = fmaxf(amax, amax_s[(is_v ? kHalfWarps : 0) + w]);
        const float need = __uint_as_float((uint32_t)(scale_exponent(amax) + 127) << 23);
        const float scale = fmaxf(old, need);
        uint8_t *dst = reinterpret_cast<uint8_t *>(is_v ? p.pool.v : p.pool.k) + base;
        if (held > 0 && scale != old) {                        // the page's scale grew: its rows are coded anew
            const float factor = old / scale;
#pragma unroll 4
            for (int i = row_in_pass; i < held; i += kRows) {
                uint2 *at = reinterpret_cast<uint2 *>(dst + i * p.pool.slot_stride);
                *at = recode_e4m3(*at, factor);
            }
        }
        if (threadIdx.x % kHalf == 0) *scales = scale;
        const float inverse = 1.0f / scale;                    // exact: a power of two
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            if (it * kRows < added) {
                const int i = it * kRows + row_in_pass;
                float (&x)[8] = kept[kKeep ? it : 0];
                if constexpr (!kKeep) value(it, x);
                if (i < added) *reinterpret_cast<uint2 *>(dst + (held + i) * p.pool.slot_stride) = pack_e4m3(x, inverse);
            }
        }
    }
}

template <int D, int THREADS, int ITERS, bool FP8, bool LIN>
static cudaError_t launch_append_t(AppendParams &p, long long kv, cudaStream_t st) {
    const int groups = (p.hq + kQueryHeads - 1) / kQueryHeads, per_cta = THREADS * 8 / D;
    const long long q = p.q_out ? ((long long)p.bt.tokens * groups + per_cta - 1) / per_cta : 0;
    if (kv + q > 0x7fffffff) return cudaErrorInvalidConfiguration;
    p.kv_blocks = (int)kv;
    return launch_pdl(append_kernel<D, THREADS, ITERS, FP8, LIN>, dim3((unsigned)(kv + q)), dim3(THREADS), 0, st, p);
}

template <int D, bool FP8, bool LIN>
static cudaError_t launch_append_d(AppendParams &p, long long kv, int rows, cudaStream_t st) {
    // A few rows per page (decoding): a warp each for keys and values, so that every CTA of a large batch is resident at
    // once (128 sequences x 8 heads: 12.7 us with the wide CTAs below, 4 with these).
    constexpr int kFew = 32 * 8 / D;   // rows of one pass of a warp
    if (rows <= kFew) return launch_append_t<D, 64, 1, FP8, LIN>(p, kv, st);
    if (rows <= 2 * kFew) return launch_append_t<D, 64, 2, FP8, LIN>(p, kv, st);
    switch (p.pool.page_size * D / 1024) {
    case 1: return launch_append_t<D, 256, 1, FP8, LIN>(p, kv, st);
    case 2: return launch_append_t<D, 256, 2, FP8, LIN>(p, kv, st);
    case 4: return launch_append_t<D, 256, 4, FP8, LIN>(p, kv, st);
    case 8: return launch_append_t<D, 256, 8, FP8, LIN>(p, kv, st);
    case 16: return launch_append_t<D, 256, 16, FP8, LIN>(p, kv, st);
    default: return cudaErrorInvalidValue;
    }
}

template <bool LIN>
static cudaError_t launch_append_l(AppendParams &p, cudaStream_t st) {
    const Batch &bt = p.bt;
    const int page = p.pool.page_size, most = bt.cu ? bt.tokens : bt.per_seq;
    long long slots;
    if (bt.cu) {
        slots = bt.tokens / page + 2ll * bt.seqs;
        p.slots = 0;
    } else {
        p.slots = bt.per_seq == 1 ? 1 : (bt.per_seq - 1) / page + 2;
        slots = (long long)p.slots * bt.seqs;
    }
    const long long kv = slots * p.pool.kv_heads;
    const int rows = most < page ? most : page;
    if (p.pool.head_dim == 64)
        return p.pool.fp8 ? launch_append_d<64, true, LIN>(p, kv, rows, st) : launch_append_d<64, false, LIN>(p, kv, rows, st);
    return p.pool.fp8 ? launch_append_d<128, true, LIN>(p, kv, rows, st) : launch_append_d<128, false, LIN>(p, kv, rows, st);
}

cudaError_t launch_append(AppendParams p, cudaStream_t st) {
    return p.from_linear ? launch_append_l<true>(p, st) : launch_append_l<false>(p, st);
}

}  // namespace paged
}  // namespace mk
