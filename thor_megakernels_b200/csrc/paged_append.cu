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
// Work split.  One CTA owns the keys or the values that a call adds to one (page, KV head), 16 bytes of
// bf16 per thread and row; every row stays in registers between the magnitude's reduction and the store, so
// that each input is read once.  Pages of one sequence belong to nobody else, hence no atomics.  Query rows
// need no such grouping: a thread keeps the table's elements of its 8 columns for a few heads of one token.
//
// What bounds it.  Prompts (7 of 601 to 2100 rows, 32 query and 8 KV heads, D = 128, E4M3): 47 us on the device,
// 4.8 TB/s.  The query rows alone run at the copy bandwidth; keys and values take half of the time for a
// quarter of the bytes, waiting for one load after the other (sequence, start, page, tables).  With products and
// sums one at a time and 64-bit divisions the instructions bounded it: 54 us, 75 % of the issue slots.
// A few rows: one launch, 2.3 to 3.5 us (128 sequences x 1 row 3.4 us).

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "batched_ops.cuh"
#include "paged.cuh"

namespace mk {
namespace paged {

constexpr int kQueryHeads = 4;        // query heads of one token that a thread rotates with the same table elements (8: no faster)
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

// Two products or sums at once, each rounded by itself.  (One statement each: put together from tcgen05.cuh's pairs they cost
// registers, 7 prompts 46.9 -> 47.3 us.)
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// What a thread needs to rotate the 8 elements at its column: where their pairs are, and the sign of the pair's sine.
struct Turn {
    bool inside, half;   // half: pairs lie rot / 2 apart, in the lane `partner`; else side by side
    int partner;
    float2 sign;
};

__device__ __forceinline__ Turn turn_of(int chunk, int lane_chunk0, int rot, bool half) {
    Turn u;
    u.inside = 8 * chunk < rot;
    u.half = half;
    const int away = rot / 16;   // chunks between the two elements of a pair
    const bool second = chunk >= away;
    u.partner = lane_chunk0 + (u.inside ? (second ? chunk - away : chunk + away) : chunk);
    const float first = half && second ? 1.f : -1.f;
    u.sign = make_float2(first, half ? first : 1.f);
    return u;
}

// Cosines and signed sines of one position at 8 columns.
struct Angles {
    float2 c[4], s[4];
};
__device__ __forceinline__ void load_angles(const float *cosines, const float *sines, long long at, const Turn &u, Angles &g) {
    const float4 c0 = __ldg(reinterpret_cast<const float4 *>(cosines + at)), c1 = __ldg(reinterpret_cast<const float4 *>(cosines + at) + 1);
    const float4 s0 = __ldg(reinterpret_cast<const float4 *>(sines + at)), s1 = __ldg(reinterpret_cast<const float4 *>(sines + at) + 1);
    g.c[0] = make_float2(c0.x, c0.y); g.c[1] = make_float2(c0.z, c0.w);
    g.c[2] = make_float2(c1.x, c1.y); g.c[3] = make_float2(c1.z, c1.w);
    g.s[0] = mul2(make_float2(s0.x, s0.y), u.sign); g.s[1] = mul2(make_float2(s0.z, s0.w), u.sign);
    g.s[2] = mul2(make_float2(s1.x, s1.y), u.sign); g.s[3] = mul2(make_float2(s1.z, s1.w), u.sign);
}

__device__ __forceinline__ void widen(uint32_t w, float2 &x) { x = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// 8 bf16 elements, rotated, in fp32: x c + pair(x) (+-s), both products rounded.  All lanes of a warp call it.
__device__ __forceinline__ void rotate8(const uint4 &raw, const Angles &g, const Turn &u, float2 (&x)[4]) {
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w}, o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[i] = u.half ? __shfl_sync(0xffffffffu, w[i], u.partner) : __byte_perm(w[i], 0, 0x1032);
        widen(w[i], x[i]);
    }
    if (u.inside) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 y;
            widen(o[i], y);
            x[i] = add2(mul2(x[i], g.c[i]), mul2(y, g.s[i]));
        }
    }
}

__device__ __forceinline__ uint4 round8(const float2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[i].x, x[i].y);
        w[i] = *reinterpret_cast<const uint32_t *>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint2 pack_e4m3(const float2 (&x)[4], float factor) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(mul2(x[i], make_float2(factor, factor)), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

__device__ __forceinline__ uint2 recode_e4m3(uint2 codes, float factor) {
    float2 x[4];
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i % 2))), __NV_E4M3);
        x[i] = __half22float2(__half2(h));
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

// D: head dimension.  ITERS: rows of one page that a thread may hold.  BOTH: half of a CTA takes a page's keys, half its
// values; else they are two CTAs.
template <int D, int THREADS, int ITERS, bool BOTH, bool FP8, bool LIN>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)   // 64 registers; 7 prompts: 80 54 us, 40 60 us (spills)
append_kernel(const AppendParams p) {
    pdl_wait();   // and no early start for the next kernel: see paged.cuh
    constexpr int kLanes = D / 8;                          // threads per row
    constexpr int kPart = BOTH ? THREADS / 2 : THREADS, kPartWarps = kPart / 32;
    constexpr int kRows = kPart / kLanes;                  // rows per pass
    __shared__ float amax_s[THREADS / 32];
    const Batch &bt = p.bt;
    const int lane = threadIdx.x & 31, chunk = threadIdx.x % kLanes, lane0 = lane - chunk;
    const bool rope = p.rope_cos != nullptr;
    const Turn turn = turn_of(chunk, lane0, p.rot, p.half);

    if ((int)blockIdx.x >= p.kv_blocks) {                  // query rows: one token, kQueryHeads heads per thread
        constexpr int kUnits = THREADS / kLanes;           // (token, group of heads) pairs per CTA
        const int unit = ((int)blockIdx.x - p.kv_blocks) * kUnits + (int)threadIdx.x / kLanes;
        int t = div(unit, p.q_groups);
        const int head0 = (unit - t * p.q_groups.d) * kQueryHeads;
        bool live = t < bt.tokens;
        t = min(t, bt.tokens - 1);
        uint4 raw[kQueryHeads];
#pragma unroll
        for (int i = 0; i < kQueryHeads; ++i) raw[i] = head0 + i < p.hq ? load8<LIN>(p, p.q, 0, t, head0 + i, 8 * chunk) : make_uint4(0u, 0u, 0u, 0u);
        int b;
        if (bt.cu) {
            b = find_sequence(bt, __shfl_sync(0xffffffffu, t, 0), [](int first, int) { return first; });
            while (b + 1 < bt.seqs && __ldg(bt.cu + b + 1) <= t) ++b;
        } else {
            b = div(t, p.per_seq);
        }
        int first, count;
        rows_of(bt, b, first, count);
        const int start = __ldg(bt.where + b);
        live = live && start >= 0 && t >= first && t < first + count;   // idle sequences' rows stay as they were
        Angles angles;
        if (rope) {
            const long long want = (long long)start + (t - first);
            const int pos = clamp_int(want, 0, p.positions - 1);
            if (live && pos != want) {                     // beyond the tables: left as it was
                atomicOr(bt.error, kErrorIndex);
                live = false;
            }
            if (turn.inside) load_angles(p.rope_cos, p.rope_sin, (long long)pos * p.rot + 8 * chunk, turn, angles);
        }
        bf16 *dst = p.q_out + ((long long)t * p.hq + head0) * D + 8 * chunk;
#pragma unroll
        for (int i = 0; i < kQueryHeads; ++i) {
            uint4 out = raw[i];
            if (rope) {
                float2 x[4];
                rotate8(raw[i], angles, turn, x);
                out = round8(x);
            }
            if (live && head0 + i < p.hq) *reinterpret_cast<uint4 *>(dst + i * D) = out;
        }
        return;
    }

    // keys and values of one (page, KV head)
    const int hkv = p.pool.kv_heads, page_size = 1 << bt.page_shift;
    const int pair = BOTH ? blockIdx.x : blockIdx.x >> 1;
    const int slot = div(pair, p.kv_heads), head = pair - slot * hkv;
    const bool is_v = BOTH ? threadIdx.x >= kPart : blockIdx.x & 1;
    const int row_in_pass = (threadIdx.x % kPart) / kLanes;
    int b, ordinal;
    if (bt.cu) {
        b = find_sequence(bt, slot, [&](int first, int at) { return first_slot(bt, first, at); });
        ordinal = slot - first_slot(bt, clamp_int(__ldg(bt.cu + b), 0, bt.tokens), b);
    } else {
        b = div(slot, p.slots);
        ordinal = slot - b * p.slots.d;
    }
    int first, count;
    rows_of(bt, b, first, count);
    const int start = __ldg(bt.where + b);
    if (start < 0 || ordinal < 0) return;                  // idle sequence; offsets that do not grow
    const long long column = (long long)(start >> bt.page_shift) + ordinal;
    const long long page_begin = column << bt.page_shift;
    const long long past = (long long)start + count;       // the position behind the sequence's rows
    if (page_begin >= past) return;                        // they end before this slot's page
    if (column >= bt.max_pages) {
        if (threadIdx.x == 0) atomicOr(bt.error, kErrorIndex);
        return;
    }
    const int held = page_begin < start ? (int)(start - page_begin) : 0;   // rows in the page before this call
    // rows that the rotary tables do not reach, and their values, are left out
    const long long stop = rope ? min(past, (long long)p.positions) : past;
    const int end = (int)max(min((long long)page_size, stop - page_begin), 0ll);
    const int added = end - held;
    const int t0 = first + (int)(page_begin + held - start);               // token row of the page's first new row

    const int page = __ldg(bt.table + b * bt.table_stride + column);
    if (stop < past && end < page_size) {
        if (page >= 0 && threadIdx.x == 0) atomicOr(bt.error, kErrorIndex);
        if (added <= 0) return;
    }
    uint4 raw[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        if (it * kRows < added) {
            const int t = t0 + min(it * kRows + row_in_pass, added - 1);   // repeated rows change nothing
            raw[it] = is_v ? load8<LIN>(p, p.v, (p.hq + hkv) * D, t, head, 8 * chunk) : load8<LIN>(p, p.k, p.hq * D, t, head, 8 * chunk);
        }
    }
    const bool rotated = rope && !is_v;
    const long long pos0 = page_begin + held;              // below p.positions where rows are rotated
    // row `it` of this thread in fp32, keys rotated
    auto value = [&](int it, float2 (&x)[4]) {
        if (rotated) {
            const int pos = (int)pos0 + min(it * kRows + row_in_pass, added - 1);
            Angles angles;
            if (turn.inside) load_angles(p.rope_cos, p.rope_sin, (long long)pos * p.rot + 8 * chunk, turn, angles);
            rotate8(raw[it], angles, turn, x);
        } else {
            widen(raw[it].x, x[0]); widen(raw[it].y, x[1]); widen(raw[it].z, x[2]); widen(raw[it].w, x[3]);
        }
    };
    // the rows are made before the page id is looked at: the tables' elements arrive with it, not after it
    float2 kept[ITERS][4];
#pragma unroll
    for (int it = 0; it < ITERS; ++it)
        if (it * kRows < added) value(it, kept[it]);
    if (page < 0) return;                                  // no page: nothing is kept
    if (page >= bt.num_pages) {
        if (threadIdx.x == 0) atomicOr(bt.error, kErrorIndex);
        return;
    }
    const long long base = page * p.pool.page_stride + head * p.pool.head_stride + 8 * chunk;
    if constexpr (!FP8) {
        bf16 *dst = reinterpret_cast<bf16 *>(is_v ? p.pool.v : p.pool.k) + base;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            if (it * kRows < added) {
                const int i = it * kRows + row_in_pass;
                if (i < added) *reinterpret_cast<uint4 *>(dst + (held + i) * p.pool.slot_stride) = round8(kept[it]);
            }
        }
    } else {
        float amax = 0.f;                                      // NaN never enters
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            if (it * kRows < added) {
#pragma unroll
                for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(kept[it][j].x), fabsf(kept[it][j].y)));
            }
        }
        if (amax == INFINITY) {                                // infinities saturate: the finite elements set the scale
            amax = 0.f;
            auto finite = [&](float a) { if (a < INFINITY) amax = fmaxf(amax, a); };
#pragma unroll
            for (int it = 0; it < ITERS; ++it)
                if (it * kRows < added)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        finite(fabsf(kept[it][j].x));
                        finite(fabsf(kept[it][j].y));
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
        for (int w = 0; w < kPartWarps; ++w) amax = fmaxf(amax, amax_s[(BOTH && is_v ? kPartWarps : 0) + w]);
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
        if (threadIdx.x % kPart == 0) *scales = scale;
        const float inverse = 1.0f / scale;                    // exact: a power of two
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            if (it * kRows < added) {
                const int i = it * kRows + row_in_pass;
                if (i < added) *reinterpret_cast<uint2 *>(dst + (held + i) * p.pool.slot_stride) = pack_e4m3(kept[it], inverse);
            }
        }
    }
}

template <int D, int THREADS, int ITERS, bool BOTH, bool FP8, bool LIN>
static cudaError_t launch_append_t(AppendParams &p, long long kv, cudaStream_t st) {
    const int groups = (p.hq + kQueryHeads - 1) / kQueryHeads, per_cta = THREADS * 8 / D;
    const long long units = p.q_out ? (long long)p.bt.tokens * groups : 0, q = (units + per_cta - 1) / per_cta;
    if (units + per_cta > 0x7fffffff) return cudaErrorInvalidConfiguration;
    p.q_groups = fast_div(groups ? groups : 1);
    p.kv_heads = fast_div(p.pool.kv_heads);
    p.per_seq = fast_div(p.bt.cu ? 1 : p.bt.per_seq);
    if (!BOTH) kv *= 2;
    if (kv + q > 0x7fffffff) return cudaErrorInvalidConfiguration;
    p.kv_blocks = (int)kv;
    return launch_pdl(append_kernel<D, THREADS, ITERS, BOTH, FP8, LIN>, dim3((unsigned)(kv + q)), dim3(THREADS), 0, st, p);
}

template <int D, bool FP8, bool LIN>
static cudaError_t launch_append_d(AppendParams &p, long long kv, int rows, cudaStream_t st) {
    // A few rows per page (decoding): a warp each for keys and values, so that every CTA of a large batch is resident at
    // once (128 sequences x 8 heads: 12.7 us with the wide CTAs below, 4 with these).
    constexpr int kFew = 32 * 8 / D;   // rows of one pass of a warp
    if (rows <= kFew) return launch_append_t<D, 64, 1, true, FP8, LIN>(p, kv, st);
    if (rows <= 2 * kFew) return launch_append_t<D, 64, 2, true, FP8, LIN>(p, kv, st);
    switch (p.pool.page_size * D / 1024) {
    case 1: return launch_append_t<D, 128, 1, false, FP8, LIN>(p, kv, st);
    case 2: return launch_append_t<D, 256, 1, false, FP8, LIN>(p, kv, st);
    case 4: return launch_append_t<D, 256, 2, false, FP8, LIN>(p, kv, st);
    case 8: return launch_append_t<D, 256, 4, false, FP8, LIN>(p, kv, st);
    case 16: return launch_append_t<D, 512, 4, false, FP8, LIN>(p, kv, st);
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
        p.slots = fast_div(1);
    } else {
        p.slots = fast_div(bt.per_seq == 1 ? 1 : (bt.per_seq - 1) / page + 2);
        slots = (long long)p.slots.d * bt.seqs;
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
