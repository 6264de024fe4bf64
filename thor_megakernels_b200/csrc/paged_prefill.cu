// Attention over a paged cache for sequences with many new rows (prompts, chunks of prompts):
// the same operator as paged_attention.cu on the 5th-generation tensor cores.
//
// Shape of the work.  A row block is 256 (query token, query head of the group) pairs of one
// sequence and KV head, two MMA tiles of 128 rows; the cache goes by in tiles of 128 positions.
// Per tile and row tile:  S = Q K^T (tcgen05.mma, operands in shared memory, S in tensor memory),
// softmax weights P by one thread per row (tensor memory to registers and back, 16-bit), and
// O += P V (P from tensor memory, V in shared memory as it lies there: positions are rows, so
// it is an MN-major operand).  Everything a row needs is in one thread: no shuffles.
//
// What bounds it: per 128 x 128 tile the tensor core needs 4 x 128 x 128 x D flops - 1024 clocks
// at D = 128 - and the softmax 128 x 128 exponentials - 1024 clocks of the special function unit.
// Two row tiles alternate, so that one's softmax runs under the other's products:
//     S0(j+1) follows O0(j), S1(j+1) follows O1(j) in the issue order,
// and weights take S's place in tensor memory.  The output is rescaled only when the running
// maximum has grown by more than 2^8 since the last time (weights stay below 256, sums are fp32);
// after the first tiles that is rare.
//
// Warp roles: 0-3 and 4-7 softmax of row tile 0 and 1 (and query loading, epilogue), 8 loader (TMA,
// one box per page), 9 tensor-memory allocation and MMA issue, and for the 8-bit cache 10 and 11
// converters: E4M3 codes land as they are in a small ring and become f16 (exact) in the swizzled
// operand tiles; queries are f16 scaled by a power of two per row, page scales enter at the scores
// and the value scale joins the exponent, as in paged_attention.cu.  A bf16 cache goes from TMA
// to the tensor core without passing a register; its weights are one bf16 term each.
//
// Values that are not finite and lie at positions some rows do not see (or behind the end) are
// taken out of the tile by the warp that fills it; rows that do see them get them in the epilogue.
//
// Work split.  With at least two row blocks per SM every CTA takes one, those with the longest
// cache first; otherwise units (row block, tile) are dealt out in equal consecutive ranges and a
// second kernel joins the parts.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/b200_megakernel.h"
#include "batched_ops.cuh"
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace mk {

void set_last_error(const char *msg);  // megakernel.cu

namespace paged {

constexpr int kTileTokens = 128;
constexpr int kBlockRows = 256;
constexpr int kPanelBytes = 128 * 128;     // 128 rows of one 128-byte swizzle row
constexpr int kChunks = kTileTokens / 16;  // a page is at least 16 positions
constexpr int kBadBuffers = 4;

template <int D, bool FP8>
struct Prefill {
    static constexpr int kConverters = 64;
    static constexpr int kThreads = FP8 ? 320 + kConverters : 320;
    static constexpr int kPanels = D / 64;
    static constexpr int kOperandBytes = kPanels * kPanelBytes;   // 128 rows x D two-byte elements
    static constexpr int kRawTokens = kTileTokens / 2, kRawStages = FP8 ? 3 : 1;
    static constexpr int kRawBytes = FP8 ? kRawTokens * D : 16;
    static constexpr int kBadKinds = FP8 ? 1 : 3;                 // E4M3 has NaN only
    struct __align__(1024) Smem {
        uint8_t q[2][kOperandBytes];
        uint8_t k[2][kOperandBytes];
        uint8_t v[2][kOperandBytes];
        uint8_t raw[kRawStages][kRawBytes];
        uint64_t raw_full[kRawStages], raw_empty[kRawStages], k_full[2], k_empty[2], v_full[2], v_empty[2], v_raw;
        uint64_t s_full[2], p_full[2], o_full[2], q_full, drain;
        float ks[4][kChunks], ev[4][kChunks], iev[4][kChunks];   // by tile counter mod 4: key scale, log2 of the value scale and its inverse
        int general[4];                                          // the tile needs them
        int bad[kBadBuffers][kBadKinds][D];                              // first position whose value in a column is NaN, +inf, -inf
        int bad_any[kBadBuffers];
        uint32_t tmem_base;
        int failed;
        int scan[kThreads / 32];
    };
};

struct PrefillParams {
    AttentionParams a;
    int min_count;      // sequences with fewer new tokens are the other kernel's
    int whole;          // every CTA takes one row block
};

struct Segment {
    int b, first, count, length, rb, head, tile0, tile1, rows;
    bool complete;      // the row block's tiles are all in this segment
    int n[2];           // tiles of the two row tiles in it
    int all_see;        // positions that every row sees
};

__device__ __forceinline__ void describe(const AttentionParams &p, Segment &s) {
    s.rows = min(kBlockRows, s.count * p.group - s.rb * kBlockRows);
    s.all_see = visible(s.length, s.count, s.rb * kBlockRows / p.group);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int last = min(s.rows, 128 * (i + 1)) - 1;
        int n = 0;
        if (last >= 128 * i) {
            const int seen = visible(s.length, s.count, (s.rb * kBlockRows + last) / p.group);
            n = max(min((seen + kTileTokens - 1) / kTileTokens, s.tile1) - s.tile0, 0);
        }
        s.n[i] = n;
    }
}

// Walks over a CTA's segments.  Every role runs its own copy.
struct Walk {
    const int *prefix;
    int u, u_end, b;
    bool done;
    __device__ __forceinline__ bool next(const PrefillParams &p, Segment &s) {
        if (u >= u_end) return false;
        const AttentionParams &a = p.a;
        int lo = b, hi = a.bt.seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (prefix[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        b = s.b = lo;
        rows_of(a.bt, b, s.first, s.count);
        s.length = length_of(a.bt, b);
        int rest = u - prefix[b];
        if (p.whole) {
            s.rb = block_count(s.count, a.group, kBlockRows) - 1 - rest / a.hkv;
            s.head = rest % a.hkv;
            s.tile0 = 0;
            s.tile1 = max(block_tiles(s.length, s.count, a.group, kBlockRows, s.rb, kTileTokens), 1);
            s.complete = true;
            u += 1;
        } else {
            s.rb = 0;
            int tiles;
            while (true) {
                tiles = max(block_tiles(s.length, s.count, a.group, kBlockRows, s.rb, kTileTokens), 1);
                if (rest < tiles * a.hkv) break;
                rest -= tiles * a.hkv;
                ++s.rb;
            }
            s.head = rest / tiles;
            s.tile0 = rest % tiles;
            s.tile1 = min(tiles, s.tile0 + (u_end - u));
            s.complete = s.tile0 == 0 && s.tile1 == tiles;
            u += s.tile1 - s.tile0;
        }
        describe(a, s);
        return true;
    }
};

__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, volatile int *failed) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long began = clock64();
    unsigned it = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++it & 63u) == 0) {
            if (*failed) return false;
            if (clock64() - began > kWaitCycles) {
                *failed = 1;
                return false;
            }
        }
    }
    return true;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// byte offset of 16-byte chunk c of row r in an operand tile (panels of 64 elements, 128-byte swizzle)
__device__ __forceinline__ uint32_t operand_chunk(int r, int c) { return (c >> 3) * kPanelBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

template <int D, bool FP8>
__global__ void __launch_bounds__(Prefill<D, FP8>::kThreads, 1)
prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefillParams pp) {
    using T = Prefill<D, FP8>;
    using Smem = typename T::Smem;
    extern __shared__ uint8_t smem_raw[];
    Smem &s = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int *prefix = reinterpret_cast<int *>(&s + 1);   // [seqs + 1]
    const AttentionParams &p = pp.a;
    const Batch &bt = p.bt;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *failed = &s.failed;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.k_full[i], FP8 ? T::kConverters : 1);
            mbar_init(&s.v_full[i], FP8 ? T::kConverters : 1);
            mbar_init(&s.k_empty[i], 1);
            mbar_init(&s.v_empty[i], 1);
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], 128);
            mbar_init(&s.o_full[i], 1);
        }
        for (int i = 0; i < T::kRawStages; ++i) {
            mbar_init(&s.raw_full[i], 1);
            mbar_init(&s.raw_empty[i], T::kConverters);
        }
        mbar_init(&s.v_raw, 1);
        mbar_init(&s.q_full, 256);
        mbar_init(&s.drain, 1);
        s.failed = 0;
        fence_barrier_init();
    }
    pdl_wait();

    // units (or row blocks) of the sequences before each one
    {
        const int per = (bt.seqs + T::kThreads - 1) / T::kThreads;
        const int b0 = min((int)threadIdx.x * per, bt.seqs), b1 = min(b0 + per, bt.seqs);
        int sum = 0;
        for (int b = b0; b < b1; ++b) {
            int first, count;
            rows_of(bt, b, first, count);
            int units = 0;
            if (count >= pp.min_count)
                units = pp.whole ? block_count(count, p.group, kBlockRows) * p.hkv
                                 : sequence_units(length_of(bt, b), count, p.group, kBlockRows, kTileTokens, p.hkv);
            prefix[b + 1] = units;
            sum += units;
        }
        int incl = sum;
#pragma unroll
        for (int off = 1; off < 32; off *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += v;
        }
        if (lane == 31) s.scan[warp] = incl;
        __syncthreads();
        int before = incl - sum;
        for (int w = 0; w < warp; ++w) before += s.scan[w];
        for (int b = b0; b < b1; ++b) {
            before += prefix[b + 1];
            prefix[b + 1] = before;
        }
        if (threadIdx.x == 0) prefix[0] = 0;
        __syncthreads();
    }
    const int units = prefix[bt.seqs];
    if (blockIdx.x == 0 && p.prefix_out && !pp.whole)
        for (int b = threadIdx.x; b <= bt.seqs; b += T::kThreads) p.prefix_out[b] = prefix[b];
    Walk walk;
    walk.prefix = prefix;
    walk.b = 0;
    if (pp.whole) {
        walk.u = blockIdx.x;
        walk.u_end = min((int)blockIdx.x + 1, units);
    } else {
        const int ctas = working_ctas(gridDim.x, units);
        walk.u = (int)blockIdx.x < ctas ? first_unit(blockIdx.x, ctas, units) : 0;
        walk.u_end = (int)blockIdx.x < ctas ? first_unit(blockIdx.x + 1, ctas, units) : 0;
    }
    if (walk.u >= walk.u_end) return;   // the whole CTA

    // Tensor memory is taken only after the kernel before this one has ended, and the next kernel is let in
    // only after that: nobody who holds it waits for somebody who wants it.
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s.tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = s.tmem_base;
    const int page_size = 1 << bt.page_shift;

    Segment seg;
    if (warp < 8) {
        // ------------------------------------------------------------------ softmax of one row tile
        const int i = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tm = tmem + lanes + i * 128, o_tm = tmem + lanes + 256 + i * 128;
        uint32_t s_parity = 0, o_parity = 0;
        int tile_ctr = 0, bearing = 0;   // tiles and tile-bearing segments of this CTA so far
        bool ok = true;
        while (ok && walk.next(pp, seg)) {
            const int r = 128 * i + row, pair = seg.rb * kBlockRows + r;
            const bool real = r < seg.rows;
            const int token = real ? pair / p.group : 0;
            // this thread's query row into the operand tile
            float c_row = fabsf(p.scale_log2e);
            {
                const bool negate = p.scale_log2e < 0.f;   // scores are compared as they come, so their factor is kept positive
                const bf16 *qp = p.q + (long long)(seg.first + token) * p.q_token + (long long)(seg.head * p.group + (real ? pair % p.group : 0)) * p.q_head;
                uint4 raw[D / 8];
#pragma unroll
                for (int c = 0; c < D / 8; ++c) raw[c] = real ? __ldg(reinterpret_cast<const uint4 *>(qp) + c) : make_uint4(0u, 0u, 0u, 0u);
                float factor = negate ? -1.f : 1.f;
                if constexpr (FP8) {
                    float amax = 0.f;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        float x[8];
                        unpack8(raw[c], x);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float a = fabsf(x[k]);
                            if (a < INFINITY) amax = fmaxf(amax, a);
                        }
                    }
                    const int e = max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -120);   // amax / 2^e in [2^14, 2^15)
                    factor *= __uint_as_float((uint32_t)(127 - e) << 23);
                    c_row *= __uint_as_float((uint32_t)(127 + e) << 23);
                }
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    uint4 w = raw[c];
                    if constexpr (FP8) {
                        float x[8];
                        unpack8(raw[c], x);
                        w = make_uint4(pack_f16(x[0] * factor, x[1] * factor), pack_f16(x[2] * factor, x[3] * factor),
                                       pack_f16(x[4] * factor, x[5] * factor), pack_f16(x[6] * factor, x[7] * factor));
                    } else if (negate) {
                        w.x ^= 0x80008000u; w.y ^= 0x80008000u; w.z ^= 0x80008000u; w.w ^= 0x80008000u;
                    }
                    *reinterpret_cast<uint4 *>(s.q[i] + operand_chunk(row, c)) = w;
                }
                fence_async_smem();
                mbar_arrive(&s.q_full);
            }
            const int limit = real ? visible(seg.length, seg.count, token) : 0;
            const int all_see = visible(seg.length, seg.count, (seg.rb * kBlockRows + 128 * i) / p.group);
            float m = -INFINITY, l = 0.f;
            const int n = seg.n[i], n_any = max(seg.n[0], seg.n[1]);

            for (int j = 0; j < n; ++j) {
                ok = __all_sync(0xffffffffu, wait_bar(&s.s_full[i], s_parity, failed));
                if (!ok) break;
                s_parity ^= 1u;
                tcgen05_fence_after();
                const int slot = (tile_ctr + j) & 3, pos0 = (seg.tile0 + j) * kTileTokens;
                const bool masked = pos0 + kTileTokens > all_see;
                const int lim = limit - pos0;   // columns below it are seen
                const bool general = FP8 || s.general[slot] != 0;
                uint32_t x[2][32];

                // largest score
                float top = -INFINITY;
                tmem_load32(s_tm, x[0]);
                tmem_load_wait(x[0]);
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    if (ch < 3) tmem_load32(s_tm + 32 * (ch + 1), x[(ch + 1) & 1]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float c = general ? c_row * s.ks[slot][2 * ch + h] : c_row;
                        const float e = general ? s.ev[slot][2 * ch + h] : 0.f;
                        if (masked) {
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                top = fmaxf(top, 32 * ch + 16 * h + k < lim ? fmaf(__uint_as_float(x[ch & 1][16 * h + k]), c, e) : -INFINITY);
                        } else {
                            float mx = __uint_as_float(x[ch & 1][16 * h]);
#pragma unroll
                            for (int k = 1; k < 16; ++k) mx = fmaxf(mx, __uint_as_float(x[ch & 1][16 * h + k]));
                            top = fmaxf(top, fmaf(mx, c, e));
                        }
                    }
                    if (ch < 3) tmem_load_wait(x[(ch + 1) & 1]);
                }
                // the running maximum, and the output if it has grown too much
                {
                    const float grown = fmaxf(m, top);
                    const bool need = grown > m + 8.f;   // also from -inf
                    if (j == 0) {
                        m = grown;
                    } else if (__any_sync(0xffffffffu, need)) {
                        const float corr = need ? exp2_fast(m - grown) : 1.f;
                        if (need) m = grown;
                        l *= corr;
#pragma unroll
                        for (int ch = 0; ch < D / 32; ++ch) {
                            tmem_load32(o_tm + 32 * ch, x[0]);
                            tmem_load_wait(x[0]);
#pragma unroll
                            for (int k = 0; k < 32; ++k) x[0][k] = __float_as_uint(__uint_as_float(x[0][k]) * corr);
                            tmem_store32(o_tm + 32 * ch, x[0]);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                // weights, in the place of the scores
                tmem_load32(s_tm, x[0]);
                tmem_load_wait(x[0]);
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    if (ch < 3) tmem_load32(s_tm + 32 * (ch + 1), x[(ch + 1) & 1]);
                    uint32_t w[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float c = general ? c_row * s.ks[slot][2 * ch + h] : c_row;
                        const float e = (general ? s.ev[slot][2 * ch + h] : 0.f) - base;
                        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            float w0 = exp2_fast(fmaf(__uint_as_float(x[ch & 1][16 * h + k]), c, e));
                            float w1 = exp2_fast(fmaf(__uint_as_float(x[ch & 1][16 * h + k + 1]), c, e));
                            if (masked) {
                                if (32 * ch + 16 * h + k >= lim) w0 = 0.f;
                                if (32 * ch + 16 * h + k + 1 >= lim) w1 = 0.f;
                            }
                            sum0 += w0;
                            sum1 += w1;
                            w[8 * h + k / 2] = FP8 ? pack_f16(w0, w1) : pack_b16(w0, w1);
                        }
                        l = general ? fmaf(sum0 + sum1, s.iev[slot][2 * ch + h], l) : l + (sum0 + sum1);
                    }
                    if (ch < 3) tmem_load_wait(x[(ch + 1) & 1]);   // a store only overwrites columns that have been read
                    tmem_store16(s_tm + 16 * ch, w);
                }
                tmem_store_wait();
                tcgen05_fence_before();
                mbar_arrive(&s.p_full[i]);
            }
            tile_ctr += n_any;
            if (!ok) break;

            // epilogue
            ok = __all_sync(0xffffffffu, wait_bar(&s.o_full[i], o_parity, failed));
            if (!ok) break;
            o_parity ^= 1u;
            tcgen05_fence_after();
            const int buffer = bearing & (kBadBuffers - 1);
            const bool bad = n > 0 && (volatile int &)s.bad_any[buffer] != 0;
            if (n_any > 0) ++bearing;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            float *part = p.partial + ((long long)blockIdx.x * 2 + (seg.tile0 == 0 ? 1 : 0)) * kBlockRows * (D + 2);
            bf16 *dst = p.out + ((long long)(seg.first + token) * p.hq + seg.head * p.group + (real ? pair % p.group : 0)) * D;
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
                uint32_t x[32];
                if (n > 0) {
                    tmem_load32(o_tm + 32 * ch, x);
                    tmem_load_wait(x);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = 0u;
                }
                if (bad) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        float y = __uint_as_float(x[k]);
                        if ((volatile int &)s.bad[buffer][0][32 * ch + k] < limit) y = __int_as_float(0x7fffffff);
                        if constexpr (!FP8) {
                            if ((volatile int &)s.bad[buffer][1][32 * ch + k] < limit) y += INFINITY;
                            if ((volatile int &)s.bad[buffer][2][32 * ch + k] < limit) y -= INFINITY;
                        }
                        x[k] = __float_as_uint(y);
                    }
                }
                if (real) {
                    if (seg.complete) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            uint4 v;
                            v.x = pack_b16(__uint_as_float(x[k]) * inv, __uint_as_float(x[k + 1]) * inv);
                            v.y = pack_b16(__uint_as_float(x[k + 2]) * inv, __uint_as_float(x[k + 3]) * inv);
                            v.z = pack_b16(__uint_as_float(x[k + 4]) * inv, __uint_as_float(x[k + 5]) * inv);
                            v.w = pack_b16(__uint_as_float(x[k + 6]) * inv, __uint_as_float(x[k + 7]) * inv);
                            *reinterpret_cast<uint4 *>(dst + 32 * ch + k) = v;
                        }
                    } else {   // four columns of 256 rows side by side
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<uint4 *>(part + ((32 * ch + k) / 4 * kBlockRows + r) * 4) = make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                    }
                }
            }
            if (real && !seg.complete) *reinterpret_cast<float2 *>(part + D * kBlockRows + 2 * r) = make_float2(m, l);
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------------ loader
        uint32_t kv_it = 0, raw_stage = 0, raw_parity = 0, raw_fills = 0, v_raw_parity = 0;
        int bearing = 0;
        bool ok = true;
        while (ok && walk.next(pp, seg)) {
            const int n = max(seg.n[0], seg.n[1]);
            if (n == 0) continue;
            const int buffer = bearing & (kBadBuffers - 1);
            ++bearing;
            for (int c = lane; c < T::kBadKinds * D; c += 32) (&s.bad[buffer][0][0])[c] = 0x7fffffff;
            if (lane == 0) s.bad_any[buffer] = 0;
            __syncwarp();
            const int *table = bt.table + seg.b * bt.table_stride;
            // page of 16-position chunk `lane` of a tile
            auto page_of = [&](int j) {
                const int pos = (seg.tile0 + j) * kTileTokens + 16 * lane;
                if (lane >= kChunks || j >= n || pos >= seg.length) return -1;
                const int id = __ldg(table + (pos >> bt.page_shift));
                if (id >= bt.num_pages) {
                    atomicOr(bt.error, kErrorIndex);
                    return -1;
                }
                return id < 0 ? -1 : id;
            };
            int page = page_of(0);
            for (int j = 0; j < n; ++j, ++kv_it) {
                const int page_next = page_of(j + 1);
                const int pos0 = (seg.tile0 + j) * kTileTokens, stage = kv_it & 1, slot = kv_it & 3;
                const uint32_t reuse = ((kv_it >> 1) & 1) ^ 1u;   // parity of the stage's last release
                float ks = 1.f, ev = -INFINITY, iev = 0.f;
                if (lane < kChunks && page >= 0) {
                    ev = 0.f;
                    iev = 1.f;
                    if constexpr (FP8) {
                        const long long at = (long long)page * p.hkv + seg.head;
                        const float vs = fmaxf(__ldg(p.v_scales + at), 0x1p-100f);
                        ks = __ldg(p.k_scales + at);
                        ev = log2f(vs);
                        iev = 1.f / vs;
                    }
                }
                const bool behind_end = pos0 + 16 * lane >= seg.length;
                const bool general = __any_sync(0xffffffffu, lane < kChunks && page < 0 && !behind_end);

                // positions [from, from + tokens) of the tile; all lanes call it, lane 0 issues
                auto boxes = [&](uint8_t *dst, const CUtensorMap *map, uint64_t *bar, int from, int tokens) {
                    const int rows = min(page_size, tokens);   // of one box
                    for (int at = 0; at < tokens; at += rows) {
                        const int id = __shfl_sync(0xffffffffu, page, (from + at) / 16), in_page = (from + at) & (page_size - 1);
                        if (lane == 0) {
                            if constexpr (FP8) {
                                tma_load_4d(smem_addr(dst) + at * D, map, 0, in_page, seg.head, id, bar);
                            } else {
#pragma unroll
                                for (int panel = 0; panel < T::kPanels; ++panel)
                                    tma_load_4d(smem_addr(dst) + panel * kPanelBytes + at * 128, map, 64 * panel, in_page, seg.head, id, bar);
                            }
                        }
                    }
                };
                if constexpr (FP8) {
                    for (int part = 0; part < 4; ++part) {   // keys, then values, in halves
                        ok = __all_sync(0xffffffffu, wait_bar(&s.raw_empty[raw_stage], raw_parity ^ 1u, failed));
                        if (!ok) break;
                        if (part == 0) {   // before the barrier that leads to this tile's scores
                            if (lane < kChunks) { s.ks[slot][lane] = ks; s.ev[slot][lane] = ev; s.iev[slot][lane] = iev; }
                            if (lane == 0) s.general[slot] = 1;
                            __syncwarp();
                        }
                        if (lane == 0) mbar_arrive_expect_tx(&s.raw_full[raw_stage], T::kRawBytes);
                        __syncwarp();
                        boxes(s.raw[raw_stage], part < 2 ? &map_k : &map_v, &s.raw_full[raw_stage], (part & 1) * T::kRawTokens, T::kRawTokens);
                        ++raw_fills;
                        if (++raw_stage == T::kRawStages) { raw_stage = 0; raw_parity ^= 1u; }
                    }
                    if (!ok) break;
                } else {
                    ok = __all_sync(0xffffffffu, wait_bar(&s.k_empty[stage], reuse, failed));
                    if (!ok) break;
                    if (lane < kChunks) { s.ks[slot][lane] = ks; s.ev[slot][lane] = ev; s.iev[slot][lane] = iev; }
                    if (lane == 0) s.general[slot] = general ? 1 : 0;
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(&s.k_full[stage], T::kOperandBytes);
                    __syncwarp();
                    boxes(s.k[stage], &map_k, &s.k_full[stage], 0, kTileTokens);
                    ok = __all_sync(0xffffffffu, wait_bar(&s.v_empty[stage], reuse, failed));
                    if (!ok) break;
                    const bool edge = pos0 + kTileTokens > seg.all_see;   // some rows do not see all of it
                    uint64_t *bar = edge ? &s.v_raw : &s.v_full[stage];
                    if (lane == 0) mbar_arrive_expect_tx(bar, T::kOperandBytes);
                    __syncwarp();
                    boxes(s.v[stage], &map_v, bar, 0, kTileTokens);
                    if (edge) {
                        ok = __all_sync(0xffffffffu, wait_bar(&s.v_raw, v_raw_parity, failed));
                        if (!ok) break;
                        v_raw_parity ^= 1u;
                        const int from = max(seg.all_see - pos0, 0);
                        for (int idx = from * (D / 8) + lane; idx < kTileTokens * (D / 8); idx += 32) {
                            const int r = idx / (D / 8), c = idx % (D / 8);
                            uint4 *at = reinterpret_cast<uint4 *>(s.v[stage] + operand_chunk(r, c));
                            if (pos0 + r >= seg.length) {
                                *at = make_uint4(0u, 0u, 0u, 0u);
                            } else {
                                const uint4 v = *at;
                                uint32_t w[4] = {v.x, v.y, v.z, v.w};
                                uint32_t odd = 0;
#pragma unroll
                                for (int k = 0; k < 4; ++k) odd |= __vcmpeq2(w[k] & 0x7f807f80u, 0x7f807f80u);
                                if (odd) {
#pragma unroll
                                    for (int k = 0; k < 8; ++k) {
                                        const uint32_t bits = (w[k / 2] >> (16 * (k & 1))) & 0xffffu;
                                        if ((bits & 0x7f80u) == 0x7f80u) {
                                            atomicMin(&s.bad[buffer][(bits & 0x7fu) ? 0 : (bits & 0x8000u) ? 2 : 1][8 * c + k], pos0 + r);
                                            w[k / 2] &= ~(0xffffu << (16 * (k & 1)));
                                        }
                                    }
                                    s.bad_any[buffer] = 1;
                                    *at = make_uint4(w[0], w[1], w[2], w[3]);
                                }
                            }
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&s.v_full[stage]);
                    }
                }
                page = page_next;
            }
        }
        // Never leave with copies in flight: in a clean run the other roles have waited for every fill.
        if (*failed && lane == 0) {
            const long long began = clock64();
            auto drain = [&](uint64_t *bar, uint32_t fills) {   // the last of a stage's fills so far
                while (fills > 0 && !mbar_try_wait(bar, (fills - 1) & 1u) && clock64() - began < kWaitCycles) {}
            };
            if constexpr (FP8) {
                for (uint32_t i = 0; i < T::kRawStages; ++i) drain(&s.raw_full[i], (raw_fills + T::kRawStages - 1 - i) / T::kRawStages);
            } else {
                drain(&s.v_raw, v_raw_parity + 1);   // the wait for it may be what ran out
                for (uint32_t i = 0; i < 2; ++i) {   // the fill of the tile in hand may be in flight already
                    drain(&s.k_full[i], (kv_it + 2 - i) / 2);
                    drain(&s.v_full[i], (kv_it + 2 - i) / 2);
                }
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------------------------------------ MMA issue
        if (lane == 0) {
            const uint32_t idesc_s = umma_idesc16(!FP8, kTileTokens, false), idesc_o = umma_idesc16(!FP8, D, true);
            uint32_t kv_it = 0, q_parity = 0, p_parity[2] = {0u, 0u};
            bool ok = true;
            auto scores = [&](int i, uint32_t it) {   // S_i = Q_i K^T
                const uint64_t dq = smem_desc_k_major_sw128(s.q[i]), dk = smem_desc_k_major_sw128(s.k[it & 1]);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t step = (uint64_t)((ks >> 2) * (kPanelBytes >> 4) + (ks & 3) * 2);
                    umma16_ss(tmem + i * 128, dq + step, dk + step, idesc_s, ks != 0);
                }
                umma_commit(&s.s_full[i]);
            };
            while (ok && walk.next(pp, seg)) {
                if (!(ok = wait_bar(&s.q_full, q_parity, failed))) break;
                q_parity ^= 1u;
                const int n = max(seg.n[0], seg.n[1]);
                for (int i = 0; i < 2; ++i)   // a row tile without positions goes on, but never ahead of this segment
                    if (seg.n[i] == 0) mbar_arrive(&s.o_full[i]);
                if (n == 0) continue;
                if (!(ok = wait_bar(&s.k_full[kv_it & 1], (kv_it >> 1) & 1, failed))) break;
                tcgen05_fence_after();
                for (int i = 0; i < 2; ++i)
                    if (seg.n[i] > 0) scores(i, kv_it);
                umma_commit(&s.k_empty[kv_it & 1]);
                for (int j = 0; ok && j < n; ++j, ++kv_it) {
                    if (!(ok = wait_bar(&s.v_full[kv_it & 1], (kv_it >> 1) & 1, failed))) break;
                    if (j + 1 < n && !(ok = wait_bar(&s.k_full[(kv_it + 1) & 1], ((kv_it + 1) >> 1) & 1, failed))) break;
                    const uint64_t dv = smem_desc_mn_major_sw128(s.v[kv_it & 1], kPanelBytes);
                    for (int i = 0; i < 2; ++i) {
                        if (j >= seg.n[i]) continue;
                        if (!(ok = wait_bar(&s.p_full[i], p_parity[i], failed))) break;
                        p_parity[i] ^= 1u;
                        tcgen05_fence_after();
#pragma unroll
                        for (int ks = 0; ks < kTileTokens / 16; ++ks)   // 16 positions: 16 rows of 128 bytes, 8 columns of weights
                            umma16_ts(tmem + 256 + i * 128, tmem + i * 128 + 8 * ks, dv + (uint64_t)(ks * (2048 >> 4)), idesc_o, (j | ks) != 0);
                        if (j + 1 < seg.n[i]) scores(i, kv_it + 1);
                        else umma_commit(&s.o_full[i]);
                    }
                    if (!ok) break;
                    umma_commit(&s.v_empty[kv_it & 1]);
                    if (j + 1 < n) umma_commit(&s.k_empty[(kv_it + 1) & 1]);
                }
            }
            if (*failed) {   // products in flight still write tensor memory and read shared memory
                umma_commit(&s.drain);
                const long long began = clock64();
                while (!mbar_try_wait(&s.drain, 0) && clock64() - began < kWaitCycles) {}
            }
        }
        __syncwarp();
    } else if constexpr (FP8) {
        // ------------------------------------------------------------------ converters
        const int tid = threadIdx.x - 320;
        constexpr int kPerRow = D / 16, kPer = T::kRawTokens * kPerRow / T::kConverters;   // 16-code chunks per row, per thread
        uint32_t kv_it = 0, raw_stage = 0, raw_parity = 0;
        int bearing = 0;
        bool ok = true;
        while (ok && walk.next(pp, seg)) {
            const int n = max(seg.n[0], seg.n[1]);
            if (n == 0) continue;
            const int buffer = bearing & (kBadBuffers - 1);
            ++bearing;
            for (int j = 0; ok && j < n; ++j, ++kv_it) {
                const int pos0 = (seg.tile0 + j) * kTileTokens, stage = kv_it & 1;
                const uint32_t reuse = ((kv_it >> 1) & 1) ^ 1u;
                const bool edge = pos0 + kTileTokens > seg.all_see;
#pragma unroll 1
                for (int part = 0; part < 4; ++part) {
                    const bool is_v = part >= 2;
                    const int half = (part & 1) * T::kRawTokens;
                    if (!(ok = wait_bar(&s.raw_full[raw_stage], raw_parity, failed))) break;
                    uint4 codes[kPer];
#pragma unroll
                    for (int it = 0; it < kPer; ++it)
                        codes[it] = *reinterpret_cast<const uint4 *>(s.raw[raw_stage] + (it * T::kConverters + tid) * 16);
                    mbar_arrive(&s.raw_empty[raw_stage]);
                    if (++raw_stage == T::kRawStages) { raw_stage = 0; raw_parity ^= 1u; }
                    if (is_v && edge) {
#pragma unroll
                        for (int it = 0; it < kPer; ++it) {
                            const int r = half + (it * T::kConverters + tid) / kPerRow, c = (it * T::kConverters + tid) % kPerRow;
                            uint32_t w[4] = {codes[it].x, codes[it].y, codes[it].z, codes[it].w};
                            if (pos0 + r >= seg.length) {
                                w[0] = w[1] = w[2] = w[3] = 0u;
                            } else if (pos0 + r >= seg.all_see) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t odd = __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                                    if (odd) {
                                        for (int y = 0; y < 4; ++y)
                                            if ((odd >> (8 * y)) & 1u) atomicMin(&s.bad[buffer][0][16 * c + 4 * k + y], pos0 + r);
                                        s.bad_any[buffer] = 1;
                                        w[k] &= ~odd;
                                    }
                                }
                            }
                            codes[it] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    if ((part & 1) == 0 && !(ok = wait_bar(is_v ? &s.v_empty[stage] : &s.k_empty[stage], reuse, failed))) break;
                    uint8_t *dst = is_v ? s.v[stage] : s.k[stage];
#pragma unroll
                    for (int it = 0; it < kPer; ++it) {
                        const int r = half + (it * T::kConverters + tid) / kPerRow, c = (it * T::kConverters + tid) % kPerRow;
                        uint4 lo, hi;
                        codes_to_f16(codes[it].x, lo.x, lo.y);
                        codes_to_f16(codes[it].y, lo.z, lo.w);
                        codes_to_f16(codes[it].z, hi.x, hi.y);
                        codes_to_f16(codes[it].w, hi.z, hi.w);
                        // the two panels' chunks alternate, so that eight lanes always write eight different bank groups
                        const bool second = D == 128 && c >= 4;
                        *reinterpret_cast<uint4 *>(dst + operand_chunk(r, 2 * c + (second ? 1 : 0))) = second ? hi : lo;
                        *reinterpret_cast<uint4 *>(dst + operand_chunk(r, 2 * c + (second ? 0 : 1))) = second ? lo : hi;
                    }
                    if (part & 1) {
                        fence_async_smem();
                        mbar_arrive(is_v ? &s.v_full[stage] : &s.k_full[stage]);
                    }
                }
            }
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (warp == 9) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (threadIdx.x == 0 && s.failed) atomicOr(bt.error, kErrorWait);
}

// Joins the parts of row blocks that several CTAs shared: one thread per row, a few columns per CTA.
constexpr int kJoinColumns = 16;
template <int D>
__global__ void __launch_bounds__(kBlockRows)
join_blocks_kernel(const PrefillParams pp, int grid) {
    pdl_launch_dependents();
    pdl_wait();
    const AttentionParams &p = pp.a;
    const Batch &bt = p.bt;
    const int b = blockIdx.x, head = blockIdx.y, d0 = blockIdx.z * kJoinColumns, r = threadIdx.x;
    const int u_seq = __ldg(p.prefix_out + b), units = __ldg(p.prefix_out + bt.seqs);
    if (__ldg(p.prefix_out + b + 1) == u_seq) return;
    const int ctas = working_ctas(grid, units);
    int first, count;
    rows_of(bt, b, first, count);
    const int length = length_of(bt, b), blocks = block_count(count, p.group, kBlockRows);
    int at = u_seq;
    for (int rb = 0; rb < blocks; ++rb) {
        const int tiles = max(block_tiles(length, count, p.group, kBlockRows, rb, kTileTokens), 1);
        const int u0 = at + head * tiles, u1 = u0 + tiles;
        at += tiles * p.hkv;
        const int c0 = owner(u0, ctas, units), c1 = owner(u1 - 1, ctas, units);
        if (c0 == c1 || r >= min(kBlockRows, count * p.group - rb * kBlockRows)) continue;
        auto part_of = [&](int c) { return p.partial + ((long long)c * 2 + (c == c0 ? 1 : 0)) * kBlockRows * (D + 2); };
        float top = -INFINITY;
        for (int c = c0; c <= c1; ++c) top = fmaxf(top, part_of(c)[D * kBlockRows + 2 * r]);
        const float base = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        float4 sum[kJoinColumns / 4];
#pragma unroll
        for (int k = 0; k < kJoinColumns / 4; ++k) sum[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int c = c0; c <= c1; ++c) {
            const float *src = part_of(c);
            const float2 ml = *reinterpret_cast<const float2 *>(src + D * kBlockRows + 2 * r);
            const float f = exp2_fast(ml.x - base);
            total = fmaf(ml.y, f, total);
#pragma unroll
            for (int k = 0; k < kJoinColumns / 4; ++k) {
                const float4 v = *reinterpret_cast<const float4 *>(src + ((d0 / 4 + k) * kBlockRows + r) * 4);
                sum[k].x = fmaf(v.x, f, sum[k].x); sum[k].y = fmaf(v.y, f, sum[k].y);
                sum[k].z = fmaf(v.z, f, sum[k].z); sum[k].w = fmaf(v.w, f, sum[k].w);
            }
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const int pair = rb * kBlockRows + r;
        bf16 *dst = p.out + ((long long)(first + pair / p.group) * p.hq + head * p.group + pair % p.group) * D + d0;
#pragma unroll
        for (int k = 0; k < kJoinColumns / 4; ++k)
            bo::store_bf16x4(dst + 4 * k, make_float4(sum[k].x * inv, sum[k].y * inv, sum[k].z * inv, sum[k].w * inv));
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

PrefillGrid prefill_grid(const Pool &pool, const Batch &bt, int hq, int min_count, int sms) {
    PrefillGrid g = {};
    const int group = hq / pool.kv_heads;
    const long long most = bt.cu ? bt.tokens : bt.per_seq;
    if (most < min_count) return g;   // no sequence can have as many rows
    const long long blocks = bt.cu ? (long long)bt.tokens * group / kBlockRows + bt.seqs : (long long)bt.seqs * block_count(bt.per_seq, group, kBlockRows);
    const long long tiles = (((long long)bt.max_pages << bt.page_shift) + kTileTokens - 1) / kTileTokens;
    // Two row blocks per SM or more (counted by rows, not by what a ragged batch could have at worst): one CTA each.
    g.whole = ((long long)bt.tokens * group / kBlockRows) * pool.kv_heads >= 2ll * sms || tiles == 1;
    const long long units = blocks * pool.kv_heads * (g.whole ? 1 : tiles);
    g.too_many = units > 0x7fffffffll;
    g.ctas = g.too_many ? 0 : g.whole || units < sms ? (int)units : sms;
    g.partial_floats = g.whole ? 0 : (long long)g.ctas * 2 * kBlockRows * (pool.head_dim + 2);
    return g;
}

template <int D, bool FP8>
static int launch_prefill_t(const PrefillParams &pp, const Pool &pool, const PrefillGrid &grid, cudaStream_t st) {
    using T = Prefill<D, FP8>;
    CUtensorMap map_k, map_v;
    const int most = FP8 ? T::kRawTokens : kTileTokens, box = pool.page_size < most ? pool.page_size : most;
    if (!make_pool_map(&map_k, pool, pool.k, box, !FP8) || !make_pool_map(&map_v, pool, pool.v, box, !FP8)) {
        set_last_error("mk_paged_attention: cuTensorMapEncodeTiled refused the cache (driver without tensor-map support?)");
        return MK_ERR_UNSUPPORTED;
    }
    const size_t smem = 1024 + sizeof(typename T::Smem) + (size_t)(pp.a.bt.seqs + 1) * sizeof(int);
    static bool allowed[64] = {};
    cudaError_t e = allow_smem((const void *)prefill_kernel<D, FP8>, allowed);
    if (e == cudaSuccess) e = launch_pdl(prefill_kernel<D, FP8>, dim3(grid.ctas), dim3(T::kThreads), smem, st, map_k, map_v, pp);
    if (e == cudaSuccess && !grid.whole)
        e = launch_pdl(join_blocks_kernel<D>, dim3(pp.a.bt.seqs, pp.a.hkv, D / kJoinColumns), dim3(kBlockRows), 0, st, pp, grid.ctas);
    return (int)e;
}

int launch_prefill(const AttentionParams &p, const Pool &pool, const PrefillGrid &grid, int min_count, cudaStream_t st) {
    PrefillParams pp;
    pp.a = p;
    pp.min_count = min_count;
    pp.whole = grid.whole ? 1 : 0;
    if (pool.head_dim == 64)
        return pool.fp8 ? launch_prefill_t<64, true>(pp, pool, grid, st) : launch_prefill_t<64, false>(pp, pool, grid, st);
    return pool.fp8 ? launch_prefill_t<128, true>(pp, pool, grid, st) : launch_prefill_t<128, false>(pp, pool, grid, st);
}

}  // namespace paged
}  // namespace mk
