// Attention over a paged cache for sequences with many new rows (prompts, chunks of prompts):
// the same operator as paged_attention.cu on the 5th-generation tensor cores.
//
// Shape of the work.  A row block is 256 (token, query head of the group) pairs of one sequence and KV
// head, two MMA tiles of 128 rows; the cache is loaded in tiles of 128 positions and worked off in steps of
// 64.  Per step and row tile:  S = Q K^T (tcgen05.mma, operands in shared memory, S in tensor memory),
// softmax weights P by one thread per row (tensor memory to registers and back, 16-bit), and
// O += P V (P from tensor memory, V in shared memory as it lies there: positions are rows, so
// it is an MN-major operand).  Everything a row needs is in one thread: no shuffles.
//
// What bounds it: per 128 rows x 128 positions the tensor core needs 4 x 128 x 128 x D flops - 1024 clocks at
// D = 128 - and the softmax 128 x 128 exponentials - 1024 clocks of the special function unit - and some 500
// instructions per warp.  To keep a row tile's threads from waiting for its products, S has two
// buffers of 64 columns per row tile: while one step's weights are made, the next step's scores are there
// already, and the one after takes the place of the weights as soon as their product is done.  The output is
// rescaled only when the running maximum has grown by more than 2^8 (E4M3: 2^4, its f16 weights are scaled by
// 2^11 besides and stay below 2^15) since the last time (sums are fp32), and only then do the softmax threads wait for the product before.
//
// Warp roles: 0-3 and 4-7 softmax of row tile 0 and 1 (and query loading, epilogue), 8 loader (TMA,
// one box per page), 9 and 10 MMA issue for one row tile each (9 also allocates tensor memory), 11 planner
// (finds the CTA's segments ahead of the others), and for the 8-bit cache 12-15
// converters: E4M3 codes land as they are in a small ring and become f16 (exact) in the swizzled
// operand tiles; queries are f16 scaled by a power of two per row, page scales enter at the scores
// and the value scale joins the exponent, as in paged_attention.cu.  A bf16 cache goes from TMA
// to the tensor core without passing a register; its weights are one bf16 term each (2^-8 of a weight, what the
// result's own rounding is: 4 prompts are 0.0017 of their norm off the 64-bit result, 0.0015 with fp32 weights; a second
// term would be half of the tensor work more and a longer chain).
//
// Values that are not finite and lie at positions some rows do not see (or behind the end) are
// taken out of the tile by the warp that fills it; rows that do see them get them in the epilogue.
//
// Work split.  One CTA per SM takes an equal consecutive range of units (tiles, and three for what a row
// block costs besides); the next row block's tiles are fetched during the last one's epilogue.
// Row blocks that a range's end cuts are joined by a second kernel.
//
// Measured (device time of this kernel + the join): 4 prompts of 333 to 3001 rows, bf16, 32 query and 8 KV heads,
// D = 128: 244 + 11 us, 0.73 PFLOP/s; 512 rows behind 8192 positions, E4M3: 99 + 8 us, 0.72 PFLOP/s.  The tensor
// pipe is busy for 35 to 37 % of the cycles and the special function unit as long: a row tile's step is one chain (scores
// from tensor memory, maximum, exponentials, weights to tensor memory, product), and two row tiles x two steps in
// flight do not fill the pipes between its parts.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/b200_megakernel.h"
#include "batched_ops.cuh"
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace mk {

void set_last_error(const char *msg);  // megakernel.cu

namespace paged {

constexpr int kTileTokens = 128;           // positions that are loaded at once
constexpr int kStepTokens = 64;            // positions of one product and softmax
constexpr int kBlockRows = 256;
constexpr int kPanelBytes = 128 * 128;     // 128 rows of one 128-byte swizzle row
constexpr int kChunks = kTileTokens / 16;  // a page is at least 16 positions
constexpr float kLeastFactor = 1.17549435e-38f;   // of a score: minus infinity (a masked score) times it stays what it is

// What the roles need of a segment besides its place.
struct Shape {
    int n[2];           // steps (half tiles) of the two row tiles in it
    int most;           // tiles that are loaded
    int all_see;        // positions that every row sees
};
// One segment as the planner hands it to the other roles.
struct Order {
    Segment seg;
    Shape shape;
    int valid;          // 0: there are no more
};
constexpr int kOrders = 4;

template <int D, bool FP8>
struct Prefill {
    static constexpr int kConverters = 128;
    static constexpr int kThreads = FP8 ? 512 : 384;
    // Registers per thread: 128 (four warpgroups) or 168 (three) at launch; a step's 64 scores stay in the softmax threads'
    // (184 or 208 there: no faster).
    static constexpr int kSoftmaxRegisters = 200, kOtherRegisters = FP8 ? 56 : 104;
    static_assert(2 * kSoftmaxRegisters + (FP8 ? 2 : 1) * kOtherRegisters <= (FP8 ? 4 * 128 : 3 * 168), "within the launch's registers");
    static constexpr float kGrowth = FP8 ? kPromptGrowth : 8.f;   // of the maximum that does not rescale the output
    static constexpr int kPanels = D / 64;
    static constexpr int kOperandBytes = kPanels * kPanelBytes;   // 128 rows x D two-byte elements
    static constexpr int kRawTokens = kTileTokens / 2, kRawStages = FP8 ? 3 : 1;
    static constexpr int kRawBytes = FP8 ? kRawTokens * D : 16;
    static constexpr int kBadKinds = FP8 ? 1 : 3;                 // E4M3 has NaN only
    // A tile-bearing segment's positions of values that are not finite, cleared by the loader when it comes to the segment and read
    // last in its epilogue.  What the loader may run ahead of the epilogues, segments of one tile each: E4M3 codes of segment n - 1
    // are all asked for once its first part is converted, so n - 2 is, for which the values' stage of n - 4 was free: that product
    // is done, its epilogue may be under way, the one of n - 5 is over (queries are loaded behind it).  bf16: the keys' stage of
    // n - 3 was free for n - 1, so the epilogue of n - 4 is over.
    static constexpr int kBadBuffers = FP8 ? 5 : 4;
    struct __align__(1024) Smem {
        uint8_t q[2][kOperandBytes];
        uint8_t k[2][kOperandBytes];
        uint8_t v[2][kOperandBytes];
        uint8_t raw[kRawStages][kRawBytes];
        uint64_t raw_full[kRawStages], raw_empty[kRawStages], k_full[2], k_empty[2], v_full[2], v_empty[2], v_raw;
        uint64_t order_full[kOrders], order_empty[kOrders];
        Order order[kOrders];
        uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2][2], drain[2];   // [row tile], [row tile][step mod 2]
        float ks[4][kChunks], ev[4][kChunks], iev[4][kChunks];   // by tile counter mod 4: key scale, log2 of the value scale and its inverse
        int bad[kBadBuffers][kBadKinds][D];                      // first position whose value in a column is NaN, +inf, -inf
        int bad_any[kBadBuffers];
        uint32_t tmem_base;
        int failed;
        int scan[kThreads / 32];
        int prefix[1];                                           // [seqs + 1]
    };
};

constexpr int kPrefillCost = 3;            // of a segment besides its tiles, in tiles (4 prompts with 2, 3, 5: 286, 274, 285 us when chosen)
__device__ constexpr Cut kPrefillCut = {kBlockRows, kTileTokens, kPrefillCost};

struct PrefillParams {
    AttentionParams a;
    int min_count;      // sequences with fewer new tokens are the other kernel's
};

__device__ __forceinline__ Shape shape_of(const AttentionParams &p, const Segment &s) {
    Shape h;
    h.all_see = visible(s.length, s.count, div(s.rb * kBlockRows, p.group));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int last = min(s.rows, 128 * (i + 1)) - 1;
        h.n[i] = 0;
        if (last >= 128 * i) {
            const int seen = visible(s.length, s.count, div(s.rb * kBlockRows + last, p.group));
            h.n[i] = max(min((seen + kStepTokens - 1) / kStepTokens, 2 * s.tile1) - 2 * s.tile0, 0);
        }
    }
    h.most = (max(h.n[0], h.n[1]) + 1) / 2;
    return h;
}

// Whether one of the positions below `limit` in a segment lies in a page of the pool.
__device__ __forceinline__ bool any_page(const Batch &bt, const Segment &s, int limit) {
    const int end = min(s.tile1 * kTileTokens, limit);
#pragma unroll 1
    for (int pos = s.tile0 * kTileTokens; pos < end; pos += 16) {
        const int id = __ldg(bt.table + s.b * bt.table_stride + (pos >> bt.page_shift));
        if (id >= 0 && id < bt.num_pages) return true;
    }
    return false;
}

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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float v;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// byte offset of 16-byte chunk c of row r in an operand tile (panels of 64 elements, 128-byte swizzle)
__device__ __forceinline__ uint32_t operand_chunk(int r, int c) { return (c >> 3) * kPanelBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

template <int D, bool FP8>
__global__ void __launch_bounds__(Prefill<D, FP8>::kThreads, 1)
prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefillParams pp) {
    using T = Prefill<D, FP8>;
    using Smem = typename T::Smem;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &s = *reinterpret_cast<Smem *>(smem_raw);
    const AttentionParams &p = pp.a;
    const Batch &bt = p.bt;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *failed = &s.failed;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.k_full[i], FP8 ? T::kConverters : 1);
            mbar_init(&s.v_full[i], FP8 ? T::kConverters : 1);
            mbar_init(&s.k_empty[i], 2);   // one arrival per row tile
            mbar_init(&s.v_empty[i], 2);
            mbar_init(&s.q_full[i], 128);
            for (int h = 0; h < 2; ++h) {
                mbar_init(&s.s_full[i][h], 1);
                mbar_init(&s.p_full[i][h], 128);
                mbar_init(&s.o_done[i][h], 1);
            }
        }
        for (int i = 0; i < T::kRawStages; ++i) {
            mbar_init(&s.raw_full[i], 1);
            mbar_init(&s.raw_empty[i], T::kConverters);
        }
        for (int i = 0; i < kOrders; ++i) {
            mbar_init(&s.order_full[i], 1);
            mbar_init(&s.order_empty[i], 8 + 1 + 2 + (FP8 ? T::kConverters / 32 : 0));   // softmax and converter warps, loader, MMA
        }
        mbar_init(&s.v_raw, 1);
        mbar_init(&s.drain[0], 1);
        mbar_init(&s.drain[1], 1);
        s.failed = 0;
        fence_barrier_init();
    }
    pdl_wait();
    Walk walk;
    plan_walk<T::kThreads>(bt, p.hkv, p.group, kPrefillCut, pp.min_count, 0x7fffffff, s.prefix, s.scan, walk);
    if (walk.u >= walk.u_end) {   // the whole CTA
        if (threadIdx.x == 0) p.entries[blockIdx.x] = JoinEntry{0, 0, 0, 0};
        return;
    }
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
    Shape shape;
    uint32_t orders = 0;   // taken so far
    // The next segment from the planner; `arrives`: this thread gives the entry back for its warp.
    auto advance = [&](bool arrives) {
        const int at = orders & (kOrders - 1);
        if (!wait_bar(&s.order_full[at], (orders / kOrders) & 1, failed)) return false;
        seg = s.order[at].seg;
        shape = s.order[at].shape;
        const bool valid = s.order[at].valid != 0;
        ++orders;
        if (arrives) mbar_arrive(&s.order_empty[at]);
        return valid;
    };
    auto advance_warp = [&]() {   // all lanes
        const int at = orders & (kOrders - 1);
        const bool valid = __all_sync(0xffffffffu, advance(false));
        if (lane == 0) mbar_arrive(&s.order_empty[at]);
        return valid;
    };
    if (warp < 8) {
        take_registers<T::kSoftmaxRegisters>();
        // ------------------------------------------------------------------ softmax of one row tile
        const int i = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_tm = tmem + lanes + i * 128, o_tm = tmem + lanes + 256 + i * 128;
        uint32_t s_parity = 0;           // bit h: of the scores of steps with that parity
        uint32_t o_parity = 0;           // bit h: of the last product of steps with that parity, once it is asked for
        // Waits for the product of the step before, the latest of its parity: one may be under way, not two, since the scores
        // of a step follow the product two steps before it.
        auto wait_output = [&](int h) {
            const bool done = __all_sync(0xffffffffu, wait_bar(&s.o_done[i][h], ((o_parity >> h) & 1) ^ 1u, failed));
            tcgen05_fence_after();
            return done;
        };
        int tile_ctr = 0, bearing = 0;   // tiles and tile-bearing segments of this CTA so far
        bool ok = true;
        // Queries: a warp loads its 32 rows side by side, kLanes lanes per row, so that a request
        // touches few lines; thread `lane` then looks after row `lane`.
        constexpr int kLanes = D / 8, kStep = 32 / kLanes, kLoads = 32 / kStep;
        const int chunk = lane % kLanes, sub = lane / kLanes, row0 = row - lane;
        while (ok && advance_warp()) {
            const int r = 128 * i + row, pair = seg.rb * kBlockRows + r;
            const bool real = r < seg.rows;
            const int token = real ? div(pair, p.group) : 0;
            // the query row into the operand tile (its last products are done: this row tile's output was waited for)
            float c_row = fabsf(p.scale_log2e);
            {
                const bool negate = p.scale_log2e < 0.f;   // scores are compared as they come, so their factor is kept positive
                int e_row = 0;
                uint4 raw[kLoads];
#pragma unroll
                for (int it = 0; it < kLoads; ++it) {
                    const int rr = 128 * i + row0 + it * kStep + sub, pr = seg.rb * kBlockRows + rr, tk = div(pr, p.group);
                    const bf16 *qp = p.q + (long long)(seg.first + tk) * p.q_token + (long long)(seg.head * p.group.d + pr - tk * p.group.d) * p.q_head;
                    raw[it] = rr < seg.rows ? __ldg(reinterpret_cast<const uint4 *>(qp) + chunk) : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int it = 0; it < kLoads; ++it) {
                    uint4 w = raw[it];
                    if constexpr (FP8) {
                        float x[8], amax = 0.f;
                        unpack8(raw[it], x);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float a = fabsf(x[k]);
                            if (a < INFINITY) amax = fmaxf(amax, a);
                        }
#pragma unroll
                        for (int off = kLanes / 2; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
                        const int e = max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -120);   // amax / 2^e in [2^14, 2^15)
                        const float factor = __uint_as_float((uint32_t)(127 - e) << 23) * (negate ? -1.f : 1.f);
                        w = make_uint4(pack_f16(x[0] * factor, x[1] * factor), pack_f16(x[2] * factor, x[3] * factor),
                                       pack_f16(x[4] * factor, x[5] * factor), pack_f16(x[6] * factor, x[7] * factor));
                        const int mine = __shfl_sync(0xffffffffu, e, (lane % kStep) * kLanes);
                        if (lane / kStep == it) e_row = mine;
                    } else if (negate) {
                        w.x ^= 0x80008000u; w.y ^= 0x80008000u; w.z ^= 0x80008000u; w.w ^= 0x80008000u;
                    }
                    *reinterpret_cast<uint4 *>(s.q[i] + operand_chunk(row0 + it * kStep + sub, chunk)) = w;
                }
                if constexpr (FP8) c_row *= __uint_as_float((uint32_t)(127 + e_row) << 23);
                fence_async_smem();
                mbar_arrive(&s.q_full[i]);
            }
            const int limit = real ? visible(seg.length, seg.count, token) : 0;
            const int all_see = visible(seg.length, seg.count, div(seg.rb * kBlockRows + 128 * i, p.group));
            float m = -INFINITY, l = 0.f;
            const int n = shape.n[i];

#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                const int h = j & 1;     // tile j / 2 of the segment, half h
                ok = __all_sync(0xffffffffu, wait_bar(&s.s_full[i][h], (s_parity >> h) & 1, failed));
                if (!ok) break;
                s_parity ^= 1u << h;
                tcgen05_fence_after();
                const int slot = (tile_ctr + j / 2) & 3, pos0 = (2 * seg.tile0 + j) * kStepTokens;
                const int lim = limit - pos0;   // columns below it are seen
                const uint32_t s_h = s_tm + h * kStepTokens;
                uint32_t x[2][32];
                tmem_load32(s_h, x[0]);
                tmem_load32(s_h + 32, x[1]);
                tmem_load_wait(x[0]);
                after_wait(x[1]);
                if (pos0 + kStepTokens > all_see) {
#pragma unroll
                    for (int k = 0; k < kStepTokens; ++k)
                        if (k >= lim) x[k / 32][k % 32] = 0xff800000u;   // -inf
                }
                // largest score; 16 positions share a page and so a key scale c and a value scale 2^e.  NaN stays NaN, and
                // with it the row.
                float c[4], e[4], top = -INFINITY;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    c[g] = fmaxf(c_row * s.ks[slot][4 * h + g], kLeastFactor);
                    e[g] = s.ev[slot][4 * h + g];
                    const uint32_t *y = &x[g / 2][16 * (g & 1)];
                    float a = __uint_as_float(y[0]), b = __uint_as_float(y[1]);
#pragma unroll
                    for (int k = 2; k < 14; k += 4) {
                        a = max3_nan(a, __uint_as_float(y[k]), __uint_as_float(y[k + 1]));
                        b = max3_nan(b, __uint_as_float(y[k + 2]), __uint_as_float(y[k + 3]));
                    }
                    a = max3_nan(max3_nan(a, __uint_as_float(y[14]), __uint_as_float(y[15])), b, b);
                    top = max3_nan(top, top, fmaf(a, c[g], e[g]));
                }
                // the running maximum, and the output if it has grown too much
                {
                    const float grown = max3_nan(m, m, top);
                    const bool need = !(grown <= m + T::kGrowth);   // also from -inf, and NaN
                    if (j == 0) {
                        m = grown;
                    } else if (__any_sync(0xffffffffu, need)) {
                        if (!(ok = wait_output(h ^ 1))) break;
                        const float corr = need ? exp2_fast(m - (grown == -INFINITY ? 0.f : grown)) : 1.f;
                        if (need) m = grown;
                        l *= corr;
#pragma unroll 1
                        for (int ch = 0; ch < D / 16; ++ch) {
                            uint32_t o[16];
                            tmem_load16(o_tm + 16 * ch, o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                            tmem_store16(o_tm + 16 * ch, o);
                        }
                    }
                }
                const float base = (m == -INFINITY ? 0.f : m == INFINITY ? __int_as_float(0x7fffffff) : m) - (FP8 ? kPromptWeight : 0.f);
                // weights, in the place of the scores
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) {
                    uint32_t w[16];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int g = 2 * ch + half;
                        const uint64_t cc = pair_f32(c[g], c[g]), ee = pair_f32(e[g] - base, e[g] - base);
                        uint64_t sum = 0;
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            float w0, w1;
                            split_f32(fma_f32x2(pair_f32(__uint_as_float(x[ch][16 * half + k]), __uint_as_float(x[ch][16 * half + k + 1])), cc, ee), w0, w1);
                            w0 = exp2_fast(w0);
                            w1 = exp2_fast(w1);
                            sum = add_f32x2(sum, pair_f32(w0, w1));
                            w[8 * half + k / 2] = FP8 ? pack_f16(w0, w1) : pack_b16(w0, w1);
                        }
                        float s0, s1;
                        split_f32(sum, s0, s1);
                        l = fmaf(FP8 ? (s0 + s1) * kPromptUnscale : s0 + s1, s.iev[slot][4 * h + g], l);
                    }
                    tmem_store16(s_h + 16 * ch, w);
                }
                tmem_store_wait();
                tcgen05_fence_before();
                mbar_arrive(&s.p_full[i][h]);
                o_parity ^= 1u << h;
            }
            tile_ctr += shape.most;
            if (!ok) break;

            // epilogue
            if (l != l && !any_page(bt, seg, limit)) {   // a query that is not finite times the zeros of pages that are not there
                m = -INFINITY;
                l = 0.f;
            }
            if (n == 0) o_parity ^= 1u;   // a segment without steps counts one, so that this row tile is never ahead of it
            if (!(ok = wait_output(n > 0 ? (n - 1) & 1 : 0))) break;
            const int buffer = bearing % T::kBadBuffers;
            const bool bad = n > 0 && (volatile int &)s.bad_any[buffer] != 0;
            if (shape.most > 0) ++bearing;
            const bool complete = seg.begins && seg.ends;
            float *part = p.partial + ((long long)blockIdx.x * 2 + (seg.begins ? 1 : 0)) * kBlockRows * (D + 2);
            uint32_t x[D / 32][32];
            if (n > 0) {
#pragma unroll
                for (int ch = 0; ch < D / 32; ++ch) tmem_load32(o_tm + 32 * ch, x[ch]);
                tmem_load_wait(x[0]);
#pragma unroll
                for (int ch = 1; ch < D / 32; ++ch) after_wait(x[ch]);
            } else {
#pragma unroll
                for (int k = 0; k < D; ++k) x[k / 32][k % 32] = 0u;
            }
            if (l == 0.f) {   // nothing seen
#pragma unroll
                for (int k = 0; k < D; ++k) x[k / 32][k % 32] = 0u;
            }
            if (bad) {
#pragma unroll
                for (int k = 0; k < D; ++k) {
                    float y = __uint_as_float(x[k / 32][k % 32]);
                    if ((volatile int &)s.bad[buffer][0][k] < limit) y = __int_as_float(0x7fffffff);
                    if constexpr (!FP8) {
                        if ((volatile int &)s.bad[buffer][1][k] < limit) y += INFINITY;
                        if ((volatile int &)s.bad[buffer][2][k] < limit) y -= INFINITY;
                    }
                    x[k / 32][k % 32] = __float_as_uint(y);
                }
            }
            const float inv = l == 0.f ? 0.f : (FP8 ? kPromptUnscale : 1.f) / l;
            if (complete) {   // through the query tile, which is idle now, to whole lines of the output
#pragma unroll
                for (int k = 0; k < D; k += 8) {
                    const uint32_t *y = &x[k / 32][k % 32];
                    uint4 v;
                    v.x = pack_b16(__uint_as_float(y[0]) * inv, __uint_as_float(y[1]) * inv);
                    v.y = pack_b16(__uint_as_float(y[2]) * inv, __uint_as_float(y[3]) * inv);
                    v.z = pack_b16(__uint_as_float(y[4]) * inv, __uint_as_float(y[5]) * inv);
                    v.w = pack_b16(__uint_as_float(y[6]) * inv, __uint_as_float(y[7]) * inv);
                    *reinterpret_cast<uint4 *>(s.q[i] + operand_chunk(row, k / 8)) = v;
                }
                __syncwarp();
#pragma unroll 4
                for (int it = 0; it < kLoads; ++it) {
                    const int rr = row0 + it * kStep + sub, pr = seg.rb * kBlockRows + 128 * i + rr, tk = div(pr, p.group);
                    if (128 * i + rr < seg.rows)
                        *reinterpret_cast<uint4 *>(p.out + ((long long)(seg.first + tk) * p.hq + seg.head * p.group.d + pr - tk * p.group.d) * D + 8 * chunk) =
                            *reinterpret_cast<const uint4 *>(s.q[i] + operand_chunk(rr, chunk));
                }
                __syncwarp();
            } else if (real) {   // four columns of 256 rows side by side
#pragma unroll
                for (int k = 0; k < D; k += 4) {
                    const uint32_t *y = &x[k / 32][k % 32];
                    *reinterpret_cast<uint4 *>(part + (k / 4 * kBlockRows + r) * 4) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
            if (real && !complete) *reinterpret_cast<float2 *>(part + D * kBlockRows + 2 * r) = make_float2(m, l);
        }
    } else {
    give_up_registers<T::kOtherRegisters>();
    if (warp == 8) {
        // ------------------------------------------------------------------ loader
        uint32_t kv_it = 0, raw_stage = 0, raw_parity = 0, raw_fills = 0, v_raw_parity = 0;
        int bearing = 0;
        bool ok = true;
        while (ok && advance_warp()) {
            const int n = shape.most;
            if (n == 0) continue;
            const int buffer = bearing % T::kBadBuffers;
            ++bearing;
            for (int c = lane; c < T::kBadKinds * D; c += 32) (&s.bad[buffer][0][0])[c] = 0x7fffffff;
            if (lane == 0) s.bad_any[buffer] = 0;
            __syncwarp();
            const int *table = bt.table + seg.b * bt.table_stride;
            // table entry of 16-position chunk `lane` of a tile; used, and checked, two tiles later
            auto entry_of = [&](int j) {
                const int pos = (seg.tile0 + j) * kTileTokens + 16 * lane;
                return lane < kChunks && j < n && pos < seg.length ? __ldg(table + (pos >> bt.page_shift)) : -1;
            };
            auto checked = [&](int id) {
                if (id >= bt.num_pages) atomicOr(bt.error, kErrorIndex);
                return id >= 0 && id < bt.num_pages ? id : -1;
            };
            // scales of a tile's pages, as they lie in memory
            auto scales_of = [&](int id, float &ks, float &vs) {
                ks = 1.f;
                vs = 1.f;
                if (FP8 && id >= 0) {
                    const long long at = (long long)id * p.hkv + seg.head;
                    ks = __ldg(p.k_scales + at);
                    vs = __ldg(p.v_scales + at);
                }
            };
            // page ids are fetched two tiles ahead, scales one
            int page = entry_of(0), page_next = entry_of(1);
            page = checked(page);
            float ks_raw, vs_raw;
            scales_of(page, ks_raw, vs_raw);
            for (int j = 0; j < n; ++j, ++kv_it) {
                const int page_after = entry_of(j + 2);
                page_next = checked(page_next);
                float ks_next, vs_next;
                scales_of(page_next, ks_next, vs_next);
                const int pos0 = (seg.tile0 + j) * kTileTokens, stage = kv_it & 1, slot = kv_it & 3;
                const uint32_t reuse = ((kv_it >> 1) & 1) ^ 1u;   // parity of the stage's last release
                const float vs = fmaxf(vs_raw, 0x1p-100f), ks = ks_raw;
                const float ev = page < 0 ? -INFINITY : FP8 ? log2f(vs) : 0.f, iev = page < 0 ? 0.f : FP8 ? 1.f / vs : 1.f;

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
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(&s.k_full[stage], T::kOperandBytes);
                    __syncwarp();
                    boxes(s.k[stage], &map_k, &s.k_full[stage], 0, kTileTokens);
                    ok = __all_sync(0xffffffffu, wait_bar(&s.v_empty[stage], reuse, failed));
                    if (!ok) break;
                    const bool edge = pos0 + kTileTokens > shape.all_see;   // some rows do not see all of it
                    uint64_t *bar = edge ? &s.v_raw : &s.v_full[stage];
                    if (lane == 0) mbar_arrive_expect_tx(bar, T::kOperandBytes);
                    __syncwarp();
                    boxes(s.v[stage], &map_v, bar, 0, kTileTokens);
                    if (edge) {
                        ok = __all_sync(0xffffffffu, wait_bar(&s.v_raw, v_raw_parity, failed));
                        if (!ok) break;
                        v_raw_parity ^= 1u;
                        const int from = max(shape.all_see - pos0, 0), end = min(max(seg.length - pos0, 0), kTileTokens);
                        // anything that is not finite among the positions that only some rows see?
                        uint32_t odd = 0;
#pragma unroll 8
                        for (int idx = from * (D / 8) + lane; idx < end * (D / 8); idx += 32) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(s.v[stage] + operand_chunk(idx / (D / 8), idx % (D / 8)));
                            odd |= not_finite_b16(v.x) | not_finite_b16(v.y) | not_finite_b16(v.z) | not_finite_b16(v.w);
                        }
                        if (__any_sync(0xffffffffu, odd != 0)) {
                            for (int idx = from * (D / 8) + lane; idx < end * (D / 8); idx += 32) {
                                const int r = idx / (D / 8), c = idx % (D / 8);
                                uint4 *at = reinterpret_cast<uint4 *>(s.v[stage] + operand_chunk(r, c));
                                const uint4 v = *at;
                                uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const uint32_t bits = (w[k / 2] >> (16 * (k & 1))) & 0xffffu;
                                    if ((bits & 0x7f80u) == 0x7f80u) {
                                        atomicMin(&s.bad[buffer][(bits & 0x7fu) ? 0 : (bits & 0x8000u) ? 2 : 1][8 * c + k], pos0 + r);
                                        w[k / 2] &= ~(0xffffu << (16 * (k & 1)));
                                    }
                                }
                                *at = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                            s.bad_any[buffer] = 1;
                        }
                        for (int idx = end * (D / 8) + lane; idx < kTileTokens * (D / 8); idx += 32)   // behind the end: anything may lie there
                            *reinterpret_cast<uint4 *>(s.v[stage] + operand_chunk(idx / (D / 8), idx % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&s.v_full[stage]);
                    }
                }
                page = page_next;
                page_next = page_after;
                ks_raw = ks_next;
                vs_raw = vs_next;
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
    } else if (warp == 9 || warp == 10) {
        // ------------------------------------------------------------------ MMA issue for one row tile
        if (lane == 0) {
            const int i = warp - 9;
            const uint32_t idesc_s = umma_idesc16(!FP8, kStepTokens, false), idesc_o = umma_idesc16(!FP8, D, true);
            const uint32_t s_tm = tmem + i * 128, o_tm = tmem + 256 + i * 128;
            uint32_t kv_it = 0, q_parity = 0, p_parity = 0;
            bool ok = true;
            const uint64_t dq = smem_desc_k_major_sw128(s.q[i]), dk0 = smem_desc_k_major_sw128(s.k[0]);
            const uint64_t dv0 = smem_desc_mn_major_sw128(s.v[0], kPanelBytes);
            constexpr uint64_t kHalf = (uint64_t)(kStepTokens * 128 >> 4);   // 64 positions further in a key or value tile
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                ok = ok && wait_bar(bar, parity, failed);
                return ok;
            };
            // S = Q K^T of half h of tile t
            auto scores = [&](uint32_t t, int h) {
                const uint64_t dk = dk0 + (t & 1) * (T::kOperandBytes >> 4) + h * kHalf;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t at = (uint64_t)((ks >> 2) * (kPanelBytes >> 4) + (ks & 3) * 2);
                    umma16_ss(s_tm + h * kStepTokens, dq + at, dk + at, idesc_s, ks != 0);
                }
                umma_commit(&s.s_full[i][h]);
            };
            // gives a stage back once this row tile's products with it are done (or at once where it has none)
            auto release = [&](uint64_t *empty, bool used) {
                if (used) umma_commit(empty);
                else mbar_arrive(empty);
            };
            while (ok && advance(true)) {
                if (!wait(&s.q_full[i], q_parity)) break;
                q_parity ^= 1u;
                const int n = shape.n[i];
                if (n == 0) mbar_arrive(&s.o_done[i][0]);
                if (shape.most == 0) continue;
                if (!wait(&s.k_full[kv_it & 1], (kv_it >> 1) & 1)) break;
                tcgen05_fence_after();
                if (n > 0) scores(kv_it, 0);
                if (n > 1) scores(kv_it, 1);
                release(&s.k_empty[kv_it & 1], n > 0);
                for (int j = 0; ok && j < shape.most; ++j, ++kv_it) {
                    const uint32_t stage = kv_it & 1;
                    if (!wait(&s.v_full[stage], (kv_it >> 1) & 1)) break;
                    const uint64_t dv = dv0 + stage * (T::kOperandBytes >> 4);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int step = 2 * j + h;
                        if (step < n) {
                            if (!wait(&s.p_full[i][h], (p_parity >> h) & 1)) break;
                            p_parity ^= 1u << h;
                            tcgen05_fence_after();
#pragma unroll
                            for (int ks = 0; ks < kStepTokens / 16; ++ks)   // 16 positions: 16 rows of 128 bytes, 8 columns of weights
                                umma16_ts(o_tm, s_tm + h * kStepTokens + 8 * ks, dv + h * kHalf + (uint64_t)(ks * (2048 >> 4)), idesc_o, (step | ks) != 0);
                            umma_commit(&s.o_done[i][h]);
                        }
                        if (j + 1 < shape.most) {   // the step after next takes the place of these weights
                            if (h == 0) {
                                if (!wait(&s.k_full[stage ^ 1], ((kv_it + 1) >> 1) & 1)) break;
                                tcgen05_fence_after();
                            }
                            if (step + 2 < n) scores(kv_it + 1, h);
                            if (h == 1) release(&s.k_empty[stage ^ 1], 2 * j + 2 < n);
                        }
                    }
                    if (!ok) break;
                    release(&s.v_empty[stage], 2 * j < n);
                }
            }
            if (*failed) {   // products in flight still write tensor memory and read shared memory
                umma_commit(&s.drain[i]);
                const long long began = clock64();
                while (!mbar_try_wait(&s.drain[i], 0) && clock64() - began < kWaitCycles) {}
            }
        }
        __syncwarp();
    } else if (warp == 11) {
        // ------------------------------------------------------------------ planner
        if (lane == 0) {
            JoinEntry entry = {0, 0, 0, 0};
            bool more = true;
            while (more) {
                more = next_segment(bt, p.hkv, p.group, kPrefillCut, walk, seg);
                if (more) {
                    shape = shape_of(p, seg);
                    if (seg.parts > 1) entry = JoinEntry{seg.parts, seg.first, seg.rb * kBlockRows, (seg.head << 16) | seg.rows};
                }
                const int at = orders & (kOrders - 1);
                if (!wait_bar(&s.order_empty[at], ((orders / kOrders) & 1) ^ 1u, failed)) break;
                s.order[at].seg = seg;
                s.order[at].shape = shape;
                s.order[at].valid = more ? 1 : 0;
                mbar_arrive(&s.order_full[at]);
                ++orders;
            }
            p.entries[blockIdx.x] = entry;
        }
        __syncwarp();
    } else if (FP8 && warp >= 12) {
        // ------------------------------------------------------------------ converters
        const int tid = threadIdx.x - 384;
        constexpr int kPerRow = D / 16, kPer = T::kRawTokens * kPerRow / T::kConverters;   // 16-code chunks per row, per thread
        uint32_t kv_it = 0, raw_stage = 0, raw_parity = 0;
        int bearing = 0;
        bool ok = true;
        while (ok && advance_warp()) {
            const int n = shape.most;
            if (n == 0) continue;
            const int buffer = bearing % T::kBadBuffers;
            ++bearing;
            for (int j = 0; ok && j < n; ++j, ++kv_it) {
                const int pos0 = (seg.tile0 + j) * kTileTokens, stage = kv_it & 1;
                const uint32_t reuse = ((kv_it >> 1) & 1) ^ 1u;
                const bool edge = pos0 + kTileTokens > shape.all_see;
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
                            } else if (pos0 + r >= shape.all_see) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if (not_finite_e4m3(w[k])) {
                                        for (int y = 0; y < 4; ++y)
                                            if (((w[k] >> (8 * y)) & 0x7fu) == 0x7fu) {
                                                atomicMin(&s.bad[buffer][0][16 * c + 4 * k + y], pos0 + r);
                                                w[k] &= ~(0xffu << (8 * y));
                                            }
                                        s.bad_any[buffer] = 1;
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
    }

    tcgen05_fence_before();
    __syncthreads();
    if (warp == 9) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (threadIdx.x == 0 && s.failed) atomicOr(bt.error, kErrorWait);
}

// Joins the parts of the row block that begins in CTA blockIdx.x's range, if there is one: one thread per
// row, a few columns per CTA.
constexpr int kJoinColumns = 16;
template <int D>
__global__ void __launch_bounds__(kBlockRows)
join_blocks_kernel(const AttentionParams p) {
    pdl_wait();   // and no early start for the next kernel: see paged.cuh
    const int4 raw = __ldg(reinterpret_cast<const int4 *>(p.entries + blockIdx.x));
    const JoinEntry e = {raw.x, raw.y, raw.z, raw.w};
    const int d0 = blockIdx.y * kJoinColumns, r = threadIdx.x, head = e.head_rows >> 16;
    if (e.parts == 0 || r >= (e.head_rows & 0xffff)) return;
    auto part_of = [&](int i) { return p.partial + ((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kBlockRows * (D + 2); };
    float top = -INFINITY, total = 0.f;
    float4 sum[kJoinColumns / 4];
#pragma unroll
    for (int k = 0; k < kJoinColumns / 4; ++k) sum[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int i = 0; i < e.parts; ++i) {
        const float *src = part_of(i);
        const float2 ml = *reinterpret_cast<const float2 *>(src + D * kBlockRows + 2 * r);
        const float now = fmaxf(top, ml.x), base = now == -INFINITY ? 0.f : now;
        const float corr = exp2_fast(top - base), f = exp2_fast(ml.x - base);
        top = now;
        total = fmaf(total, corr, ml.y * f);
#pragma unroll
        for (int k = 0; k < kJoinColumns / 4; ++k) {
            const float4 v = *reinterpret_cast<const float4 *>(src + ((d0 / 4 + k) * kBlockRows + r) * 4);
            sum[k].x = fmaf(sum[k].x, corr, v.x * f); sum[k].y = fmaf(sum[k].y, corr, v.y * f);
            sum[k].z = fmaf(sum[k].z, corr, v.z * f); sum[k].w = fmaf(sum[k].w, corr, v.w * f);
        }
    }
    const float inv = total == 0.f ? 0.f : (p.k_scales ? kPromptUnscale : 1.f) / total;   // E4M3: the parts' outputs are scaled
    const int pair = e.pair + r;
    bf16 *dst = p.out + ((long long)(e.row + div(pair, p.group)) * p.hq + head * p.group.d + pair - div(pair, p.group) * p.group.d) * D + d0;
#pragma unroll
    for (int k = 0; k < kJoinColumns / 4; ++k)
        bo::store_bf16x4(dst + 4 * k, make_float4(sum[k].x * inv, sum[k].y * inv, sum[k].z * inv, sum[k].w * inv));
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
    const long long units = blocks * pool.kv_heads * (tiles + kPrefillCost);
    g.too_many = units >= 0x7fffffffll;
    g.ctas = g.too_many ? 0 : units < sms ? (int)units : sms;
    g.partial_floats = (long long)g.ctas * 2 * kBlockRows * (pool.head_dim + 2);
    return g;
}

template <int D, bool FP8>
static int launch_prefill_t(const PrefillParams &pp, const Pool &pool, const PrefillGrid &grid, cudaStream_t st) {
    using T = Prefill<D, FP8>;
    using Smem = typename T::Smem;
    CUtensorMap map_k, map_v;
    const int most = FP8 ? T::kRawTokens : kTileTokens, box = pool.page_size < most ? pool.page_size : most;
    if (!make_pool_map(&map_k, pool, pool.k, box, !FP8) || !make_pool_map(&map_v, pool, pool.v, box, !FP8)) {
        set_last_error("mk_paged_attention: cuTensorMapEncodeTiled refused the cache (driver without tensor-map support?)");
        return MK_ERR_UNSUPPORTED;
    }
    static_assert(offsetof(Smem, prefix) + (MK_PAGED_ATTENTION_MAX_SEQS + 1) * sizeof(int) <= 227 * 1024, "shared memory of a block");
    const size_t smem = offsetof(Smem, prefix) + (size_t)(pp.a.bt.seqs + 1) * sizeof(int);
    static bool allowed[64] = {};
    cudaError_t e = allow_smem((const void *)prefill_kernel<D, FP8>, allowed);
    if (e == cudaSuccess) e = launch_pdl(prefill_kernel<D, FP8>, dim3(grid.ctas), dim3(T::kThreads), smem, st, map_k, map_v, pp);
    if (e == cudaSuccess) e = launch_pdl(join_blocks_kernel<D>, dim3(grid.ctas, D / kJoinColumns), dim3(kBlockRows), 0, st, pp.a);
    return (int)e;
}

int launch_prefill(const AttentionParams &p, const Pool &pool, const PrefillGrid &grid, int min_count, cudaStream_t st) {
    PrefillParams pp;
    pp.a = p;
    pp.min_count = min_count;
    if (pool.head_dim == 64)
        return pool.fp8 ? launch_prefill_t<64, true>(pp, pool, grid, st) : launch_prefill_t<64, false>(pp, pool, grid, st);
    return pool.fp8 ? launch_prefill_t<128, true>(pp, pool, grid, st) : launch_prefill_t<128, false>(pp, pool, grid, st);
}

}  // namespace paged
}  // namespace mk
