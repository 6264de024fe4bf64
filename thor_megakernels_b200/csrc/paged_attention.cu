// Attention over a paged cache (bf16, or E4M3 with one scale per page and KV head): causal
// queries at the end of every sequence, grouped query heads, any number of rows.
//
//   s[r, j] = scale * ks(page j) * q_r . k_j    for the positions j that row r sees
//   out_r   = sum_j 2^(x_rj - m) vs(page j) v_j / sum_j 2^(x_rj - m),   x = s log2 e
//
// in one pass with a running maximum.  A row that sees nothing gives zeros.
//
// What bounds it.  With one or a few query tokens per sequence every cache byte is used for
// a handful of rows: the kernel has to keep HBM busy and spend few instructions per byte.
//   * Every warp is a worker of its own: it fills a private ring of shared-memory tiles (16 or
//     32 positions of keys and values) with tiled TMA copies, one lane issuing, and no warp
//     waits for another until the end of a segment.  The copies swizzle, so ldmatrix reads are
//     free of bank conflicts, and read any page / head / slot pitch.  A page id outside the pool
//     is outside the tensor map: the copy fills zeros.
//   * Products are mma.sync.m16n8k16 with the CACHE as the 16-row operand (positions for the
//     scores, head dimensions for the output) and the query rows as the 8 columns: a group of 4
//     to 8 query heads fills the narrow side, so a cache element costs half the tensor
//     instructions of the usual orientation.  The score fragment becomes the second product's
//     operand through movmatrix (an 8x8 transpose inside the warp).  Both accumulators keep
//     query rows in the same register positions: rescaling needs no shuffles.
//   * E4M3 codes become f16 in registers (exact).  For keys, four consecutive codes of a row are
//     one register; the columns' order inside a 16-wide step is then a permutation that the query
//     fragment shares.  Values come through ldmatrix.trans on pairs of codes: one byte shuffle
//     and two conversions give the fragment of even and odd columns.  Query rows enter as f16
//     scaled by a power of two per row (exact for elements within 2^-31 of the row's largest).
//   * The value scale joins the exponent: x + log2 vs is what the maximum runs over, so a weight
//     that meets a page of large values is large in f16.  f16 weights are scaled by 2^14: eleven
//     bits down to 2^-28 of the largest, nothing below 2^-39, half of f16's smallest number.
//     The sum of the weights is taken in fp32 without the value scale.
//   * A bf16 cache keeps bf16 operands; a weight enters as two terms (value and remainder).
//
// Work split.  Units of (row block, KV head, tile of 4 warp tiles) are dealt to the resident
// CTAs in equal consecutive ranges: sequences of any lengths finish together, without knowing the
// lengths on the host.  A segment that one CTA holds entirely is written at once; the others
// leave (m, sum, output) in the workspace and a second kernel joins them in order.  The next
// segment's first tiles are requested before the last one's merge.
//
// Measured (device time of this kernel + the join, one token each, 32 query and 8 KV heads, D = 128): 128 sequences
// of 512 to 4096 positions, E4M3, 600 MB: 105 + 4 us, 5.5 TB/s, HBM-bound; 17 sequences of them in bf16, 167 MB:
// 32 + 5 us; one of 65521, E4M3, 134 MB: 30 + 7 us.  The shorter the call, the more of it are the start (planning,
// first tiles: some 4 us) and the join; 115 positions take 5.3 us.

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
#include "tma_host.cuh"

namespace mk {

void set_last_error(const char *msg);  // megakernel.cu

namespace paged {

// CTAs per SM, by what their registers allow
__host__ __device__ constexpr int resident_ctas(int row_tiles) { return row_tiles == 1 ? 3 : 2; }

template <int D, bool FP8>
struct Tile {
    static constexpr int kRowBytes = D * (FP8 ? 1 : 2);
    static constexpr int kPanelBytes = kRowBytes < 128 ? kRowBytes : 128;   // one swizzle row
    static constexpr int kPanels = kRowBytes / kPanelBytes;
    static constexpr int kTokens = kRowBytes == 256 ? 16 : 32;              // positions per warp tile
    static constexpr int kBytes = kTokens * kRowBytes;                      // keys (and values)
    static constexpr int kStages = kRowBytes == 64 ? 4 : 2;                 // 16 KiB per warp
    static constexpr int kRing = kStages * 2 * kBytes;
    static constexpr int kUnit = kWarps * kTokens;                          // positions per unit
    static constexpr int kMmaTiles = kTokens / 16;
};

constexpr int kSegmentCost = 1;   // of a segment besides its tiles (its queries and its merge), in units

template <int D, bool FP8, int NT>
struct __align__(1024) DecodeSmem {
    uint8_t ring[kWarps][Tile<D, FP8>::kRing];
    float merge[2][8 * NT * D];
    float stat_m[kWarps][8 * NT], stat_l[kWarps][8 * NT];
    uint64_t full[kWarps][Tile<D, FP8>::kStages];
    int scan[kWarps];
    int prefix[1];   // [seqs + 1]
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// NT: tiles of 8 query rows per row block.
template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(kWarps * 32, resident_ctas(NT))
decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttentionParams p) {
    using T = Tile<D, FP8>;
    using Smem = DecodeSmem<D, FP8, NT>;
    constexpr int kRows = 8 * NT;
    constexpr Cut kCut = {kRows, T::kUnit, kSegmentCost};
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Batch &bt = p.bt;
    pdl_launch_dependents();
    if (lane == 0)
        for (int i = 0; i < T::kStages; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_barrier_init();
    pdl_wait();
    Walk walk;
    plan_walk<kWarps * 32>(bt, p.hkv, p.group, kCut, 0, p.max_count, sm.prefix, sm.scan, walk);

    const uint32_t ring = smem_addr(sm.ring[warp]);
    const int page_mask = (1 << bt.page_shift) - 1;
    const bool two = page_mask + 1 < T::kTokens;   // a tile of 32 positions over two pages of 16
    constexpr int kPages = 2;

    // this warp's tiles of a segment: positions from + i * kUnit, i < n
    struct Share {
        int from, n, seen;      // seen: positions the row block looks at
        const int *table;
    };
    auto share_of = [&](const Segment &s) {
        Share h;
        h.seen = min(s.tile1 * T::kUnit, visible(s.length, s.count, min(div((s.rb + 1) * kRows - 1, p.group), s.count - 1)));
        h.from = s.tile0 * T::kUnit + warp * T::kTokens;
        h.n = h.seen > h.from ? (h.seen - h.from + T::kUnit - 1) / T::kUnit : 0;
        h.table = bt.table + s.b * bt.table_stride;
        return h;
    };
    // pages of 32 tiles from i0 on, one tile per lane
    auto load_pages = [&](const Share &h, int i0, int (&page)[kPages]) {
#pragma unroll
        for (int k = 0; k < kPages; ++k) {
            const int pos = h.from + (i0 + lane) * T::kUnit + 16 * k;
            page[k] = -1;
            if (i0 + lane < h.n && pos < h.seen && (k == 0 || two)) {
                const int id = __ldg(h.table + (pos >> bt.page_shift));
                if (id >= bt.num_pages) atomicOr(bt.error, kErrorIndex);
                else page[k] = id;
            }
        }
    };
    auto load_scales = [&](const int (&page)[kPages], int head, float (&ks)[kPages], float (&vs)[kPages]) {
        if constexpr (FP8) {
#pragma unroll
            for (int k = 0; k < kPages; ++k) {
                ks[k] = 1.f;
                vs[k] = 0.f;
                if (page[k] >= 0) {
                    const long long at = (long long)page[k] * p.hkv + head;
                    ks[k] = __ldg(p.k_scales + at);
                    vs[k] = log2f(fmaxf(__ldg(p.v_scales + at), 0x1p-100f));
                }
            }
        }
    };
    // copy of a tile into ring stage st
    auto issue = [&](const Share &h, int head, int i, const int (&pages)[kPages], uint32_t st) {
        const int page0 = __shfl_sync(0xffffffffu, pages[0], i & 31), page1 = two ? __shfl_sync(0xffffffffu, pages[1], i & 31) : 0;
        if (lane == 0) {
            const int pos = h.from + i * T::kUnit;
            const uint32_t dst = ring + st * 2 * T::kBytes;
            uint64_t *bar = &sm.full[warp][st];
            mbar_arrive_expect_tx(bar, 2 * T::kBytes);
#pragma unroll
            for (int panel = 0; panel < T::kPanels; ++panel) {
                const uint32_t at = dst + panel * T::kTokens * T::kPanelBytes;
                const int x = panel * T::kPanelBytes / (FP8 ? 1 : 2);
                tma_load_4d(at, &map_k, x, pos & page_mask, head, page0, bar);
                tma_load_4d(at + T::kBytes, &map_v, x, pos & page_mask, head, page0, bar);
                if (two) {
                    tma_load_4d(at + 16 * T::kPanelBytes, &map_k, x, 0, head, page1, bar);
                    tma_load_4d(at + 16 * T::kPanelBytes + T::kBytes, &map_v, x, 0, head, page1, bar);
                }
            }
        }
    };

    uint32_t stage = 0, parity = 0;   // the tile consumed next (kStages: a wait ran out)
    uint32_t fill = 0;                // the stage filled next
    int in_flight = 0, odd = 0;       // filled stages; segments so far, mod 2
    JoinEntry entry = {0, 0, 0, 0};
    Segment cur, next;
    Share mine, mine_next;
    int page_cur[kPages], page_next[kPages];   // of 32 tiles; page_next: the 32 after them, in this segment or the next
    float ks_cur[kPages], vs_cur[kPages], ks_next[kPages], vs_next[kPages];
    int ahead = 0;                             // tiles of the next segment that have been asked for
    bool have = next_segment(bt, p.hkv, p.group, kCut, walk, cur);
    if (have) {
        mine = share_of(cur);
        load_pages(mine, 0, page_cur);
    }

    while (have) {
        int asked = ahead;   // tiles of this segment that have been asked for
        ahead = 0;
        if (stage == T::kStages) mine.n = 0;
        while (in_flight < T::kStages && asked < mine.n && asked < 32) {
            issue(mine, cur.head, asked++, page_cur, fill);
            if (++fill == T::kStages) fill = 0;
            ++in_flight;
        }
        load_scales(page_cur, cur.head, ks_cur, vs_cur);

        // query fragments: row g of tile nt, with the columns' order of the key fragments
        uint32_t qf[D / 16][NT][2];
        float q_scale[NT][2];   // of the columns 2t, 2t + 1 of a score fragment
        int limit[NT][2];       // positions those rows see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g, pair = cur.rb * kRows + r;
            const bool real = r < cur.rows;
            const bf16 *qp = p.q + (long long)(cur.first + (real ? div(pair, p.group) : 0)) * p.q_token +
                             (long long)(cur.head * p.group.d + (real ? pair - div(pair, p.group) * p.group.d : 0)) * p.q_head;
            float unscale = 1.f;
            if constexpr (FP8) {
                uint32_t raw[D / 16][2];
                float amax = 0.f;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint2 v = real ? __ldg(reinterpret_cast<const uint2 *>(qp + 16 * ks + 4 * t)) : make_uint2(0u, 0u);
                    raw[ks][0] = v.x;
                    raw[ks][1] = v.y;
                }
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float a = fabsf(bf16_lo(raw[ks][i])), c = fabsf(bf16_hi(raw[ks][i]));
                        if (a < INFINITY) amax = fmaxf(amax, a);
                        if (c < INFINITY) amax = fmaxf(amax, c);
                    }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // 2^e with amax / 2^e in [2^14, 2^15); e stays where both it and its inverse are normal numbers
                const int e = max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -120);
                const float factor = __uint_as_float((uint32_t)(127 - e) << 23);
                unscale = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i) qf[ks][nt][i] = pack_f16(bf16_lo(raw[ks][i]) * factor, bf16_hi(raw[ks][i]) * factor);
            } else {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        qf[ks][nt][i] = real ? __ldg(reinterpret_cast<const uint32_t *>(qp + 16 * ks + 2 * t + 8 * i)) : 0u;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                q_scale[nt][e] = FP8 ? p.scale_log2e * __shfl_sync(0xffffffffu, unscale, (2 * t + e) * 4) : p.scale_log2e;
                const int r2 = nt * 8 + 2 * t + e;
                limit[nt][e] = r2 < cur.rows ? visible(cur.length, cur.count, div(cur.rb * kRows + r2, p.group)) : 0;
            }
        }
        const int all_see = visible(cur.length, cur.count, div(cur.rb * kRows, p.group));   // positions that every row sees

        // the next segment, while the first copies of this one are under way
        const bool have_next = next_segment(bt, p.hkv, p.group, kCut, walk, next);
        if (have_next) mine_next = share_of(next);
        else mine_next.n = 0;

        float m[NT][2], l[NT][2];
        float o[D / 16][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) o[c][nt][0] = o[c][nt][1] = o[c][nt][2] = o[c][nt][3] = 0.f;
        }
        bool next_paged = false;   // page_next holds the next segment's first pages

        for (int i = 0; i < mine.n; ++i) {
            const int cur0 = i & ~31;
            const bool last = cur0 + 32 >= mine.n;
            if (i == cur0) {
                if (i) {
#pragma unroll
                    for (int k = 0; k < kPages; ++k) { page_cur[k] = page_next[k]; ks_cur[k] = ks_next[k]; vs_cur[k] = vs_next[k]; }
                }
                if (!last) load_pages(mine, cur0 + 32, page_next);
                else if (have_next) load_pages(mine_next, 0, page_next);
                next_paged = last && have_next;
            }
            if ((i & 31) == 24 && !last) load_scales(page_next, cur.head, ks_next, vs_next);

            float ks[T::kMmaTiles], vs[T::kMmaTiles];
            const int pg0 = __shfl_sync(0xffffffffu, page_cur[0], i & 31), pg1 = two ? __shfl_sync(0xffffffffu, page_cur[1], i & 31) : pg0;
#pragma unroll
            for (int mt = 0; mt < T::kMmaTiles; ++mt) {
                if (FP8 && (mt == 0 || two)) {
                    ks[mt] = __shfl_sync(0xffffffffu, ks_cur[mt], i & 31);
                    vs[mt] = __shfl_sync(0xffffffffu, vs_cur[mt], i & 31);
                } else {
                    ks[mt] = FP8 ? ks[0] : 1.f;
                    vs[mt] = FP8 ? vs[0] : 0.f;
                }
            }

            const uint32_t kt = ring + stage * 2 * T::kBytes, vt = kt + T::kBytes;
            const int pos0 = mine.from + i * T::kUnit;
            if (!__all_sync(0xffffffffu, mbar_try_wait(&sm.full[warp][stage], parity))) {
                const auto wait = [&](uint64_t *bar, uint32_t par, long long began) {
                    bool done;
                    while (!(done = mbar_try_wait(bar, par)) && clock64() - began <= kWaitCycles) {}
                    return done;
                };
                if (!__all_sync(0xffffffffu, wait(&sm.full[warp][stage], parity, clock64()))) {
                    // The warp asks for no more tiles, here and in the segments to come, and does not leave with copies under way.
                    if (lane == 0) atomicOr(bt.error, kErrorWait);
                    const long long began = clock64();
                    for (int k = 0; k < in_flight; ++k) {
                        const RingFill f = ring_fill(stage, parity, k, T::kStages);
                        wait(&sm.full[warp][f.stage], f.parity, began);
                    }
                    __syncwarp();
                    stage = T::kStages;   // no stage: given up
                    break;
                }
            }
            __syncwarp();

            // scores [position][query row]
            float sc[T::kMmaTiles][NT][4];
#pragma unroll
            for (int mt = 0; mt < T::kMmaTiles; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sc[mt][nt][0] = sc[mt][nt][1] = sc[mt][nt][2] = sc[mt][nt][3] = 0.f;
            const int mat = lane >> 3;
            // address of 16-byte chunk c of position r in a tile
            auto chunk_at = [&](uint32_t tile, int r, int c) {
                if constexpr (T::kPanelBytes == 128)
                    return tile + (c >> 3) * (T::kTokens * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                else
                    return tile + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
            };
#pragma unroll
            for (int c2 = 0; c2 < T::kRowBytes / 32; ++c2) {
#pragma unroll
                for (int mt = 0; mt < T::kMmaTiles; ++mt) {
                    uint32_t kf[4];
                    ldsm4(chunk_at(kt, mt * 16 + (mat & 1) * 8 + (lane & 7), 2 * c2 + (mat >> 1)), kf);
                    if constexpr (FP8) {   // two 16-wide steps: chunk 2 c2 and chunk 2 c2 + 1
                        uint32_t a[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) codes_to_f16(kf[j], a[2 * j], a[2 * j + 1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<true>(sc[mt][nt], a[0], a[2], a[1], a[3], qf[2 * c2][nt][0], qf[2 * c2][nt][1]);
                            mma16816<true>(sc[mt][nt], a[4], a[6], a[5], a[7], qf[2 * c2 + 1][nt][0], qf[2 * c2 + 1][nt][1]);
                        }
                    } else {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16816<false>(sc[mt][nt], kf[0], kf[1], kf[2], kf[3], qf[c2][nt][0], qf[c2][nt][1]);
                    }
                }
            }

            // rows that look past their own last position, positions past the sequence, pages that are not there
            const bool masked = pg0 < 0 || pg1 < 0 || pos0 + T::kTokens > all_see;
            if (masked) {
                // A value that is not finite must not meet the zero weight of a row that does not see it: take it out
                // of the tile, and give it to the rows that see it by hand.
                uint32_t bad = 0;
                for (int c = lane; c < T::kTokens * (T::kRowBytes / 16); c += 32) {
                    const int r = c / (T::kRowBytes / 16), pos = pos0 + r;
                    const uint32_t addr = chunk_at(vt, r, c % (T::kRowBytes / 16));
                    if (pos >= cur.length) {
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0u) : "memory");
                    } else if (pos >= all_see) {
                        uint32_t w[4];
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
#pragma unroll
                        for (int j = 0; j < 4; ++j) bad |= FP8 ? not_finite_e4m3(w[j]) : not_finite_b16(w[j]);
                    }
                }
                __syncwarp();
                if (__any_sync(0xffffffffu, bad != 0)) {
                    for (int r = max(all_see - pos0, 0); r < min(T::kTokens, cur.length - pos0); ++r) {
#pragma unroll
                        for (int c = 0; c < D / 16; ++c)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {   // accumulator rows g and g + 8 of tile c
                                const int d = FP8 ? 16 * c + 2 * g + half : 16 * c + 8 * half + g;
                                const uint32_t at = chunk_at(vt, r, d * (FP8 ? 1 : 2) / 16) + d * (FP8 ? 1 : 2) % 16;
                                uint32_t bits;
                                if constexpr (FP8) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(bits) : "r"(at));
                                else asm volatile("ld.shared.u16 %0, [%1];" : "=r"(bits) : "r"(at));
                                if (FP8 ? (bits & 0x7fu) == 0x7fu : (bits & 0x7f80u) == 0x7f80u) {
                                    const float value = FP8 ? __int_as_float(0x7fffffff) : __uint_as_float(bits << 16);
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                        for (int e = 0; e < 2; ++e)
                                            if (pos0 + r < limit[nt][e]) o[c][nt][2 * half + e] += value;
                                }
                            }
                    }
                    __syncwarp();
                    for (int c = lane; c < T::kTokens * (T::kRowBytes / 4); c += 32) {
                        const int r = c / (T::kRowBytes / 4), byte = c % (T::kRowBytes / 4) * 4;
                        if (pos0 + r < all_see || pos0 + r >= cur.length) continue;
                        const uint32_t at = chunk_at(vt, r, byte / 16) + byte % 16;
                        uint32_t w;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
                        w &= ~(FP8 ? __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) : __vcmpeq2(w & 0x7f807f80u, 0x7f807f80u));
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy into this tile
                __syncwarp();
            }

            // online softmax of rows 2t, 2t + 1 of every tile over this tile's positions
            uint32_t pf[T::kMmaTiles][NT][2], pf_lo[T::kMmaTiles][NT][2];
            bool rescale = false;
            float corr[NT][2], inv_vs[T::kMmaTiles];
#pragma unroll
            for (int mt = 0; mt < T::kMmaTiles; ++mt) inv_vs[mt] = FP8 ? exp2_fast(-vs[mt]) : 1.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int mt = 0; mt < T::kMmaTiles; ++mt) {
                        const float c = q_scale[nt][e] * ks[mt];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float x = FP8 ? fmaf(sc[mt][nt][2 * h + e], c, vs[mt]) : sc[mt][nt][2 * h + e] * c;
                            if (masked) {
                                const int pos = pos0 + mt * 16 + h * 8 + g;
                                if (!((mt == 1 ? pg1 : pg0) >= 0 && pos < limit[nt][e])) x = -INFINITY;
                            }
                            sc[mt][nt][2 * h + e] = x;
                            mx = fmaxf(mx, x);
                        }
                    }
#pragma unroll
                    for (int off = 4; off < 32; off *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                    const float mn = fmaxf(m[nt][e], mx);
                    const float base = mn == -INFINITY ? 0.f : mn, base_w = FP8 ? base - kFewWeight : base;
                    // before the first score only an infinite value given by hand can be in the output: times 0 it would be NaN
                    corr[nt][e] = !FP8 && m[nt][e] == -INFINITY ? 1.f : exp2_fast(m[nt][e] - base);
                    rescale = rescale || mn != m[nt][e];
                    m[nt][e] = mn;
                    float add = 0.f;
#pragma unroll
                    for (int mt = 0; mt < T::kMmaTiles; ++mt) {
                        const float w0 = exp2_fast(sc[mt][nt][e] - base_w), w1 = exp2_fast(sc[mt][nt][2 + e] - base_w);
                        sc[mt][nt][e] = w0;
                        sc[mt][nt][2 + e] = w1;
                        add = fmaf(FP8 ? (w0 + w1) * kFewUnscale : w0 + w1, inv_vs[mt], add);
                    }
                    l[nt][e] = fmaf(l[nt][e], corr[nt][e], add);
                }
#pragma unroll
                for (int mt = 0; mt < T::kMmaTiles; ++mt) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float w0 = sc[mt][nt][2 * h], w1 = sc[mt][nt][2 * h + 1];
                        if constexpr (FP8) {
                            pf[mt][nt][h] = transpose8(pack_f16(w0, w1));
                        } else {
                            // cut off, not rounded, so that the remainder has the weight's sign, and kept above zero: an infinite
                            // value times the two terms is infinite, not NaN (2^-126 is the least weight there is)
                            const uint32_t hi = __byte_perm(__float_as_uint(w0), __float_as_uint(w1), 0x7632);
                            const float r0 = fmaxf(w0 - bf16_lo(hi), fminf(w0, 0x1p-126f)), r1 = fmaxf(w1 - bf16_hi(hi), fminf(w1, 0x1p-126f));
                            pf[mt][nt][h] = transpose8(hi);
                            pf_lo[mt][nt][h] = transpose8(pack_b16(r0, r1));
                        }
                    }
                }
            }
            if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < D / 16; ++c)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[c][nt][j] *= corr[nt][j & 1];
            }

            // output [dimension][query row] += values^T weights
#pragma unroll
            for (int mt = 0; mt < T::kMmaTiles; ++mt) {
#pragma unroll
                for (int c2 = 0; c2 < T::kRowBytes / 32; ++c2) {
                    uint32_t vf[4];
                    if constexpr (FP8) {
                        ldsm4_trans(chunk_at(vt, mt * 16 + (mat & 1) * 8 + (lane & 7), 2 * c2 + (mat >> 1)), vf);
                        uint32_t a[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) codes_to_f16(__byte_perm(vf[j], 0u, 0x3120), a[2 * j], a[2 * j + 1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<true>(o[2 * c2][nt], a[0], a[1], a[2], a[3], pf[mt][nt][0], pf[mt][nt][1]);
                            mma16816<true>(o[2 * c2 + 1][nt], a[4], a[5], a[6], a[7], pf[mt][nt][0], pf[mt][nt][1]);
                        }
                    } else {
                        ldsm4_trans(chunk_at(vt, mt * 16 + (mat >> 1) * 8 + (lane & 7), 2 * c2 + (mat & 1)), vf);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<false>(o[c2][nt], vf[0], vf[1], vf[2], vf[3], pf[mt][nt][0], pf[mt][nt][1]);
                            mma16816<false>(o[c2][nt], vf[0], vf[1], vf[2], vf[3], pf_lo[mt][nt][0], pf_lo[mt][nt][1]);
                        }
                    }
                }
            }
            __syncwarp();
            --in_flight;
            if (++stage == T::kStages) { stage = 0; parity ^= 1u; }
            // ask for what comes next: this segment's tiles, then the next one's
            while (in_flight < T::kStages) {
                if (asked < mine.n) {
                    if (asked < cur0 + 32) issue(mine, cur.head, asked, page_cur, fill);
                    else issue(mine, cur.head, asked, page_next, fill);
                    ++asked;
                } else if (next_paged && ahead < mine_next.n && ahead < 32) {
                    issue(mine_next, next.head, ahead, page_next, fill);
                    ++ahead;
                } else {
                    break;
                }
                if (++fill == T::kStages) fill = 0;
                ++in_flight;
            }
        }

        // The warps' states meet, in an order that does not depend on timing: two warps leave theirs in shared memory, the
        // others add them, and one adds the last pair and writes.  The roles swap from segment to segment, so that a
        // buffer's next writer is the warp that read it last.
        const int swapped = odd, role = swapped ? 3 - warp : warp;
        odd ^= 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int off = 4; off < 32; off *= 2) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
                if (g == 0) {
                    sm.stat_m[warp][nt * 8 + 2 * t + e] = m[nt][e];
                    sm.stat_l[warp][nt * 8 + 2 * t + e] = l[nt][e];
                }
            }
        auto leave = [&](float *buffer) {   // lane-major: one fragment register of all lanes side by side
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
                    *reinterpret_cast<float4 *>(buffer + ((nt * (D / 16) + c) * 32 + lane) * 4) = make_float4(o[c][nt][0], o[c][nt][1], o[c][nt][2], o[c][nt][3]);
        };
        auto add = [&](const float *buffer, const float (&f)[NT][2]) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const float4 v = *reinterpret_cast<const float4 *>(buffer + ((nt * (D / 16) + c) * 32 + lane) * 4);
                    o[c][nt][0] = fmaf(v.x, f[nt][0], o[c][nt][0]);
                    o[c][nt][1] = fmaf(v.y, f[nt][1], o[c][nt][1]);
                    o[c][nt][2] = fmaf(v.z, f[nt][0], o[c][nt][2]);
                    o[c][nt][3] = fmaf(v.w, f[nt][1], o[c][nt][3]);
                }
        };
        if (role >= 2) leave(sm.merge[role - 2]);
        __syncthreads();
        float M[NT][2], L[NT][2];
        if (role < 2) {
            const int partner = swapped ? 1 - role : 2 + role;   // the warp whose state lies in merge[role]
            float f_own[NT][2], f_partner[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = nt * 8 + 2 * t + e;
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.stat_m[w][r]);
                    const float base = top == -INFINITY ? 0.f : top;
                    float total = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) total = fmaf(sm.stat_l[w][r], exp2_fast(sm.stat_m[w][r] - base), total);
                    M[nt][e] = top;
                    L[nt][e] = total;
                    f_own[nt][e] = exp2_fast(m[nt][e] - base) * (FP8 ? kFewUnscale : 1.f);
                    f_partner[nt][e] = exp2_fast(sm.stat_m[partner][r] - base) * (FP8 ? kFewUnscale : 1.f);
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[c][nt][j] *= f_own[nt][j & 1];
            add(sm.merge[role], f_partner);
            if (role == 1) leave(sm.merge[1]);
        }
        __syncthreads();
        if (role == 0) {
            float ones[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) ones[nt][0] = ones[nt][1] = 1.f;
            add(sm.merge[1], ones);
            const bool complete = cur.begins && cur.ends;
            float *part = p.partial + ((long long)blockIdx.x * 2 + (cur.begins ? 1 : 0)) * kRows * (D + 2);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = nt * 8 + 2 * t + e;
                    if (r >= cur.rows) continue;
                    const int pair = cur.rb * kRows + r;
                    bf16 *dst = p.out + ((long long)(cur.first + div(pair, p.group)) * p.hq + cur.head * p.group.d + pair - div(pair, p.group) * p.group.d) * D;
                    const float inv = L[nt][e] == 0.f ? 0.f : 1.f / L[nt][e];
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        const float x = o[c][nt][e], y = o[c][nt][2 + e];
                        if constexpr (FP8) {   // columns 16 c + 2 g and the next one
                            if (complete) *reinterpret_cast<__nv_bfloat162 *>(dst + 16 * c + 2 * g) = __floats2bfloat162_rn(x * inv, y * inv);
                            else *reinterpret_cast<float2 *>(part + r * (D + 2) + 16 * c + 2 * g) = make_float2(x, y);
                        } else {               // columns 16 c + g and 16 c + 8 + g
                            if (complete) {
                                dst[16 * c + g] = __float2bfloat16_rn(x * inv);
                                dst[16 * c + 8 + g] = __float2bfloat16_rn(y * inv);
                            } else {
                                part[r * (D + 2) + 16 * c + g] = x;
                                part[r * (D + 2) + 16 * c + 8 + g] = y;
                            }
                        }
                    }
                    if (!complete && g == 0) *reinterpret_cast<float2 *>(part + r * (D + 2) + D) = make_float2(M[nt][e], L[nt][e]);
                }
        }
        if (cur.parts > 1) entry = JoinEntry{cur.parts, cur.first, cur.rb * kRows, (cur.head << 16) | cur.rows};
        if (have_next && !next_paged) load_pages(mine_next, 0, page_next);   // this warp had no tile in the segment
        have = have_next;
        cur = next;
        mine = mine_next;
#pragma unroll
        for (int k = 0; k < kPages; ++k) page_cur[k] = page_next[k];
    }
    if (p.entries && threadIdx.x == 0) p.entries[blockIdx.x] = entry;
}

// Joins the parts of a segment that several CTAs shared, from CTA `from` on: this CTA's share of its rows.  A warp
// takes a row, or with fewer than eight rows a share of a row's parts; its lanes read the statistics of 32 parts at
// once, then the parts one after the other, D / 32 columns each.  The order of the sums is fixed.
template <int D>
__device__ __forceinline__ void join_segment(const AttentionParams &p, const JoinEntry &e, int from, int rows_per_block, float (&sum_o)[8][D],
                                             float (&sum_m)[8], float (&sum_l)[8]) {
    constexpr int kCols = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = e.head_rows & 0xffff, head = e.head_rows >> 16;
    const int share = (rows + gridDim.y - 1) / gridDim.y, row_end = min(rows, (int)(blockIdx.y + 1) * share);   // rows of this CTA
    const int per = share > 4 ? 1 : share > 2 ? 2 : share > 1 ? 4 : 8;                                          // warps per row
    for (int row0 = blockIdx.y * share; row0 < row_end; row0 += 8 / per) {
        const int r = row0 + warp / per, sub = warp % per;
        float M = -INFINITY, L = 0.f, O[kCols];
#pragma unroll
        for (int k = 0; k < kCols; ++k) O[k] = 0.f;
        auto part_of = [&](int i) {   // part i of the segment, this row
            return p.partial + (((long long)(from + i) * 2 + (i == 0 ? 1 : 0)) * rows_per_block + r) * (D + 2);
        };
        if (r < row_end) {
            for (int base = sub; base < e.parts; base += 32 * per) {
                const int mine = base + lane * per;
                const float2 ml = mine < e.parts ? *reinterpret_cast<const float2 *>(part_of(mine) + D) : make_float2(-INFINITY, 0.f);
                float top = ml.x;
#pragma unroll
                for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                top = fmaxf(top, M);
                const float zero = top == -INFINITY ? 0.f : top, corr = exp2_fast(M - zero), f = exp2_fast(ml.x - zero);
                float total = ml.y * f;
#pragma unroll
                for (int off = 16; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
                L = fmaf(L, corr, total);
                M = top;
#pragma unroll
                for (int k = 0; k < kCols; ++k) O[k] *= corr;
                const int n = min(32, (e.parts - base + per - 1) / per);
#pragma unroll 8
                for (int i = 0; i < n; ++i) {
                    const float w = __shfl_sync(0xffffffffu, f, i);
                    const float *src = part_of(base + i * per) + kCols * lane;
#pragma unroll
                    for (int k = 0; k < kCols; k += 2) {
                        const float2 v = *reinterpret_cast<const float2 *>(src + k);
                        O[k] = fmaf(v.x, w, O[k]);
                        O[k + 1] = fmaf(v.y, w, O[k + 1]);
                    }
                }
            }
        }
        if (per > 1) {   // the row's warps meet
            __syncthreads();
            if (lane == 0) { sum_m[warp] = M; sum_l[warp] = L; }
#pragma unroll
            for (int k = 0; k < kCols; ++k) sum_o[warp][kCols * lane + k] = O[k];
            __syncthreads();
            M = -INFINITY;
            for (int w = 0; w < per; ++w) M = fmaxf(M, sum_m[warp - sub + w]);
            const float zero = M == -INFINITY ? 0.f : M;
            L = 0.f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) O[k] = 0.f;
            for (int w = 0; w < per; ++w) {
                const float f = exp2_fast(sum_m[warp - sub + w] - zero);
                L = fmaf(sum_l[warp - sub + w], f, L);
#pragma unroll
                for (int k = 0; k < kCols; ++k) O[k] = fmaf(sum_o[warp - sub + w][kCols * lane + k], f, O[k]);
            }
        }
        if (r < row_end && sub == 0) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            const int pair = e.pair + r;
            bf16 *dst = p.out + ((long long)(e.row + div(pair, p.group)) * p.hq + head * p.group.d + pair - div(pair, p.group) * p.group.d) * D + kCols * lane;
#pragma unroll
            for (int k = 0; k < kCols; k += 2) *reinterpret_cast<__nv_bfloat162 *>(dst + k) = __floats2bfloat162_rn(O[k] * inv, O[k + 1] * inv);
        }
    }
}

// The segments that begin in the ranges of `entries` CTAs from blockIdx.x * entries on: few segments leave most
// entries empty, and a CTA looks at 32 of them at once.
template <int D>
__global__ void __launch_bounds__(256)
join_kernel(const AttentionParams p, int rows_per_block, int entries, int ctas) {
    pdl_wait();   // and no early start for the next kernel: see paged.cuh
    __shared__ float sum_o[8][D], sum_m[8], sum_l[8];
    const int begin = blockIdx.x * entries, end = min(begin + entries, ctas), lane = threadIdx.x & 31;
    for (int base = begin; base < end; base += 32) {
        const int4 mine = base + lane < end ? __ldg(reinterpret_cast<const int4 *>(p.entries + base + lane)) : make_int4(0, 0, 0, 0);
        for (unsigned todo = __ballot_sync(0xffffffffu, mine.x != 0); todo; todo &= todo - 1) {
            const int l = __ffs(todo) - 1;
            const JoinEntry e = {__shfl_sync(0xffffffffu, mine.x, l), __shfl_sync(0xffffffffu, mine.y, l), __shfl_sync(0xffffffffu, mine.z, l),
                                 __shfl_sync(0xffffffffu, mine.w, l)};
            join_segment<D>(p, e, base + l, rows_per_block, sum_o, sum_m, sum_l);
            __syncthreads();   // the sums are the next segment's
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Query rows that a sequence of this call can have at most.
static long long most_rows(const Batch &bt, int group, int max_count) {
    return (long long)(bt.cu ? (bt.tokens < max_count ? bt.tokens : max_count) : bt.per_seq) * group;
}

// Tiles of 8 query rows per row block: one where no sequence of this call can have more rows, else two.  Four
// would read the cache once for 17 to 32 rows, but their accumulators leave too few registers: 32 sequences x 5
// tokens x 4 heads of a group against up to 16384 positions of E4M3, D = 128: one tile 256 us, two 187, four 294;
// 16 x 5 x 4 against 4000 of bf16: 122, 86 and 108.  (12 rows: one tile 43.4, two 36.8.)
static int row_tiles(const Batch &bt, int group, int max_count) { return most_rows(bt, group, max_count) <= 8 ? 1 : 2; }

bool make_pool_map(CUtensorMap *map, const Pool &pool, const void *base, int box_tokens, bool swizzle) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const int bytes = pool.fp8 ? 1 : 2;
    const int panel = !swizzle || pool.head_dim * bytes < 128 ? pool.head_dim * bytes : 128;
    const cuuint64_t dims[4] = {(cuuint64_t)pool.head_dim, (cuuint64_t)pool.page_size, (cuuint64_t)pool.kv_heads, (cuuint64_t)pool.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)(pool.slot_stride * bytes), (cuuint64_t)(pool.head_stride * bytes),
                                   (cuuint64_t)(pool.page_stride * bytes)};
    const cuuint32_t box[4] = {(cuuint32_t)(panel / bytes), (cuuint32_t)box_tokens, 1, 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    return fn(map, pool.fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides,
              box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, !swizzle ? CU_TENSOR_MAP_SWIZZLE_NONE : panel == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool FP8, int NT>
static int launch_decode_t(const AttentionParams &p, const Pool &pool, int sms, cudaStream_t st) {
    using T = Tile<D, FP8>;
    using DecodeSmemOf = DecodeSmem<D, FP8, NT>;
    CUtensorMap map_k, map_v;
    const int box = pool.page_size < T::kTokens ? pool.page_size : T::kTokens;
    if (!make_pool_map(&map_k, pool, pool.k, box, true) || !make_pool_map(&map_v, pool, pool.v, box, true)) {
        set_last_error("mk_paged_attention: cuTensorMapEncodeTiled refused the cache (driver without tensor-map support?)");
        return MK_ERR_UNSUPPORTED;
    }
    const size_t smem = offsetof(DecodeSmemOf, prefix) + (size_t)(p.bt.seqs + 1) * sizeof(int);
    static bool allowed[64] = {};
    cudaError_t e = allow_smem((const void *)decode_kernel<D, FP8, NT>, allowed);
    if (e != cudaSuccess) return (int)e;
    const DecodeGrid grid = decode_grid(pool, p.bt, p.hq, p.max_count, sms);
    e = launch_pdl(decode_kernel<D, FP8, NT>, dim3(grid.ctas), dim3(kWarps * 32), smem, st, map_k, map_v, p);
    if (e == cudaSuccess && grid.split)
        e = launch_pdl(join_kernel<D>, dim3((grid.ctas + grid.join_entries - 1) / grid.join_entries, grid.join_turns), dim3(256), 0, st, p,
                       8 * NT, grid.join_entries, grid.ctas);
    return (int)e;
}

template <int D, bool FP8>
static int launch_decode_d(const AttentionParams &p, const Pool &pool, int sms, cudaStream_t st) {
    if (row_tiles(p.bt, p.group.d, p.max_count) == 1) return launch_decode_t<D, FP8, 1>(p, pool, sms, st);
    return launch_decode_t<D, FP8, 2>(p, pool, sms, st);
}

DecodeGrid decode_grid(const Pool &pool, const Batch &bt, int hq, int max_count, int sms) {
    const int row_bytes = pool.head_dim * (pool.fp8 ? 1 : 2);
    const int unit = kWarps * (row_bytes == 256 ? 16 : 32);
    const int group = hq / pool.kv_heads, rows = 8 * row_tiles(bt, group, max_count);
    const long long tiles = (((long long)bt.max_pages << bt.page_shift) + unit - 1) / unit;
    const long long blocks = bt.cu ? (long long)bt.tokens * group / rows + bt.seqs : (long long)bt.seqs * block_count(bt.per_seq, group, rows);
    const long long most = blocks * pool.kv_heads * (tiles + kSegmentCost);
    DecodeGrid g;
    const long long resident = (long long)resident_ctas(rows / 8) * sms;
    g.ctas = (int)(most < resident ? most : resident);
    // segments to join: as many as there are row blocks, or CTAs where that is less; rows are dealt out until the GPU is full
    const long long joins = blocks * pool.kv_heads < g.ctas ? blocks * pool.kv_heads : g.ctas, turns = (sms + joins - 1) / joins;
    const long long held = most_rows(bt, group, max_count) < rows ? most_rows(bt, group, max_count) : rows;   // rows a block can have
    g.join_turns = (int)(turns < held ? turns : held);
    // few segments: their first CTAs lie ctas / joins apart, and CTAs of the join for every one between would only be launched
    g.join_entries = g.ctas > 2 * joins ? (int)(g.ctas / (2 * joins)) : 1;
    g.split = tiles > 1;
    g.too_many = most >= 0x7fffffffll;
    g.partial_floats = g.split ? (long long)g.ctas * 2 * rows * (pool.head_dim + 2) : 0;
    return g;
}

int launch_decode(const AttentionParams &p, const Pool &pool, int sms, cudaStream_t st) {
    if (pool.head_dim == 64)
        return pool.fp8 ? launch_decode_d<64, true>(p, pool, sms, st) : launch_decode_d<64, false>(p, pool, sms, st);
    return pool.fp8 ? launch_decode_d<128, true>(p, pool, sms, st) : launch_decode_d<128, false>(p, pool, sms, st);
}

// Most new tokens of a sequence that the few-row kernel takes: 32 rows, two row blocks (the second finds the
// cache's tiles in L2).  More are work for the large tiles of tcgen05, which always compute 256 rows: 20 rows
// against up to 16384 positions of E4M3 187 us here, 259 there; with bf16 (16 x 4000) 86 and 62, but there a
// weight is one bf16 term, here two, and a draft's tokens should meet the sums that single tokens meet.
static int most_few(int group) { return group >= 32 ? 1 : 32 / group; }

struct Plan {
    bool few;             // the few-row kernel has (or may have) sequences
    DecodeGrid decode;
    PrefillGrid prefill;
    long long entries, decode_floats, bytes;   // entries: of both kernels, in words
};

static Plan plan_attention(const Batch &bt, const Pool &pool, int hq, int sms) {
    Plan plan = {};
    const int limit = most_few(hq / pool.kv_heads);
    plan.few = bt.cu || bt.per_seq <= limit;
    if (plan.few) plan.decode = decode_grid(pool, bt, hq, limit, sms);
    plan.prefill = prefill_grid(pool, bt, hq, limit + 1, sms);
    plan.entries = 4ll * ((plan.decode.split ? plan.decode.ctas : 0) + plan.prefill.ctas);
    plan.decode_floats = (plan.decode.partial_floats + 3) & ~3ll;
    if (plan.decode.partial_floats || plan.prefill.partial_floats)
        plan.bytes = 4 * (plan.entries + plan.decode_floats + plan.prefill.partial_floats);
    return plan;
}

long long attention_workspace(const Batch &bt, const Pool &pool, int hq, int sms) {
    const Plan plan = plan_attention(bt, pool, hq, sms);
    return plan.decode.too_many || plan.prefill.too_many ? -1 : plan.bytes;
}

int launch_attention(AttentionParams p, const Pool &pool, void *workspace, int sms, cudaStream_t st) {
    const Plan plan = plan_attention(p.bt, pool, p.hq, sms);
    const int limit = most_few(p.group.d);
    int code = 0;
    float *floats = reinterpret_cast<float *>(workspace);
    if (plan.few) {
        p.max_count = limit;
        p.entries = plan.decode.split ? reinterpret_cast<JoinEntry *>(workspace) : nullptr;
        p.partial = floats + plan.entries;
        code = launch_decode(p, pool, sms, st);
    }
    if (code == 0 && plan.prefill.ctas) {
        p.entries = reinterpret_cast<JoinEntry *>(workspace) + (plan.decode.split ? plan.decode.ctas : 0);
        p.partial = floats + plan.entries + plan.decode_floats;
        code = launch_prefill(p, pool, plan.prefill, limit + 1, st);
    }
    return code;
}

}  // namespace paged
}  // namespace mk
