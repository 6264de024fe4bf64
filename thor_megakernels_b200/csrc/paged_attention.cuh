// What the kernels of attention over a paged cache share.
#pragma once

#include <cuda_fp16.h>

#include "paged.cuh"

namespace mk {
namespace paged {

constexpr int kWarps = 4;                          // warps per CTA of the few-row kernel
constexpr long long kWaitCycles = 2000000000ll;    // limit of a wait, about a second

// E4M3 pages: weights go to the tensor core as f16, times a power of two that uses the exponents above 1, so that what stands far
// below the running maximum is not lost: its position may have small values, or none (sums of weights and results are divided by
// it).  Without it a weight 17.4 (natural logarithm) below the maximum was gone from the numerator and still in the denominator.
// Few rows: weights are at most 1 before it; prompts: at most 2^kPromptGrowth, the growth of the maximum that does not rescale.
constexpr float kFewWeight = 14.f, kFewUnscale = 0x1p-14f;
constexpr float kPromptGrowth = 4.f, kPromptWeight = 11.f, kPromptUnscale = 0x1p-11f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// four E4M3 codes -> two f16 pairs (low codes first)
__device__ __forceinline__ void codes_to_f16(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
}
// non-zero where one of the codes / values of a word is not finite: all ones in the exponent (and, E4M3, the mantissa) carry
__device__ __forceinline__ uint32_t not_finite_e4m3(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t not_finite_b16(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_b16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int slot, int head, int page, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_addr(bar)) : "memory");
}

// The fills of a ring that are under way, oldest first from the stage that is consumed next: stage of the k-th and parity of its
// barrier.
struct RingFill {
    uint32_t stage, parity;
};
__host__ __device__ inline RingFill ring_fill(uint32_t stage, uint32_t parity, uint32_t k, uint32_t stages) {
    const uint32_t s = stage + k;
    return s < stages ? RingFill{s, parity} : RingFill{s - stages, parity ^ 1u};
}

struct DecodeGrid {
    int ctas;
    bool split;                     // a segment may be shared by several CTAs
    bool too_many;                  // more units than 32 bits count
    int join_turns;                 // CTAs that share a segment's rows in the join
    int join_entries;               // CTAs of this kernel whose entries one of the join's looks at
    long long partial_floats;
};

DecodeGrid decode_grid(const Pool &pool, const Batch &bt, int hq, int max_count, int sms);
int launch_decode(const AttentionParams &p, const Pool &pool, int sms, cudaStream_t st);
// tensor map [pages, heads, slots, dim] of a pool; boxes of box_tokens slots and up to 128 bytes with the matching swizzle, or of
// whole rows without one
bool make_pool_map(CUtensorMap *map, const Pool &pool, const void *base, int box_tokens, bool swizzle);

struct PrefillGrid {
    int ctas;                       // 0: no sequence of the call can have enough rows
    bool too_many;
    long long partial_floats;
};
PrefillGrid prefill_grid(const Pool &pool, const Batch &bt, int hq, int min_count, int sms);
int launch_prefill(const AttentionParams &p, const Pool &pool, const PrefillGrid &grid, int min_count, cudaStream_t st);

}  // namespace paged
}  // namespace mk
