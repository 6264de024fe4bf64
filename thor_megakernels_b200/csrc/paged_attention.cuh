// What the kernels of attention over a paged cache share on the host.
#pragma once

#include "paged.cuh"

namespace mk {
namespace paged {

constexpr int kWarps = 4;                          // warps per CTA of the few-row kernel
constexpr long long kWaitCycles = 2000000000ll;    // limit of a wait, about a second

struct DecodeGrid {
    int ctas;
    bool split;                     // a segment may be shared by several CTAs
    bool too_many;                  // more units than 32 bits count
    long long partial_floats;
};

DecodeGrid decode_grid(const Pool &pool, const Batch &bt, int hq, int max_count, int sms);
int launch_decode(const AttentionParams &p, const Pool &pool, int sms, cudaStream_t st);
bool make_pool_map(CUtensorMap *map, const Pool &pool, const void *base, int box_tokens);

}  // namespace paged
}  // namespace mk
