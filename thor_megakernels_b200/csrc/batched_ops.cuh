// Launchers of the memory-bound operators of a batched decode step
// (batched_ops.cu) and of the tensor-core linear (linear_batched.cu).
#pragma once

#include <cuda_runtime.h>

#include "mk_device.cuh"

namespace mk {
namespace bo {

struct LinOut {
    const bf16 *y;
    const float *partials;
    int splits, batch, n;
    float scale;
    int group;  // residual adds only: consecutive splits that form one bf16-rounded addend (0: all of them)
};

// A LinOut is the result of a batched linear as its consumers
// read it: bf16 y [batch, n], or the fp32 split-K partial sums [splits, batch, n],
// which are added here in split order, scaled and rounded to bf16 once - the
// value y would hold.
__device__ __forceinline__ float lin_value(const LinOut &o, int b, int i) {
    if (o.partials == nullptr) return __bfloat162float(o.y[(size_t)b * o.n + i]);
    float total = 0.f;
    for (int s = 0; s < o.splits; ++s) total += o.partials[((size_t)s * o.batch + b) * o.n + i];
    return round_bf16(total * o.scale);
}

// Two / four consecutive elements (i even / a multiple of 4): vector loads, the splits'
// loads independent of one another so that they are in flight together.
__device__ __forceinline__ float2 lin_value2(const LinOut &o, int b, int i) {
    if (o.partials == nullptr) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(o.y + (size_t)b * o.n + i));
    float2 total = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < o.splits; ++s) {
        const float2 v = *reinterpret_cast<const float2 *>(o.partials + ((size_t)s * o.batch + b) * o.n + i);
        total.x += v.x; total.y += v.y;
    }
    return make_float2(round_bf16(total.x * o.scale), round_bf16(total.y * o.scale));
}

__device__ __forceinline__ float4 load_bf16x4(const bf16 *p) {
    const uint2 raw = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store_bf16x4(bf16 *p, const float4 &v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    uint2 raw;
    raw.x = *reinterpret_cast<const uint32_t *>(&a);
    raw.y = *reinterpret_cast<const uint32_t *>(&b);
    *reinterpret_cast<uint2 *>(p) = raw;
}

// sum of splits [s0, s1) for elements i..i+3, times the scale, rounded to bf16
__device__ __forceinline__ float4 partial_sum4(const LinOut &o, int b, int i, int s0, int s1) {
    float4 total = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = s0; s < s1; ++s) {
        const float4 v = *reinterpret_cast<const float4 *>(o.partials + ((size_t)s * o.batch + b) * o.n + i);
        total.x += v.x; total.y += v.y; total.z += v.z; total.w += v.w;
    }
    return make_float4(round_bf16(total.x * o.scale), round_bf16(total.y * o.scale), round_bf16(total.z * o.scale),
                       round_bf16(total.w * o.scale));
}
__device__ __forceinline__ float4 lin_value4(const LinOut &o, int b, int i) {
    if (o.partials == nullptr) return load_bf16x4(o.y + (size_t)b * o.n + i);
    return partial_sum4(o, b, i, 0, o.splits);
}

}  // namespace bo

// Launch on `st` with the programmatic-stream-serialization attribute (see pdl_wait in
// mk_device.cuh): the kernel may be scheduled while its predecessor is still running.
// mk_batched_set_overlap(0) turns the attribute off (plain stream order).
bool launch_overlap_enabled();
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = launch_overlap_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

cudaError_t launch_embed(const bf16 *embed, const int *tokens, bf16 *hidden, int batch, int hidden_size, int vocab, int *error,
                         cudaStream_t st);
cudaError_t launch_residual_norm(bf16 *hidden, const bo::LinOut &lin, int add, const bf16 *weight, bf16 *normed, int batch,
                                 int hidden_size, float eps, cudaStream_t st);
cudaError_t launch_rope_append(const bo::LinOut &qkv, const int *pos_ids, const float *rope_cos, const float *rope_sin, bf16 *q_out,
                               bf16 *k_cache, bf16 *v_cache, int layer, int rows, int cache_batch, int kv_len, int hq, int hkv,
                               int hd, int half_split, int slot_fixed, cudaStream_t st);
cudaError_t launch_sanitize_positions(const int *pos_ids, int *pos_out, int batch, int pos_limit, bool idle, int *error, cudaStream_t st);
cudaError_t launch_fill_int(int *dst, int value, int step, int n, cudaStream_t st);
cudaError_t launch_barrier_fill(int *barriers, const int *covered, int layers, int batch, int cols, int batch_blocks, int hq,
                                int hkv, int out_blocks, int inter_blocks, cudaStream_t st);
int attention_batched_splits(int batch, int hkv, int sms, int max_splits);
cudaError_t launch_attention_batched(const bf16 *q, const bf16 *k_cache, const bf16 *v_cache, const int *pos_ids, bf16 *out,
                                     float *partial, int splits, int layer, int batch, int cache_batch, int kv_len, int hq, int hkv,
                                     int hd, float attn_scale, int slot_fixed, cudaStream_t st);
cudaError_t launch_silu_mul(const bo::LinOut &up, const bo::LinOut &gate, bf16 *act, int batch, int inter, int round_silu,
                            cudaStream_t st);
cudaError_t launch_argmax(const bf16 *logits, int *tokens, int batch, int vocab, cudaStream_t st);

}  // namespace mk
