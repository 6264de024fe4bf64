// C entry points of the paged cache: argument checks, then the launches of
// paged_append.cu and paged_attention.cu.

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/b200_megakernel.h"
#include "paged.cuh"

namespace mk {

void set_last_error(const char *msg);  // megakernel.cu

namespace paged {

static int refuse(int code, const char *who, const char *text) {
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", who, text);
    set_last_error(msg);
    return code;
}

constexpr int kMaxKvHeads = 0x7fff;   // JoinEntry keeps a head in 16 bits

static bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// Pool and batch of a call, or an error code.
int read_cache(const MkPagedCache &c, const MkPagedBatch &b, int max_seqs, Pool &pool, Batch &bt, const char *who) {
    if (!c.k_pages || !c.v_pages || !b.page_table || !b.positions || !b.error_word)
        return refuse(MK_ERR_BAD_ARGUMENT, who, "null pointer");
    if (c.format != MK_CACHE_BF16 && c.format != MK_CACHE_E4M3) return refuse(MK_ERR_UNSUPPORTED, who, "unknown cache format");
    const bool fp8 = c.format == MK_CACHE_E4M3;
    if (fp8 && (!c.k_scales || !c.v_scales)) return refuse(MK_ERR_BAD_ARGUMENT, who, "an 8-bit cache needs its scales");
    if (c.head_dim != 64 && c.head_dim != 128) return refuse(MK_ERR_UNSUPPORTED, who, "head_dim must be 64 or 128");
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
        return refuse(MK_ERR_UNSUPPORTED, who, "page_size must be 16, 32, 64 or 128");
    if (c.num_pages < 1 || c.num_kv_heads < 1 || b.seqs < 1 || b.tokens < 1 || b.max_pages < 1)
        return refuse(MK_ERR_BAD_ARGUMENT, who, "empty cache or batch");
    if (b.seqs > max_seqs) return refuse(MK_ERR_UNSUPPORTED, who, "more sequences than one call takes");
    if (!b.cu_tokens && b.tokens % b.seqs) return refuse(MK_ERR_BAD_ARGUMENT, who, "rows do not divide evenly over the sequences");
    if (b.table_stride < b.max_pages && b.seqs > 1) return refuse(MK_ERR_BAD_ARGUMENT, who, "page table rows overlap");
    const int unit = fp8 ? 16 : 8;   // elements in 16 bytes
    if (misaligned(c.k_pages) || misaligned(c.v_pages) || c.page_stride <= 0 || c.head_stride <= 0 || c.slot_stride < c.head_dim ||
        c.page_stride % unit || c.head_stride % unit || c.slot_stride % unit || c.page_stride >= (1ll << 39) / (fp8 ? 1 : 2))
        return refuse(MK_ERR_UNSUPPORTED, who, "pages must start on 16-byte boundaries");
    pool.k = c.k_pages; pool.v = c.v_pages; pool.k_scales = fp8 ? c.k_scales : nullptr; pool.v_scales = fp8 ? c.v_scales : nullptr;
    pool.page_stride = c.page_stride; pool.head_stride = c.head_stride; pool.slot_stride = c.slot_stride;
    pool.num_pages = c.num_pages; pool.page_size = c.page_size; pool.kv_heads = c.num_kv_heads; pool.head_dim = c.head_dim; pool.fp8 = fp8;
    bt.table = b.page_table; bt.table_stride = b.table_stride; bt.where = b.positions; bt.cu = b.cu_tokens;
    bt.seqs = b.seqs; bt.tokens = b.tokens; bt.per_seq = b.cu_tokens ? 0 : b.tokens / b.seqs;
    bt.max_pages = b.max_pages; bt.num_pages = c.num_pages; bt.error = b.error_word; bt.where_offset = 0;
    bt.page_shift = 4;
    while ((1 << bt.page_shift) < c.page_size) ++bt.page_shift;
    return 0;
}

static bool bad_rows(const void *p, int64_t token, int64_t head) { return !p || misaligned(p) || token % 8 || head % 8 || token < 0 || head < 0; }

// SMs of the current device, asked for once per device.
static int sm_count(int &sms) {
    static int known[64] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && device < 64 && known[device]) {
        sms = known[device];
        return 0;
    }
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) set_last_error(cudaGetErrorString(e));
    else if (device < 64) known[device] = sms;
    return (int)e;
}

}  // namespace paged
}  // namespace mk

using namespace mk;
using namespace mk::paged;

extern "C" int mk_paged_append(const MkPagedCache *cache, const MkPagedBatch *batch, const MkPagedAppend *a, void *stream) {
    const char *who = "mk_paged_append";
    if (!cache || !batch || !a) return refuse(MK_ERR_BAD_ARGUMENT, who, "null argument");
    AppendParams p = {};
    int code = read_cache(*cache, *batch, MK_PAGED_MAX_SEQS, p.pool, p.bt, who);
    if (code) return code;
    if (cache->k_pages == cache->v_pages || (p.pool.fp8 && cache->k_scales == cache->v_scales))
        return refuse(MK_ERR_BAD_ARGUMENT, who, "keys and values need pages and scales of their own");
    if (bad_rows(a->k, a->k_token_stride, a->k_head_stride) || bad_rows(a->v, a->v_token_stride, a->v_head_stride))
        return refuse(MK_ERR_BAD_ARGUMENT, who, "key or value rows null or not on 16-byte boundaries");
    if ((a->q == nullptr) != (a->q_out == nullptr)) return refuse(MK_ERR_BAD_ARGUMENT, who, "q and q_out go together");
    if (a->q && (bad_rows(a->q, a->q_token_stride, a->q_head_stride) || misaligned(a->q_out) || a->num_q_heads < 1))
        return refuse(MK_ERR_BAD_ARGUMENT, who, "query rows null or not on 16-byte boundaries");
    if ((a->rope_cos == nullptr) != (a->rope_sin == nullptr)) return refuse(MK_ERR_BAD_ARGUMENT, who, "rope_cos and rope_sin go together");
    if (a->rope_cos && (a->rot_dim < 16 || a->rot_dim > cache->head_dim || a->rot_dim % 16 || a->rope_positions < 1 || misaligned(a->rope_cos) ||
                        misaligned(a->rope_sin)))
        return refuse(MK_ERR_UNSUPPORTED, who, "rotary tables need 16-byte alignment and a width that is a multiple of 16, at most head_dim");
    p.q = Rows{(const bf16 *)a->q, a->q_token_stride, a->q_head_stride};
    p.k = Rows{(const bf16 *)a->k, a->k_token_stride, a->k_head_stride};
    p.v = Rows{(const bf16 *)a->v, a->v_token_stride, a->v_head_stride};
    p.from_linear = false;
    p.q_out = (bf16 *)a->q_out;
    p.hq = a->q ? a->num_q_heads : 0;
    p.rope_cos = a->rope_cos; p.rope_sin = a->rope_sin; p.rot = a->rot_dim; p.positions = a->rope_positions;
    p.half = a->half_layout != 0;
    const cudaError_t e = launch_append(p, (cudaStream_t)stream);
    if (e != cudaSuccess) set_last_error(cudaGetErrorString(e));
    return (int)e;
}

extern "C" int64_t mk_paged_attention_workspace(const MkPagedCache *cache, const MkPagedBatch *batch, int32_t num_q_heads) {
    const char *who = "mk_paged_attention_workspace";
    Pool pool;
    Batch bt;
    if (!cache || !batch) return refuse(MK_ERR_BAD_ARGUMENT, who, "null argument"), -1;
    int sms = 0;
    if (read_cache(*cache, *batch, MK_PAGED_ATTENTION_MAX_SEQS, pool, bt, who) || sm_count(sms)) return -1;
    if (num_q_heads < 1 || num_q_heads % pool.kv_heads) return refuse(MK_ERR_UNSUPPORTED, who, "query heads are not a multiple of the KV heads"), -1;
    if (pool.kv_heads > kMaxKvHeads) return refuse(MK_ERR_UNSUPPORTED, who, "more KV heads than one call takes"), -1;
    const long long bytes = attention_workspace(bt, pool, num_q_heads, sms);
    if (bytes < 0) refuse(MK_ERR_UNSUPPORTED, who, "more rows times positions than one call takes");
    return bytes;
}

extern "C" int mk_paged_attention(const MkPagedCache *cache, const MkPagedBatch *batch, const MkPagedAttention *a, void *stream) {
    const char *who = "mk_paged_attention";
    if (!cache || !batch || !a) return refuse(MK_ERR_BAD_ARGUMENT, who, "null argument");
    AttentionParams p = {};
    Pool pool;
    int code = read_cache(*cache, *batch, MK_PAGED_ATTENTION_MAX_SEQS, pool, p.bt, who);
    if (code) return code;
    if (bad_rows(a->q, a->q_token_stride, a->q_head_stride) || !a->out || misaligned(a->out))
        return refuse(MK_ERR_BAD_ARGUMENT, who, "query or output rows null or not on 16-byte boundaries");
    if (a->num_q_heads < 1 || a->num_q_heads % pool.kv_heads)
        return refuse(MK_ERR_UNSUPPORTED, who, "query heads are not a multiple of the KV heads");
    if (pool.kv_heads > kMaxKvHeads) return refuse(MK_ERR_UNSUPPORTED, who, "more KV heads than one call takes");
    if (!(fabsf(a->scale) <= 3.0e38f)) return refuse(MK_ERR_BAD_ARGUMENT, who, "scale is not finite");
    int sms = 0;
    code = sm_count(sms);
    if (code) return code;
    const long long need = attention_workspace(p.bt, pool, a->num_q_heads, sms);
    if (need < 0) return refuse(MK_ERR_UNSUPPORTED, who, "more rows times positions than one call takes");
    if (need > 0 && (!a->workspace || misaligned(a->workspace) || a->workspace_bytes < need))
        return refuse(MK_ERR_BAD_ARGUMENT, who, "workspace null, misaligned or smaller than mk_paged_attention_workspace says");
    p.q = (const bf16 *)a->q; p.q_token = a->q_token_stride; p.q_head = a->q_head_stride;
    p.out = (bf16 *)a->out;
    p.k_scales = pool.k_scales; p.v_scales = pool.v_scales;
    p.hq = a->num_q_heads; p.hkv = pool.kv_heads; p.group = fast_div(a->num_q_heads / pool.kv_heads);
    p.scale_log2e = a->scale * 1.4426950408889634f;
    code = launch_attention(p, pool, a->workspace, sms, (cudaStream_t)stream);
    if (code > 0 && code < 10000) set_last_error(cudaGetErrorString((cudaError_t)code));
    return code;
}
