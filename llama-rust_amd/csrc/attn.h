// Host-callable launchers of the paged-cache operators (attn.hip).  Arguments have passed attn_plan.h's checks, and a call is launched only
// if .._fits() says that its launches hold it, which also says what workspace the launch takes.
#pragma once
#include <hip/hip_runtime.h>

#include "attn_plan.h"

namespace nh {

struct KvStoreCall {
    const lnh_kv_cache *cache;
    const lnh_kv_seqs *seqs;
    size_t layer;
    const float *k, *v;
    size_t k_stride, v_stride;
};
bool kv_store_fits(const KvStoreCall &c);
hipError_t launch_kv_store(hipStream_t stream, const KvStoreCall &c);

struct AttnCall {
    const lnh_kv_cache *cache;
    const lnh_kv_seqs *seqs;
    size_t layer, n_head;
    const float *q;
    float *out;
    size_t q_stride, out_stride;
    float scale;
    size_t window, sinks;
    bool weights;
    float decay;
};
// cus: compute units of the GPU.  ws holds at least *workspace bytes of the same call, 16-byte aligned.
bool attn_fits(const AttnCall &c, uint32_t cus, size_t *workspace);
hipError_t launch_attn(hipStream_t stream, const AttnCall &c, uint32_t cus, void *ws);

struct KvEvictCall {
    const lnh_kv_cache *cache;
    const lnh_kv_seqs *seqs;
    size_t first_layer, n_layers, keep, first, recent;
    const uint32_t *dst_tables;  // null: in place
    size_t dst_stride;
    uint32_t *new_lens;
};
bool kv_evict_fits(const KvEvictCall &c, size_t *workspace);
hipError_t launch_kv_evict(hipStream_t stream, const KvEvictCall &c, uint32_t cus, void *ws);

}  // namespace nh
