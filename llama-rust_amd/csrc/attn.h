// Host-callable launchers of the paged-cache operators (attn.hip).  Arguments have passed attn_plan.h's checks, and a call is launched only
// if .._fits() says that its launches hold it, which also says what workspace the launch takes.
#pragma once
#include <hip/hip_runtime.h>

#include "attn_launch_plan.h"

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

// The rotation on the way and q with it; launch_kv_load: k and v are written.
struct KvAppendCall {
    const lnh_kv_cache *cache;
    const lnh_kv_seqs *seqs;
    size_t layer;
    const lnh_rope *rope;  // may be null
    size_t n_head;
    const float *q;
    float *q_out;
    size_t q_stride, q_out_stride;
    const float *k, *v;
    size_t k_stride, v_stride;
};
bool kv_append_fits(const KvAppendCall &c);
hipError_t launch_kv_append(hipStream_t stream, const KvAppendCall &c);
hipError_t launch_kv_load(hipStream_t stream, const KvAppendCall &c, float *k, float *v);
hipError_t launch_rope_table(hipStream_t stream, uint32_t n_rot, double base, double scale, const float *divisors, size_t n_positions, float *angles,
                             size_t stride);

// cus: compute units of the GPU.  ws holds at least what attn_fits() said of the same call, 16-byte aligned.
hipError_t launch_attn(hipStream_t stream, const AttnCall &c, uint32_t cus, void *ws);

struct KvBoundsCall {
    const lnh_kv_cache *cache;
    const lnh_kv_seqs *seqs;
    size_t layer;
    void *bounds;
};
bool kv_bounds_fits(const KvBoundsCall &c);
hipError_t launch_kv_bounds(hipStream_t stream, const KvBoundsCall &c);

hipError_t launch_attn_select(hipStream_t stream, const AttnSelectCall &c, uint32_t cus, void *ws);

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
