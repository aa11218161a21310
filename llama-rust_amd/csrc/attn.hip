// Operators over a paged K/V cache for gfx950 (include/native_hip_attention.h): kernels and their launchers.
//
// A row is a query head of a new token.  The G = n_head / n_head_kv query heads of a key-value head read the same cache
// rows, so the rows of a sequence and key-value head are kept together, token after token: row r is head r % G of new
// token r / G.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn.h"

namespace nh {

namespace {

using half8 = _Float16 __attribute__((ext_vector_type(8)));
using half4 = _Float16 __attribute__((ext_vector_type(4)));
using float4v = float __attribute__((ext_vector_type(4)));
using uint4v = uint32_t __attribute__((ext_vector_type(4)));
using uint2v = uint32_t __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896340736f;

#include "attn_q4.inc"
#include "attn_rows.inc"
#include "attn_split.inc"
#include "attn_chunk.inc"
#include "attn_weights.inc"
#include "kv_append.inc"
#include "kv_store.inc"
#include "kv_evict.inc"
#include "kv_bounds.inc"

KvPlace kv_place(const lnh_kv_cache &c, const uint32_t *tables, size_t stride) {
    KvPlace p;
    p.tables = tables;
    p.table_stride = (uint32_t)stride;
    p.n_blocks = c.n_blocks;
    p.block_rows = c.n_layer * c.n_head_kv * c.kv_block;
    p.kv_block = fast_div(c.kv_block);
    return p;
}

KvSeqsView kv_seqs(const lnh_kv_seqs &s) {
    return {s.device_starts, s.device_lens, (uint32_t)s.n_tokens, (uint32_t)std::min(s.max_new, s.n_tokens), (uint32_t)s.max_len, (uint32_t)s.n_seqs};
}

}  // namespace

#include "attn_launch.inc"

}  // namespace nh
