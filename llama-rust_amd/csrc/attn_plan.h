// Operators over the paged K/V cache (include/native_hip_attention.h): what is checked before a launch, which tiles of
// positions a group of rows reads, where a position lies.  No device needed; the kernels use the same functions.
#ifndef NATIVE_HIP_ATTN_PLAN_H
#define NATIVE_HIP_ATTN_PLAN_H

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "../../include/native_hip_attention.h"

#if defined(__HIPCC__)
#define NH_ATTN_HD __host__ __device__ __forceinline__
#else
#define NH_ATTN_HD inline
#endif

namespace nh {

constexpr size_t ATTN_MAX_POSITIONS = ((size_t)1 << 31) - 4096;  // positions are kept in 32 bits with room for a tile
constexpr size_t ATTN_MAX_ROWS = (size_t)1 << 31;                // of head_dim, in the whole cache
constexpr uint32_t ATTN_MAX_HEAD_DIM = 256;

// n / d for n < 2^31 and 0 < d <= 2^31 by a multiplication.
struct FastDiv {
    uint32_t d, magic, shift;
};
inline FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while (f.shift < 32 && ((uint64_t)1 << f.shift) < d) f.shift++;
    f.magic = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << f.shift) - d)) / d + 1);
    return f;
}
NH_ATTN_HD uint32_t div_by(const FastDiv &f, uint32_t n) {
    return ((uint32_t)(((uint64_t)f.magic * n) >> 32) + n) >> f.shift;
}

// A sequence of the call: its rows of the token-major arrays, how many of them the call takes, where they stand.
struct SeqRows {
    uint32_t row0, n;   // first row, rows taken (at most max_new)
    int32_t first_pos;  // position of the first new token, below zero where there are more new tokens than positions
    uint32_t len;
};
NH_ATTN_HD SeqRows seq_rows(const uint32_t *starts, const uint32_t *lens, uint32_t b, uint32_t n_tokens, uint32_t max_new, uint32_t max_len) {
    SeqRows s;
    uint32_t from = starts ? starts[b] : b, to = starts ? starts[b + 1] : b + 1;
    to = to < n_tokens ? to : n_tokens;
    from = from < to ? from : to;
    s.row0 = from;
    const uint32_t all = to - from;
    s.n = all < max_new ? all : max_new;
    s.len = lens[b] < max_len ? lens[b] : max_len;
    s.first_pos = (int32_t)s.len - (int32_t)all;
    return s;
}

// Whether the token at position p sees position t (a token below zero sees nothing).
NH_ATTN_HD bool attn_sees(int32_t p, uint32_t t, uint32_t window, uint32_t sinks) {
    if (p < 0 || t > (uint32_t)p) return false;
    return window == 0 || (uint32_t)p - t < window || t < sinks;
}

// The sequence's new tokens that see position t: from .. to.
struct SeenBy {
    uint32_t from, to;
};
NH_ATTN_HD SeenBy attn_seen_by(const SeqRows &s, uint32_t t, uint32_t window, uint32_t sinks) {
    const int64_t from = (int64_t)t - s.first_pos, to = from + window, n = s.n;
    return {(uint32_t)(from < 0 ? 0 : from < n ? from : n), (uint32_t)(window == 0 || t < sinks || to > n ? n : to < 0 ? 0 : to)};
}

// The tiles of `tp` positions that tokens at first_pos .. last_pos read, the first tokens' and then the window's, none twice.
struct AttnTiles {
    uint32_t sink_tiles, from, count;
    uint32_t lo, hi;  // positions of the window, of all tokens together
};
NH_ATTN_HD AttnTiles attn_tiles(int32_t first_pos, int32_t last_pos, uint32_t window, uint32_t sinks, uint32_t tp) {
    AttnTiles r{0, 0, 0, 0, 0};
    if (last_pos < 0) return r;
    const uint32_t p0 = first_pos > 0 ? (uint32_t)first_pos : 0u;
    r.hi = (uint32_t)last_pos + 1;
    r.lo = window != 0 && p0 + 1 > window ? p0 + 1 - window : 0;
    r.from = r.lo / tp;
    const uint32_t first = sinks < r.lo ? sinks : r.lo;
    const uint32_t st = (first + tp - 1) / tp;
    r.sink_tiles = st < r.from ? st : r.from;
    r.count = r.sink_tiles + (r.hi + tp - 1) / tp - r.from;
    return r;
}
NH_ATTN_HD uint32_t attn_tile(const AttnTiles &r, uint32_t j) { return j < r.sink_tiles ? j : r.from + (j - r.sink_tiles); }
// Share s of n: tiles [begin, end).
NH_ATTN_HD uint32_t attn_share(uint32_t count, uint32_t s, uint32_t n) { return (uint32_t)((uint64_t)count * s / n); }

// Sequences of a call whose launches are made together, the others behind them.  Few rows: every workgroup looks at all of them, which takes a
// call's time with their square (8192 of up to 200 f16 positions, 8 heads: 18.4 ms at once, 4.1 in parts of 1024, 3.1 of 512, 2.7 of 256; 512
// of them 196 and 169 us).  score_bytes: workspace for the weights that a sequence takes by its bounds.
constexpr size_t ATTN_SEQS_AT_ONCE = 256, ATTN_SCORES_AT_ONCE = (size_t)1 << 30;
inline size_t attn_seqs_at_once(size_t n_seqs, bool few_rows, size_t score_bytes) {
    size_t most = few_rows && n_seqs > ATTN_SEQS_AT_ONCE ? ATTN_SEQS_AT_ONCE : n_seqs;
    if (score_bytes != 0 && most > ATTN_SCORES_AT_ONCE / score_bytes) most = ATTN_SCORES_AT_ONCE / score_bytes;
    if (most == 0) most = 1;
    const size_t parts = (n_seqs + most - 1) / most;
    return parts ? (n_seqs + parts - 1) / parts : 0;
}

// Where a position lies, in rows of head_dim from the start of K or V; ATTN_NOWHERE for a block the cache does not have or
// an entry the table does not have.
constexpr uint32_t ATTN_NOWHERE = 0xffffffffu;
struct KvPlace {
    const uint32_t *tables;
    uint32_t table_stride, n_blocks;
    uint32_t block_rows;  // n_layer * n_head_kv * kv_block
    FastDiv kv_block;
};
NH_ATTN_HD uint32_t kv_row(const KvPlace &k, const uint32_t *table, uint32_t head_rows, uint32_t t) {
    const uint32_t e = div_by(k.kv_block, t);
    if (e >= k.table_stride) return ATTN_NOWHERE;
    const uint32_t id = table[e];
    if (id >= k.n_blocks) return ATTN_NOWHERE;
    return id * k.block_rows + head_rows + (t - e * k.kv_block.d);
}

// The many-row kernels keep a row of K or V in LDS as 16-byte pieces, attn_pitch of them; their registers take dp head elements.
constexpr uint32_t attn_piece(bool half) { return half ? 8 : 4; }  // head elements of a piece
constexpr uint32_t attn_many_dims(bool half, uint32_t d) {
    return d <= 64 ? 64 : half && d <= 96 ? 96 : d <= 128 ? 128 : half && d <= 192 ? 192 : 256;
}
constexpr uint32_t attn_pitch(bool half, uint32_t dp) { return half ? (dp > 128 ? 32 : dp > 64 ? 16 : 8) : dp / 4; }
// Whether piece c of a place in LDS is loaded: only what the row has, d elements.  Where dp == d is known but the place is wider than the
// row (f16 heads of 96 and 192), the pieces behind it are the next row's or, behind the last row, nobody's.
NH_ATTN_HD bool attn_brings(bool half, uint32_t dp, uint32_t d, uint32_t c) {
    return (dp == d && attn_pitch(half, dp) * attn_piece(half) == dp) || c * attn_piece(half) < d;
}

// ------------------------------------------------------------------ checks: a code and a message, LNH_OK and null if fine
struct AttnCheck {
    int code;
    const char *what;
};
inline bool attn_misaligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

inline AttnCheck check_kv_cache(const lnh_kv_cache *c, bool weights) {
    if (!c) return {LNH_ERR_INVALID, "K/V cache description is null"};
    if (c->ggml_type != LNH_TYPE_F32 && c->ggml_type != LNH_TYPE_F16) return {LNH_ERR_UNSUPPORTED, "the K/V cache is f32 or f16"};
    if (c->n_layer == 0 || c->n_head_kv == 0 || c->head_dim == 0 || c->kv_block == 0 || c->n_blocks == 0)
        return {LNH_ERR_INVALID, "K/V cache dimensions must be positive"};
    if (c->head_dim % 8 != 0 || c->head_dim > ATTN_MAX_HEAD_DIM)
        return {LNH_ERR_UNSUPPORTED, "the K/V cache takes head sizes that are multiples of 8, at most 256"};
    size_t rows = 1;
    for (const uint32_t n : {c->n_layer, c->n_head_kv, c->kv_block, c->n_blocks}) {
        rows *= n;  // below 2^31 times at most 2^32
        if (rows > ATTN_MAX_ROWS) return {LNH_ERR_INVALID, "the K/V cache exceeds 2^31 rows"};
    }
    if (!c->device_k || !c->device_v) return {LNH_ERR_INVALID, "buffer pointer is null"};
    if (weights && !c->device_w) return {LNH_ERR_INVALID, "the K/V cache has no weights"};
    if (attn_misaligned(c->device_k, 16) || attn_misaligned(c->device_v, 16) || attn_misaligned(c->device_w, 16))
        return {LNH_ERR_INVALID, "device buffers must be 16-byte aligned"};
    return {LNH_OK, nullptr};
}

inline AttnCheck check_kv_seqs(const lnh_kv_cache *c, const lnh_kv_seqs *s, bool rows) {
    if (!s) return {LNH_ERR_INVALID, "sequence description is null"};
    if (s->n_seqs == 0) return {LNH_OK, nullptr};
    if (!s->device_tables || !s->device_lens) return {LNH_ERR_INVALID, "buffer pointer is null"};
    if (attn_misaligned(s->device_tables, 4) || attn_misaligned(s->device_lens, 4) || attn_misaligned(s->device_starts, 4))
        return {LNH_ERR_INVALID, "device tables, lengths and starts must be 4-byte aligned"};
    if (s->n_seqs > ATTN_MAX_POSITIONS || s->max_len > ATTN_MAX_POSITIONS || s->table_stride > ATTN_MAX_POSITIONS)
        return {LNH_ERR_INVALID, "sequences, positions or table entries exceed 31 bits"};
    if (s->max_len > s->table_stride * (size_t)c->kv_block) return {LNH_ERR_INVALID, "max_len exceeds what the block tables hold"};
    if (!rows) return {LNH_OK, nullptr};
    if (s->n_tokens > ATTN_MAX_POSITIONS || s->max_new > ATTN_MAX_POSITIONS) return {LNH_ERR_INVALID, "tokens exceed 31 bits"};
    if (!s->device_starts && s->n_tokens != s->n_seqs) return {LNH_ERR_INVALID, "without row starts there is one token per sequence"};
    return {LNH_OK, nullptr};
}

inline AttnCheck check_rows(const void *p, size_t stride, size_t width) {
    if (!p) return {LNH_ERR_INVALID, "buffer pointer is null"};
    if (attn_misaligned(p, 16)) return {LNH_ERR_INVALID, "device buffers must be 16-byte aligned"};
    if (stride % 4 != 0) return {LNH_ERR_INVALID, "row strides must be multiples of four floats"};
    if (stride < width) return {LNH_ERR_INVALID, "a row stride is less than the row"};
    if (stride > ((size_t)1 << 40)) return {LNH_ERR_INVALID, "a row stride exceeds 2^40"};
    return {LNH_OK, nullptr};
}

inline AttnCheck check_attn(const lnh_kv_cache *c, const lnh_kv_seqs *s, size_t layer, size_t n_head, const float *q, size_t q_stride,
                            const float *out, size_t out_stride, float scale, size_t window, size_t sinks, int weights, float decay) {
    AttnCheck r = check_kv_cache(c, weights != 0);
    if (!r.what) r = check_kv_seqs(c, s, true);
    if (r.what) return r;
    if (layer >= c->n_layer) return {LNH_ERR_INVALID, "the K/V cache has no such layer"};
    if (n_head == 0 || n_head % c->n_head_kv != 0) return {LNH_ERR_INVALID, "query heads must be a multiple of the key-value heads"};
    if (n_head > 65536) return {LNH_ERR_INVALID, "more than 65536 query heads"};
    if (s->max_new > ATTN_MAX_POSITIONS / (n_head / c->n_head_kv)) return {LNH_ERR_INVALID, "tokens times query heads exceed 31 bits"};
    if (!std::isfinite(scale) || !std::isfinite(decay)) return {LNH_ERR_INVALID, "scale and decay must be finite"};
    // places that a row does not see are given minus infinity before the multiplication; 2^127 leaves room for log2(e)
    if (scale <= 0.f || scale > 0x1p127f) return {LNH_ERR_INVALID, "scale must be positive, at most 2^127"};
    if (window > ATTN_MAX_POSITIONS || sinks > ATTN_MAX_POSITIONS) return {LNH_ERR_INVALID, "window or sinks exceed 31 bits"};
    if (window == 0 && sinks != 0) return {LNH_ERR_INVALID, "first tokens stay visible beside a window: sinks without one"};
    if (s->n_seqs == 0 || s->n_tokens == 0 || s->max_new == 0) return {LNH_OK, nullptr};
    r = check_rows(q, q_stride, n_head * c->head_dim);
    if (!r.what) r = check_rows(out, out_stride, n_head * c->head_dim);
    if (!r.what && q == out) r = {LNH_ERR_INVALID, "the output must not be the input"};
    return r;
}

inline AttnCheck check_kv_store(const lnh_kv_cache *c, const lnh_kv_seqs *s, size_t layer, const float *k, size_t k_stride, const float *v,
                                size_t v_stride) {
    AttnCheck r = check_kv_cache(c, false);
    if (!r.what) r = check_kv_seqs(c, s, true);
    if (r.what) return r;
    if (layer >= c->n_layer) return {LNH_ERR_INVALID, "the K/V cache has no such layer"};
    if (s->n_seqs == 0 || s->n_tokens == 0 || s->max_new == 0) return {LNH_OK, nullptr};
    const size_t width = (size_t)c->n_head_kv * c->head_dim;
    r = check_rows(k, k_stride, width);
    return r.what ? r : check_rows(v, v_stride, width);
}

inline AttnCheck check_kv_evict(const lnh_kv_cache *c, const lnh_kv_seqs *s, size_t first_layer, size_t n_layers, size_t keep, size_t first,
                                size_t recent, const uint32_t *dst, size_t dst_stride, const uint32_t *new_lens) {
    AttnCheck r = check_kv_cache(c, true);
    if (!r.what) r = check_kv_seqs(c, s, false);
    if (r.what) return r;
    if (n_layers == 0 || first_layer >= c->n_layer || n_layers > c->n_layer - first_layer)
        return {LNH_ERR_INVALID, "the K/V cache has no such layers"};
    if (keep > ATTN_MAX_POSITIONS) return {LNH_ERR_INVALID, "keep exceeds 31 bits"};
    if (first > keep || recent > keep - first) return {LNH_ERR_INVALID, "first and recent positions together exceed those to keep"};
    if (s->n_seqs == 0) return {LNH_OK, nullptr};
    if (!new_lens) return {LNH_ERR_INVALID, "buffer pointer is null"};
    if (attn_misaligned(dst, 4) || attn_misaligned(new_lens, 4)) return {LNH_ERR_INVALID, "device tables, lengths and starts must be 4-byte aligned"};
    if (dst && dst != s->device_tables) {
        const size_t most = keep < s->max_len ? keep : s->max_len;
        if (dst_stride > ATTN_MAX_POSITIONS) return {LNH_ERR_INVALID, "sequences, positions or table entries exceed 31 bits"};
        if (most > dst_stride * (size_t)c->kv_block) return {LNH_ERR_INVALID, "the destination tables do not hold what is kept"};
    }
    return {LNH_OK, nullptr};
}

}  // namespace nh
#endif
