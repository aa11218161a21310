// Attention over the paged cache: which kernels a call takes, how it is cut for them, what workspace that wants.  No device needed.
#ifndef NATIVE_HIP_ATTN_LAUNCH_PLAN_H
#define NATIVE_HIP_ATTN_LAUNCH_PLAN_H

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_plan.h"

namespace nh {

// Workgroups of a launch: a launch counts its threads, at most 512 a workgroup (eviction: 1024), in 32 bits.
constexpr size_t MOST_GROUPS = 0x3fffff;

constexpr size_t ROW_WEIGHT_BYTES = 8;  // attn_rows.inc's RowWeight

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
    size_t head_tables;  // entries of a key-value head's own table, every row a sequence (launch_attn_select); else 0
};

struct AttnSelectCall {
    AttnCall attn;  // no window, no weights
    const void *bounds;
    size_t n_select, first, recent;
    uint32_t *chosen;  // may be null
};

constexpr size_t CHUNK_SUMS_BYTES = (size_t)256 << 20;  // attn_chunk_kernel: what shares may leave

struct AttnPlan {
    bool fits;  // every launch holds its workgroups
    uint32_t row_tiles;
    uint32_t chunk_rows, splits;  // the many-row kernel: rows of a workgroup (0: the few-row kernel runs), shares of a unit's tiles
    uint32_t least_tiles, rounds_of, most_shares, groups;  // the few-row kernel: AttnArgs's, and its workgroups
    uint32_t part_rows;
    bool few_rows;  // eight a unit at most
    bool joined;  // the few-row kernel: units may have several shares
    uint32_t unit_waves;  // not joined: wavefronts of a unit, log2
    uint32_t first_blocks;
    float *piece_sums;
    size_t units;                 // sequences x key-value heads x row tiles
    uint32_t score_rows;          // weights from kept scores: rows of a key-value head, else 0
    uint32_t chunk_groups, weight_groups;  // workgroups of attn_chunk_kernel and attn_weights_kernel
    uint32_t weight_rows, weight_splits;  // weights of more rows: attn_weights_kernel's chunk_rows and splits
    size_t score_stride, stat_at, parts_at, row_weight_at, score_at, bytes;
};

// How blocks of rows are cut: the last block of a sequence into `shares`, the others into shares of that size.
struct ChunkCut {
    uint32_t shares;
    float us;  // by the estimate below
};
// What a position of a block takes, one workgroup on a compute unit and two; what every round of workgroups takes besides; what shares take: a
// launch, and a share's sums their way through memory.
struct ChunkCost {
    float alone, beside, start, join, part;
};
// Of `blocks` blocks that read `first` to `most` positions, evenly, two workgroups at a time on each of `cus` compute units.
inline ChunkCut cut_blocks(size_t blocks, float first, float most, uint32_t cus, const ChunkCost &c, size_t most_shares) {
    const float n = (float)blocks, units = (float)cus;
    const float rounds = n / (2.f * units);
    // whole blocks, the longest first: all at once, short ways beside long ones (chunk_order), or in turn, the shortest last
    float t = n <= units       ? most * c.alone
              : rounds <= 1.f ? std::max(first * c.beside + (most - first) * c.alone, (first + most) / 2.f * c.beside)
                              : rounds * (first + most) / 2.f * c.beside + first * (std::ceil(rounds) - rounds) * c.alone;
    ChunkCut best{1, t + c.start * std::ceil(rounds)};
    for (uint32_t shares = 2; shares <= std::min<size_t>(most_shares, 64); shares++) {
        const float all = n * ((first + most) * (float)shares + most - first) / (2.f * most), whole = std::floor(all / (2.f * units)), rest = all - whole * 2.f * units;
        t = most / (float)shares * (whole * c.beside + (rest <= 0.f ? 0.f : rest <= units ? c.alone : c.beside)) + c.start * std::ceil(all / (2.f * units)) + c.join +
            c.part * all;
        if (t < best.us) best = {shares, t};
    }
    return best;
}

// Blocks of n rows that a call is likely to have, sequences as long as they may be and their new tokens as many as there are rows, and the
// positions that the first and the last of a sequence read.
struct BlockReads {
    size_t blocks;
    float first, most;
};
inline BlockReads block_reads(const AttnCall &c, size_t n, size_t seen, size_t max_new) {
    const size_t group = c.n_head / c.cache->n_head_kv;
    const size_t blocks = std::min(c.seqs->n_seqs * ((max_new * group + n - 1) / n), (c.seqs->n_tokens * group + n - 1) / n + c.seqs->n_seqs / 2);
    if (c.window != 0) seen = std::min(seen, c.window + c.sinks + n / group + 64);
    const size_t first = c.window != 0 ? seen : seen > max_new ? seen - max_new : 0;
    return {std::max<size_t>(blocks, 1) * c.cache->n_head_kv, (float)first, (float)std::max<size_t>(seen, 1)};
}

inline AttnPlan attn_plan(const AttnCall &c, uint32_t cus) {
    AttnPlan p{};
    p.fits = true;
    const size_t group = c.n_head / c.cache->n_head_kv, max_new = std::min(c.seqs->max_new, c.seqs->n_tokens), rows = max_new * group;
    const size_t heads = c.seqs->n_seqs * c.cache->n_head_kv;
    if (rows == 0 || heads == 0) return p;  // nothing to do
    p.row_tiles = (uint32_t)((rows + 15) / 16);
    p.fits = heads <= MOST_GROUPS && heads * p.row_tiles <= MOST_GROUPS;
    if (!p.fits) return p;
    p.units = heads * (size_t)p.row_tiles;
    const bool half = c.cache->ggml_type != LNH_TYPE_F32;  // f16 operands
    const size_t tp = half ? 32 : 16;
    size_t seen = c.seqs->max_len;
    if (c.window != 0) seen = std::min(seen, c.window + max_new + c.sinks + 2 * tp);
    size_t slots = 0;  // of sums that are joined
    p.splits = 1;
    if (rows > 32) {
        // 128 rows a workgroup read the cache half as often as 64, which balance better; shares fill the chip.  The costs are those of heads of
        // 128 on MI355X, with which the estimate is within a tenth of the time of most calls.  8 key-value heads of 4 query heads, us, the
        // chosen and what else there is: 512 f16 tokens alone 21 in blocks of 64 (three shares 27, 128 rows in four 32), behind 3584
        // positions 79 in four shares of 128 rows (64 whole 111, in two 87, 128 whole 156); 1024 f32 tokens alone 101 in blocks of 64 (128
        // rows in three 127); 16 tokens of each of 32 sequences of 4096 f16 119 in two shares (whole 162, three 147), f32 347 (447, 375)
        const float width = (float)c.cache->head_dim / 128.f;
        // room for sums is by sequences and their bounds, which may be far beyond the rows that there are
        const size_t most_shares = std::max<size_t>(1, CHUNK_SUMS_BYTES / (p.units * 16 * c.cache->head_dim * 4));
        const auto cut = [&](size_t n, float alone, float beside) {
            const ChunkCost cost{alone * width, beside * width, 3.f, 6.f, (float)n * width * 512.f * 2.f / 4e6f};
            const BlockReads r = block_reads(c, n, seen, max_new);
            return cut_blocks(r.blocks, r.first, r.most, cus, cost, std::min((size_t)(r.most + 127.f) / 128, most_shares));
        };
        const bool packed = c.cache->ggml_type == LNH_TYPE_Q4_0;  // every block of rows unpacks what it reads
        const ChunkCut small = packed ? cut(64, 0.040f, 0.055f) : half ? cut(64, 0.025f, 0.033f) : cut(64, 0.095f, 0.150f);
        const ChunkCut large = packed ? cut(128, 0.050f, 0.075f) : half ? cut(128, 0.036f, 0.052f) : cut(128, 0.152f, 0.260f);
        p.chunk_rows = c.cache->head_dim > 128 || small.us <= large.us ? 64 : 128;
        p.splits = p.chunk_rows == 64 ? small.shares : large.shares;
        const size_t groups = (rows + p.chunk_rows - 1) / p.chunk_rows * heads;
        slots = p.splits > 1 ? p.units * p.splits : 0;
        // 2048 f32 tokens, 128 rows a workgroup: dealt so 337 us, the longest first 413; behind 6144 positions 1892 and 1990 us, f16 410 and 423
        p.first_blocks = p.splits == 1 && groups <= 2 * (size_t)cus ? (uint32_t)((cus + heads - 1) / heads) : 0xffffffffu;
    } else {
        // a tile on each SIMD: with two in turn a call behind 200 f32 positions took 13 us and no join, with two at a time 11.7 us
        p.few_rows = rows <= 8;
        // (4-bit tiles, whose rows take an instruction an element or so, one a wavefront: behind 1000 to 2000 positions 11.5 us, 13 with two)
        p.least_tiles = c.cache->ggml_type == LNH_TYPE_Q4_0 ? 8 : 4;
        // Whole units, with nothing to find and to join, where a call is short whatever its lengths (256 sequences of up to 30 positions, 8 heads of
        // 128: f16 63 us as shares, 36 a workgroup a unit, 10.6 eight a workgroup, a wavefront each; f32 64, 39, 12; one of 4 bits behind 60 8.2 and 6.6)
        // or whole units of the longest would be done sooner than shares of lengths that differ (shares and whole: one behind 400 positions, 4 bits 11.7
        // and 9.4 us, f16 11.4 and 10.2, behind 1500 12.7 and 15.2, 12.2 and 20.7; 32 sequences of lengths up to 1000 4 bits 17.5 and 12.3, f16 24.7 and
        // 18.7, up to 400 f32 24.4 and 19.1; 256 of up to 700 93 and 38, 133 and 87), and where chosen blocks, which have one length,
        // are more than one unit a compute unit (2048 tokens of 1024 f16 positions each, with the choice, 1510 and 920).
        const size_t tiles = (seen + tp - 1) / tp, waves = c.cache->head_dim > 128 ? 4 : 8;
        const bool packed = c.cache->ggml_type == LNH_TYPE_Q4_0, chosen = c.head_tables != 0;
        const float tile_us = (packed ? 1.5f : half ? 2.9f : 4.f) * (0.4f + 0.6f * (float)c.cache->head_dim / 128.f);
        const float alone_us = p.few_rows ? 5.f : 6.5f;  // what a workgroup takes besides
        // rounds of workgroups with `n` units each, every unit the longest
        const auto whole_us = [&](size_t n) { return (float)((p.units + n * cus - 1) / (n * cus)) * (alone_us + (float)((tiles * n + waves - 1) / waves) * tile_us); };
        size_t side = 1;  // units of a workgroup
        for (size_t n = 2; n <= waves; n *= 2)
            if (whole_us(n) < whole_us(side)) side = n;
        // shares: finding and joining them, and, once few compute units are left over, a round for every unit a compute unit with its tiles, half as many as
        // of the longest, evenly (chosen blocks: as many).  Over f32 and f16 caches without that round up to half of the compute units, where a long
        // sequence beside short ones would wait for its one workgroup (16 sequences of 30 positions and one of 700, f16: 10.5 us as shares, 13.5 whole;
        // all of 700: 17.8 and 15.4)
        const float load = (float)p.units / (float)cus, round_us = !packed && !chosen && load <= 0.5f ? 0.f : 6.f;
        const float shares_us = 11.5f + (round_us + (float)tiles / (chosen ? 1.f : 2.f) / waves * tile_us) * std::max(load - 0.2f, 0.f);
        const bool soon = whole_us(side) <= shares_us;
        // shares count the tiles of all units together, in 32 bits
        const bool counted = c.seqs->max_len / tp + 2 <= 0x7fffffffu / p.units;
        p.joined = tiles > p.least_tiles && !soon && !(chosen && (p.units > cus || !counted));
        p.fits = !p.joined || counted;
        if (!p.joined) {
            p.unit_waves = (uint32_t)__builtin_ctz((uint32_t)(waves / side));
            p.groups = (uint32_t)((c.seqs->n_seqs * p.row_tiles + side - 1) / side * c.cache->n_head_kv);
        } else if (p.units <= cus) {
            // one share a compute unit, in one round; where the units leave less than half of those for the shares of long ones, as many more
            // workgroups in case (32 sequences of 8 key-value heads, one of 30000 f16 positions beside 31 of 100: 37 us, 334 without)
            p.rounds_of = p.most_shares = cus;
            slots = p.units <= cus / 2 ? cus : p.units + cus;
        } else {
            // units alone are more than one round: shares small enough that the last round's end is a small part of all (64 sequences of
            // 8 key-value heads, up to 2000 f16 positions: 67, 67, 73, 87 us with one, two, four, eight times as many shares as compute units,
            // f32 137, 132, 134, 152)
            p.rounds_of = 2 * cus;
            p.most_shares = 0xffffffffu;
            slots = p.units + p.rounds_of;
        }
        if (p.joined) p.groups = (uint32_t)slots;
    }
    p.part_rows = (uint32_t)std::min<size_t>(rows, 16);
    p.stat_at = (slots * p.part_rows * c.cache->head_dim * 4 + 15) / 16 * 16;
    p.parts_at = p.stat_at + slots * p.part_rows * 8;
    p.row_weight_at = p.parts_at + (p.chunk_rows ? 0 : p.units * 8);
    p.score_at = (p.row_weight_at + (c.weights ? c.seqs->n_tokens * c.n_head * ROW_WEIGHT_BYTES : 0) + 15) / 16 * 16;
    // kept scores are a word a row and position where K and V are head_dim / 2 or head_dim words, read once anyway
    p.score_rows = c.weights && rows <= 16 ? (uint32_t)rows : 0;
    p.score_stride = (c.seqs->max_len + 31) / 32 * 32;
    size_t weight_blocks = 0;
    if (c.weights && p.score_rows == 0) {
        // the more rows, the less often K comes: 256 against 128 rows a workgroup, 2048 f16 tokens behind 6144: 240 and 312 us; up to 64
        // rows would leave most of its wavefronts without any (8 tokens of 4 heads behind 4096: 45 and 27 us)
        p.weight_rows = rows <= 64 ? 64 : c.cache->head_dim > 128 ? 128 : 256;
        weight_blocks = (rows + p.weight_rows - 1) / p.weight_rows;
        // a share loads its rows' q, and has no sums to join; of 64 rows four workgroups share a compute unit (16 tokens of each of 32 sequences of
        // 4096, f16: 69 us in four shares, 90 in two), of more two
        const float us = (half ? 0.0002f : 0.0010f) * (float)p.weight_rows * (float)c.cache->head_dim / 128.f;
        const BlockReads r = block_reads(c, p.weight_rows, seen, max_new);
        p.weight_splits = cut_blocks(r.blocks, r.first, r.most, p.weight_rows == 64 ? 2 * cus : cus, ChunkCost{us * 0.7f, us, 5.f, 0.f, 0.f}, (size_t)(r.most + 127.f) / 128).shares;
    }
    p.bytes = p.score_at + (p.units * p.score_rows + weight_blocks * heads) * p.score_stride * 4;
    const auto groups_of = [&](size_t n, size_t splits) { return n ? ((size_t)p.row_tiles * 16 + n - 1) / n * heads * splits : 0; };
    const size_t chunk_groups = groups_of(p.chunk_rows, p.splits), weight_groups = groups_of(p.weight_rows, p.weight_splits);
    for (const size_t n : {p.units, slots, (size_t)p.groups, chunk_groups, weight_groups, c.weights ? (c.seqs->max_len + 255) / 256 * heads : 0}) p.fits = p.fits && n <= MOST_GROUPS;
    p.chunk_groups = (uint32_t)chunk_groups;
    p.weight_groups = (uint32_t)weight_groups;
    return p;
}

inline size_t attn_part_seqs(const AttnCall &c, const AttnPlan &whole) {
    const size_t rows = std::min(c.seqs->max_new, c.seqs->n_tokens) * (c.n_head / c.cache->n_head_kv);
    const size_t score_rows = whole.score_rows ? rows : whole.weight_rows ? (rows + whole.weight_rows - 1) / whole.weight_rows : 0;
    return attn_seqs_at_once(c.seqs->n_seqs, whole.chunk_rows == 0 && whole.joined, score_rows * c.cache->n_head_kv * whole.score_stride * 4);
}

// `n` sequences of a call from the `first` on.
struct AttnPart {
    lnh_kv_seqs seqs;
    AttnCall call;
    AttnPart(const AttnCall &c, size_t first, size_t n) : seqs(*c.seqs), call(c) {
        seqs.n_seqs = n;
        seqs.device_tables += first * seqs.table_stride;
        seqs.device_lens += first;
        if (seqs.device_starts) {
            seqs.device_starts += first;
        } else {
            seqs.n_tokens = n;
            call.q += first * c.q_stride;
            call.out += first * c.out_stride;
        }
        call.seqs = &seqs;
    }
};

// Whether the call's launches hold it, and what workspace they take; cus: compute units of the GPU.
inline bool attn_fits(const AttnCall &c, uint32_t cus, size_t *workspace) {
    const AttnPlan whole = attn_plan(c, cus);
    *workspace = whole.bytes;
    if (!whole.fits) return false;
    const size_t n = c.seqs->n_seqs, at_once = attn_part_seqs(c, whole);
    if (at_once < n) *workspace = std::max(attn_plan(AttnPart(c, 0, at_once).call, cus).bytes, attn_plan(AttnPart(c, 0, (n - 1) % at_once + 1).call, cus).bytes);
    return true;
}

// What a call of chosen blocks keeps in the workspace: lists of the rows it takes at a time, scores, then what the attention over them keeps.
struct SelectPlan {
    size_t pages, list;      // blocks of the longest sequence, and of a row's list
    size_t rows;             // at a time
    size_t keys_at, tables_at, lens_at, attn_at, bytes;
    bool fits;
};
// The attention over `n` rows' lists from row `first` on: every row a sequence of its chosen blocks.
struct ChosenRows {
    lnh_kv_seqs seqs;
    AttnCall call;
    ChosenRows(const AttnSelectCall &c, const SelectPlan &p, size_t first, size_t n, const uint32_t *tables, const uint32_t *lens)
        : seqs{n, n, 1, p.list * c.attn.cache->kv_block, tables, p.list * c.attn.cache->n_head_kv, lens, nullptr}, call(c.attn) {
        call.seqs = &seqs;
        call.head_tables = p.list;
        call.q += first * c.attn.q_stride;
        call.out += first * c.attn.out_stride;
    }
};
constexpr size_t SELECT_WORKSPACE = (size_t)1 << 30;  // of scores and lists

inline SelectPlan select_plan(const AttnSelectCall &c, uint32_t cus) {
    SelectPlan p{};
    p.fits = true;
    const lnh_kv_seqs &s = *c.attn.seqs;
    const size_t heads = c.attn.cache->n_head_kv, tokens = s.n_tokens;
    if (s.n_seqs == 0 || tokens == 0 || s.max_new == 0) return p;
    p.pages = std::max<size_t>(1, (s.max_len + c.attn.cache->kv_block - 1) / c.attn.cache->kv_block);
    p.list = std::min(c.n_select, p.pages);
    const size_t keys = p.pages > c.n_select ? p.pages : 0, row = (heads * (keys + p.list) + 1) * 4;
    const size_t group = c.attn.n_head / heads, units = heads * ((group + 15) / 16);  // of a row, in the attention over it
    p.rows = std::max<size_t>(1, std::min({tokens, SELECT_WORKSPACE / row, MOST_GROUPS / 2 / units}));
    p.tables_at = (p.rows * heads * keys * 4 + 15) / 16 * 16;
    p.lens_at = p.tables_at + (p.rows * heads * p.list * 4 + 15) / 16 * 16;
    p.attn_at = p.lens_at + (p.rows * 4 + 15) / 16 * 16;
    size_t attn = 0;
    for (const size_t n : {p.rows, (tokens - 1) % p.rows + 1}) {
        size_t bytes = 0;
        p.fits = p.fits && attn_fits(ChosenRows(c, p, 0, n, nullptr, nullptr).call, cus, &bytes);
        attn = std::max(attn, bytes);
    }
    // (blocks times lanes, and a sequence's rows of q, are numbers of 32 bits)
    p.fits = p.fits && s.n_seqs * heads <= MOST_GROUPS && p.pages <= 0xffffffffu / 16 && std::min(s.max_new, tokens) * group <= 0xffffffffu;
    p.bytes = p.attn_at + attn;
    return p;
}

inline bool attn_select_fits(const AttnSelectCall &c, uint32_t cus, size_t *workspace) {
    const SelectPlan p = select_plan(c, cus);
    *workspace = p.bytes;
    return p.fits;
}

}  // namespace nh
#endif
