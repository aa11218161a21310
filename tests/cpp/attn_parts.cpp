// Checks of what the paged-cache operators do before and around a launch (llama-rust_amd/csrc/attn_plan.h), for the host
// compiler alone.  Prints "OK" and returns 0, or says what failed and returns 1.
#include <cstdio>
#include <cstring>
#include <limits>
#include <vector>

#include "../../llama-rust_amd/csrc/attn_plan.h"

static int failures = 0;
#define CHECK(cond)                                                \
    do {                                                           \
        if (!(cond)) {                                             \
            if (failures < 20) std::printf("%s:%d: %s\n", __FILE__, __LINE__, #cond); \
            failures++;                                            \
        }                                                          \
    } while (0)

static void division() {
    const uint32_t divisors[] = {1, 2, 3, 5, 7, 16, 20, 24, 31, 64, 100, 127, 1000, 65535, 65536, 65537, 0x7fffffffu, 0x80000000u};
    for (const uint32_t d : divisors) {
        const nh::FastDiv f = nh::fast_div(d);
        for (uint32_t n = 0; n < 3000; n++) CHECK(nh::div_by(f, n) == n / d);
        for (uint64_t m = 1; m < 40; m++)
            for (int64_t o = -2; o <= 2; o++) {
                const int64_t n = (int64_t)(m * d) + o;
                if (n >= 0 && n < ((int64_t)1 << 31)) CHECK(nh::div_by(f, (uint32_t)n) == (uint32_t)n / d);
            }
        CHECK(nh::div_by(f, 0x7fffffffu) == 0x7fffffffu / d);
    }
}

// Every position that a row sees lies in exactly one of the tiles, those come in shares without gap or overlap, and [lo, hi) with the
// first tokens is no smaller than what is seen.
static void tiles() {
    for (const uint32_t tp : {16u, 32u, 64u})
        for (const uint32_t window : {0u, 1u, 5u, 31u, 32u, 33u, 100u, 5000u})
            for (const uint32_t sinks : {0u, 1u, 4u, 16u, 40u, 200u, 5000u}) {
                if (window == 0 && sinks != 0) continue;
                for (const int32_t first : {-20, -1, 0, 1, 15, 31, 32, 63, 64, 130, 700})
                    for (const int32_t more : {0, 1, 3, 15, 40}) {
                        const int32_t last = first + more;
                        const nh::AttnTiles t = nh::attn_tiles(first, last, window, sinks, tp);
                        std::vector<int> seen((size_t)(last < 0 ? 0 : last) + 2 * tp, 0);
                        for (const uint32_t n : {1u, 2u, 3u, 7u}) {
                            uint32_t at = 0;
                            for (uint32_t s = 0; s < n; s++) {
                                CHECK(nh::attn_share(t.count, s, n) == at);
                                at = nh::attn_share(t.count, s + 1, n);
                            }
                            CHECK(at == t.count);
                        }
                        for (uint32_t j = 0; j < t.count; j++) {
                            const uint32_t tile = nh::attn_tile(t, j);
                            for (uint32_t i = 0; i < tp; i++) {
                                CHECK(tile * tp + i < seen.size());
                                if (tile * tp + i < seen.size()) seen[tile * tp + i]++;
                            }
                        }
                        for (size_t p = 0; p < seen.size(); p++) {
                            CHECK(seen[p] <= 1);
                            bool any = false;
                            for (int32_t r = first; r <= last; r++) any = any || nh::attn_sees(r, (uint32_t)p, window, sinks);
                            if (any) {
                                CHECK(seen[p] == 1);
                                CHECK(p < t.hi && (p >= t.lo || p < sinks));
                            }
                        }
                    }
            }
}

static void sight() {
    CHECK(!nh::attn_sees(-1, 0, 0, 0));
    CHECK(nh::attn_sees(0, 0, 0, 0));
    CHECK(!nh::attn_sees(3, 4, 0, 0));
    CHECK(nh::attn_sees(9, 0, 10, 0) && !nh::attn_sees(10, 0, 10, 0) && nh::attn_sees(10, 0, 10, 1));
    CHECK(nh::attn_sees(7, 7, 1, 0) && !nh::attn_sees(7, 6, 1, 0));
}

// Tables that name blocks the cache does not have, positions behind the table: nothing is followed.
static void bad_pages() {
    const uint32_t table[4] = {2, 0xffffffffu, 3, 0};
    const nh::KvPlace p{table, 4, 3, 2 * 5 * 20, nh::fast_div(20)};  // 3 blocks, 2 layers, 5 heads, 20 positions
    const uint32_t head_rows = (1 * 5 + 2) * 20;
    CHECK(nh::kv_row(p, table, head_rows, 0) == 2 * 200 + 140);
    CHECK(nh::kv_row(p, table, head_rows, 19) == 2 * 200 + 140 + 19);
    for (uint32_t t = 20; t < 60; t++) CHECK(nh::kv_row(p, table, head_rows, t) == nh::ATTN_NOWHERE);
    CHECK(nh::kv_row(p, table, head_rows, 79) == 140 + 19);
    for (const uint32_t t : {80u, 81u, 1000u, 0x7fffffffu}) CHECK(nh::kv_row(p, table, head_rows, t) == nh::ATTN_NOWHERE);
}

// Row starts and lengths that are not what they should be stay within the arrays.
static void rows() {
    const uint32_t lens[5] = {10, 3, 0, 99, 7};
    const uint32_t starts[6] = {0, 2, 7, 5, 30, 31};  // descending once, behind the last token once
    nh::SeqRows s = nh::seq_rows(starts, lens, 0, 20, 8, 50);
    CHECK(s.row0 == 0 && s.n == 2 && s.first_pos == 8 && s.len == 10);
    s = nh::seq_rows(starts, lens, 1, 20, 8, 50);
    CHECK(s.n == 5 && s.first_pos == -2);
    s = nh::seq_rows(starts, lens, 2, 20, 8, 50);
    CHECK(s.n == 0);
    s = nh::seq_rows(starts, lens, 3, 20, 8, 50);
    CHECK(s.row0 == 5 && s.n == 8 && s.len == 50 && s.first_pos == 50 - 15);
    s = nh::seq_rows(starts, lens, 4, 20, 8, 50);
    CHECK(s.n == 0 && s.row0 <= 20);
    s = nh::seq_rows(nullptr, lens, 2, 5, 1, 50);
    CHECK(s.row0 == 2 && s.n == 1 && s.first_pos == -1);
}

static void refusals() {
    alignas(16) static float buf[64];
    alignas(16) static uint32_t idx[64];
    const lnh_kv_cache good{LNH_TYPE_F16, 2, 4, 64, 16, 10, buf, buf + 16, buf + 32};
    const lnh_kv_seqs seqs{3, 3, 1, 100, idx, 7, idx + 16, nullptr};
    const auto attn = [&](const lnh_kv_cache &c, const lnh_kv_seqs &s) {
        return nh::check_attn(&c, &s, 1, 8, buf, 512, buf + 48, 512, 0.1f, 0, 0, 1, 1.f).code;
    };
    const auto cache_with = [&](auto change) {
        lnh_kv_cache c = good;
        change(c);
        return attn(c, seqs);
    };
    const auto seqs_with = [&](auto change) {
        lnh_kv_seqs s = seqs;
        change(s);
        return attn(good, s);
    };
    CHECK(attn(good, seqs) == LNH_OK);
    CHECK(cache_with([](lnh_kv_cache &c) { c.ggml_type = LNH_TYPE_Q8_0; }) == LNH_ERR_UNSUPPORTED);
    CHECK(cache_with([](lnh_kv_cache &c) { c.head_dim = 60; }) == LNH_ERR_UNSUPPORTED);
    CHECK(cache_with([](lnh_kv_cache &c) { c.head_dim = 264; }) == LNH_ERR_UNSUPPORTED);
    CHECK(cache_with([](lnh_kv_cache &c) { c.head_dim = 0; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.n_blocks = 0; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.kv_block = 0; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.n_blocks = 0xffffffffu; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.n_layer = c.kv_block = c.n_blocks = 0xffffffffu; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.n_blocks = (1u << 24); }) == LNH_OK);  // 2^31 rows
    CHECK(cache_with([](lnh_kv_cache &c) { c.n_blocks = (1u << 24) + 1; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.device_k = nullptr; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.device_v = nullptr; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.device_w = nullptr; }) == LNH_ERR_INVALID);
    CHECK(cache_with([](lnh_kv_cache &c) { c.device_v = reinterpret_cast<char *>(c.device_v) + 2; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.max_len = 112; }) == LNH_OK);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.max_len = 113; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.device_lens = nullptr; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.device_tables = nullptr; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.n_tokens = 4; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.n_tokens = 4, s.device_starts = idx; }) == LNH_OK);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.device_starts = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(idx) + 1); }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.table_stride = SIZE_MAX; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.max_len = SIZE_MAX; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.max_new = (size_t)1 << 31; }) == LNH_ERR_INVALID);
    CHECK(seqs_with([](lnh_kv_seqs &s) { s.n_seqs = 0, s.n_tokens = 0, s.device_tables = nullptr; }) == LNH_OK);
    const auto call = [&](size_t layer, size_t heads, const float *q, size_t qs, float *out, size_t os, float scale, size_t window, size_t sinks,
                          float decay) { return nh::check_attn(&good, &seqs, layer, heads, q, qs, out, os, scale, window, sinks, 1, decay).code; };
    CHECK(call(0, 4, buf, 256, buf + 48, 260, 1.f, 5, 4, 0.f) == LNH_OK);
    CHECK(call(2, 4, buf, 256, buf + 48, 256, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 6, buf, 512, buf + 48, 512, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 0, buf, 512, buf + 48, 512, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf + 1, 256, buf + 48, 256, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf, 255, buf + 48, 256, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf, 252, buf + 48, 256, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf, 256, buf, 256, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, nullptr, 256, buf, 256, 1.f, 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf, 256, buf + 48, 256, std::numeric_limits<float>::quiet_NaN(), 0, 0, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf, 256, buf + 48, 256, 1.f, 0, 0, std::numeric_limits<float>::infinity()) == LNH_ERR_INVALID);
    for (const float scale : {0.f, -0.f, -0.125f, std::numeric_limits<float>::max()}) CHECK(call(0, 4, buf, 256, buf + 48, 256, scale, 0, 0, 1.f) == LNH_ERR_INVALID);
    for (const float scale : {1e-30f, 0x1p127f}) CHECK(call(0, 4, buf, 256, buf + 48, 256, scale, 0, 0, 1.f) == LNH_OK);
    CHECK(call(0, 4, buf, 256, buf + 48, 256, 1.f, 0, 4, 1.f) == LNH_ERR_INVALID);
    CHECK(call(0, 4, buf, 256, buf + 48, 256, 1.f, (size_t)1 << 31, 4, 1.f) == LNH_ERR_INVALID);
    CHECK(nh::check_kv_store(&good, &seqs, 0, buf, 256, buf, 256).code == LNH_OK);
    CHECK(nh::check_kv_store(&good, &seqs, 2, buf, 256, buf, 256).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_store(&good, &seqs, 0, buf, 256, nullptr, 256).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_store(&good, &seqs, 0, buf, 128, buf, 256).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_store(nullptr, &seqs, 0, buf, 256, buf, 256).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_store(&good, nullptr, 0, buf, 256, buf, 256).code == LNH_ERR_INVALID);
    const auto evict = [&](size_t l0, size_t nl, size_t keep, size_t first, size_t recent, const uint32_t *dst, size_t stride, const uint32_t *out) {
        return nh::check_kv_evict(&good, &seqs, l0, nl, keep, first, recent, dst, stride, out).code;
    };
    CHECK(evict(0, 2, 50, 4, 46, nullptr, 0, idx) == LNH_OK);
    CHECK(evict(0, 2, 0, 0, 0, nullptr, 0, idx) == LNH_OK);
    CHECK(evict(0, 2, 50, 4, 47, nullptr, 0, idx) == LNH_ERR_INVALID);
    CHECK(evict(0, 2, 50, 51, 0, nullptr, 0, idx) == LNH_ERR_INVALID);
    CHECK(evict(0, 2, 50, SIZE_MAX, SIZE_MAX, nullptr, 0, idx) == LNH_ERR_INVALID);
    CHECK(evict(1, 2, 50, 4, 4, nullptr, 0, idx) == LNH_ERR_INVALID);
    CHECK(evict(0, 0, 50, 4, 4, nullptr, 0, idx) == LNH_ERR_INVALID);
    CHECK(evict(0, SIZE_MAX, 50, 4, 4, nullptr, 0, idx) == LNH_ERR_INVALID);
    CHECK(evict(0, 1, 50, 4, 4, nullptr, 0, nullptr) == LNH_ERR_INVALID);
    CHECK(evict(0, 1, 50, 4, 4, idx + 32, 3, idx) == LNH_ERR_INVALID);
    CHECK(evict(0, 1, 50, 4, 4, idx + 32, 4, idx) == LNH_OK);
    CHECK(evict(0, 1, 500, 4, 4, idx + 32, 7, idx) == LNH_OK);  // never more than max_len
}

// The tokens that see a position, by the position.
static void seen_by() {
    for (const uint32_t n : {0u, 1u, 7u, 40u})
        for (const int32_t first : {-41, -5, 0, 3, 100})
            for (const uint32_t window : {0u, 1u, 6u, 30u, 0x7fffefffu})
                for (const uint32_t sinks : {0u, 2u, 50u, 0x7fffefffu}) {
                    if (window == 0 && sinks != 0) continue;
                    const nh::SeqRows s{0, n, first, first + (int32_t)n > 0 ? (uint32_t)(first + (int32_t)n) : 0u};
                    for (uint32_t t = 0; t < 160; t++) {
                        const nh::SeenBy by = nh::attn_seen_by(s, t, window, sinks);
                        CHECK(by.from <= n && by.to <= n);
                        for (uint32_t i = 0; i < n; i++) CHECK(nh::attn_sees(first + (int32_t)i, t, window, sinks) == (by.from <= i && i < by.to));
                    }
                }
}

// What the many-row kernels load of a row lies within it, and of what they multiply, everything else is cleared instead.
static void pieces() {
    for (const bool half : {false, true})
        for (uint32_t d = 8; d <= nh::ATTN_MAX_HEAD_DIM; d += 8) {
            const uint32_t dp = nh::attn_many_dims(half, d), piece = nh::attn_piece(half), pitch = nh::attn_pitch(half, dp);
            CHECK(dp >= d && dp % 32 == 0 && pitch * piece >= dp);
            for (uint32_t c = 0; c < pitch; c++) {
                const bool there = (c + 1) * piece <= d;
                CHECK(nh::attn_brings(half, dp, d, c) == there);
                if (!there && c < dp / piece) CHECK(dp != d);  // the kernels clear the places where dp != d
            }
        }
}

// Sequences go in parts of nearly one size: few enough for few rows, with no more workspace for weights than there is to be, one at least.
static void parts() {
    for (const size_t n : {0, 1, 2, 64, 255, 256, 257, 300, 512, 513, 1000, 8192, 0x3fffff})
        for (const bool few : {false, true})
            for (const size_t bytes : {(size_t)0, (size_t)1, (size_t)1 << 20, ((size_t)1 << 24) + 1, (size_t)1 << 30, ((size_t)1 << 30) + 1, (size_t)1 << 50}) {
                const size_t at_once = nh::attn_seqs_at_once(n, few, bytes);
                CHECK(at_once <= n && (at_once >= 1 || n == 0));
                if (few) CHECK(at_once <= 256);
                if (at_once > 1) CHECK(at_once * bytes <= (size_t)1 << 30);
                if (!few && n * bytes <= (size_t)1 << 30) CHECK(at_once == n);
                if (few && n <= 256 && n * bytes <= (size_t)1 << 30) CHECK(at_once == n);
                if (at_once) CHECK(n - (n - 1) / at_once * at_once + (n + at_once - 1) / at_once > at_once);  // the last part is short by less than there are parts
            }
}

int main() {
    parts();
    pieces();
    seen_by();
    division();
    tiles();
    sight();
    bad_pages();
    rows();
    refusals();
    if (failures) return 1;
    std::printf("OK\n");
    return 0;
}
