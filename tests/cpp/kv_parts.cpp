// Checks before launches of the rotated append, the read back, the 4-bit cache and chosen blocks (llama-rust_amd/csrc/attn_plan.h), with no device.
#include <cstdio>
#include <initializer_list>
#include <limits>

#include "../../llama-rust_amd/csrc/attn_plan.h"

static int failures = 0;
#define CHECK(x)                                                                  \
    do {                                                                          \
        if (!(x)) {                                                               \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);                   \
            failures++;                                                           \
        }                                                                         \
    } while (0)

alignas(16) static float buf[4096];
alignas(16) static uint32_t idx[64];
static const lnh_kv_cache good{LNH_TYPE_Q4_0, 2, 4, 64, 16, 10, buf, buf + 16, nullptr};
static const lnh_kv_seqs seqs{3, 3, 1, 100, idx, 7, idx + 16, nullptr};
static const lnh_rope rope{buf, 32, 128, 64, 0, nullptr};

static void four_bits() {
    const auto with = [](auto change) {
        lnh_kv_cache c = good;
        change(c);
        return nh::check_attn(&c, &seqs, 1, 8, buf, 2048, buf + 48, 2048, 0.1f, 0, 0, 0, 1.f).code;
    };
    CHECK(with([](lnh_kv_cache &) {}) == LNH_OK);
    for (const uint32_t d : {32u, 96u, 128u, 224u, 256u}) CHECK(with([&](lnh_kv_cache &c) { c.head_dim = d; }) == LNH_OK);
    for (const uint32_t d : {8u, 40u, 80u, 120u, 248u, 288u}) CHECK(with([&](lnh_kv_cache &c) { c.head_dim = d; }) == LNH_ERR_UNSUPPORTED);
    for (const uint32_t kind : {(uint32_t)LNH_TYPE_Q5_0, (uint32_t)LNH_TYPE_Q8_0, (uint32_t)LNH_TYPE_Q4_K, 77u})
        CHECK(with([&](lnh_kv_cache &c) { c.ggml_type = kind; }) == LNH_ERR_UNSUPPORTED);
    for (const uint32_t block : {1u, 7u, 20u}) CHECK(with([&](lnh_kv_cache &c) { c.kv_block = block, c.n_blocks = 200; }) == (block < 15 ? LNH_ERR_INVALID : LNH_OK));
    CHECK(with([](lnh_kv_cache &c) { c.device_k = buf + 1; }) == LNH_ERR_INVALID);
}

static void append() {
    struct Call {
        lnh_kv_cache cache = good;
        lnh_kv_seqs seqs = ::seqs;
        lnh_rope rope = ::rope;
        const lnh_rope *with = &rope;
        size_t layer = 1, heads = 8, qs = 512, os = 512, ks = 256, vs = 256;
        const float *q = buf, *out = buf + 1024, *k = buf + 2048, *v = buf + 2064;
    };
    const auto code = [](auto change) {
        Call c;
        change(c);
        return nh::check_kv_append(&c.cache, &c.seqs, c.layer, c.with, c.heads, c.q, c.qs, c.out, c.os, c.k, c.ks, c.v, c.vs).code;
    };
    CHECK(code([](Call &) {}) == LNH_OK);
    CHECK(code([](Call &c) { c.with = nullptr; }) == LNH_OK);
    CHECK(code([](Call &c) { c.heads = 0, c.q = c.out = nullptr; }) == LNH_OK);
    CHECK(code([](Call &c) { c.heads = 5; }) == LNH_OK);  // q and k need not go together here
    CHECK(code([](Call &c) { c.out = c.q; }) == LNH_OK);
    CHECK(code([](Call &c) { c.out = c.q, c.os = 516; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.heads = 65537, c.qs = c.os = (size_t)1 << 30; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.layer = 2; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.q = nullptr; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.out = nullptr; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.k = nullptr; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.v = c.v + 1; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.qs = 508; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.os = 514; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.ks = 252; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.vs = SIZE_MAX - 3; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.n_rot = 0, c.rope.device_angles = nullptr; }) == LNH_OK);
    CHECK(code([](Call &c) { c.rope.n_rot = 20; }) == LNH_OK);
    CHECK(code([](Call &c) { c.rope.n_rot = 63; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.n_rot = 66; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.device_angles = nullptr; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.device_angles = buf + 1; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.device_positions = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(idx) + 2); }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.angle_stride = 31; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.angle_stride = SIZE_MAX; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.n_positions = 0; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.rope.n_positions = ((size_t)1 << 31) + 1; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.seqs.n_seqs = c.seqs.n_tokens = 0, c.q = c.out = c.k = c.v = nullptr, c.rope.device_angles = nullptr; }) == LNH_OK);
    CHECK(nh::check_kv_append(nullptr, &seqs, 0, nullptr, 0, nullptr, 0, nullptr, 0, buf, 256, buf, 256).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_append(&good, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, buf, 256, buf, 256).code == LNH_ERR_INVALID);
}

static void angles() {
    const double inf = std::numeric_limits<double>::infinity(), nan = std::numeric_limits<double>::quiet_NaN();
    const auto code = [](uint32_t n_rot, double base, double scale, size_t n, const float *to, size_t stride, const float *div = nullptr) {
        return nh::check_rope_table(n_rot, base, scale, div, n, to, stride).code;
    };
    CHECK(code(64, 1e4, 1, 100, buf, 32) == LNH_OK);
    CHECK(code(64, 1e4, 0.25, 100, buf, 33, buf + 1) == LNH_OK);
    CHECK(code(64, 1e4, 1, 0, nullptr, 32) == LNH_OK);
    for (const double x : {0.0, -1.0, inf, nan}) CHECK(code(64, x, 1, 100, buf, 32) == LNH_ERR_INVALID && code(64, 1e4, x, 100, buf, 32) == LNH_ERR_INVALID);
    for (const uint32_t n : {0u, 1u, 63u}) CHECK(code(n, 1e4, 1, 100, buf, 64) == LNH_ERR_INVALID);
    CHECK(code(64, 1e4, 1, 100, nullptr, 32) == LNH_ERR_INVALID);
    CHECK(code(64, 1e4, 1, 100, buf + 1, 32) == LNH_ERR_INVALID);
    CHECK(code(64, 1e4, 1, 100, buf, 31) == LNH_ERR_INVALID);
    CHECK(code(64, 1e4, 1, SIZE_MAX, buf, 32) == LNH_ERR_INVALID);
}

static void chosen_blocks() {
    struct Call {
        lnh_kv_cache cache = good;
        lnh_kv_seqs seqs = ::seqs;
        size_t layer = 1, heads = 8, most = 4, first = 1, recent = 2, qs = 512, os = 512;
        const void *bounds = buf + 512;
        const float *q = buf, *out = buf + 1024;
        float scale = 0.125f;
        const uint32_t *chosen = idx;
    };
    const auto code = [](auto change) {
        Call c;
        change(c);
        return nh::check_attn_select(&c.cache, &c.seqs, c.layer, c.heads, c.bounds, c.most, c.first, c.recent, c.q, c.qs, c.out, c.os, c.scale, c.chosen).code;
    };
    CHECK(code([](Call &) {}) == LNH_OK);
    CHECK(code([](Call &c) { c.chosen = nullptr; }) == LNH_OK);
    CHECK(code([](Call &c) { c.first = 2; }) == LNH_OK);
    CHECK(code([](Call &c) { c.first = 3; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.first = SIZE_MAX; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.recent = SIZE_MAX; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.recent = 0; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.most = SIZE_MAX; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.most = nh::ATTN_MAX_POSITIONS / 16; }) == LNH_OK);
    CHECK(code([](Call &c) { c.bounds = nullptr; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.bounds = buf + 1; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.chosen = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(idx) + 1); }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.heads = 6; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.layer = 2; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.scale = -1.f; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.out = c.q; }) == LNH_ERR_INVALID);
    CHECK(code([](Call &c) { c.seqs.n_seqs = c.seqs.n_tokens = 0, c.bounds = c.q = c.out = nullptr; }) == LNH_OK);
    CHECK(nh::check_kv_bounds(&good, &seqs, 0, buf).code == LNH_OK);
    CHECK(nh::check_kv_bounds(&good, &seqs, 2, buf).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_bounds(&good, &seqs, 0, nullptr).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_bounds(&good, &seqs, 0, buf + 2).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_bounds(nullptr, &seqs, 0, buf).code == LNH_ERR_INVALID);
    CHECK(nh::check_kv_bounds(&good, nullptr, 0, buf).code == LNH_ERR_INVALID);
}

int main() {
    chosen_blocks();
    four_bits();
    append();
    angles();
    if (failures) return 1;
    std::printf("OK\n");
    return 0;
}
