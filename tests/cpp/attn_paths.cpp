// Which kernels a call of attention over the paged cache takes (llama-rust_amd/csrc/attn_launch_plan.h), with no device.  With no arguments: checks.
// With a line of numbers a call on standard input - ggml type, n_head, n_head_kv, head_dim, kv_block, n_seqs, n_tokens, max_new, max_len, window, sinks,
// weights, n_select (0: all blocks) -: the path of each.
#include <cstdio>
#include <cstring>

#include "../../llama-rust_amd/csrc/attn_launch_plan.h"

static int failures = 0;
#define CHECK(x)                                                                  \
    do {                                                                          \
        if (!(x)) {                                                               \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);                   \
            failures++;                                                           \
        }                                                                         \
    } while (0)

constexpr uint32_t CUS = 256;
static uint32_t starts[1];

struct Given {
    unsigned type = LNH_TYPE_F16, heads = 32, heads_kv = 8, dim = 128, block = 16;
    size_t seqs = 1, tokens = 1, max_new = 1, max_len = 100, window = 0, sinks = 0;
    int weights = 0;
    size_t select = 0;
    lnh_kv_cache cache() const { return {type, 1, heads_kv, dim, block, 1, nullptr, nullptr, nullptr}; }
    lnh_kv_seqs rows() const { return {seqs, tokens, max_new, max_len, nullptr, (max_len + block - 1) / block, nullptr, tokens == seqs ? nullptr : starts}; }
    nh::AttnCall call(const lnh_kv_cache &c, const lnh_kv_seqs &s) const { return {&c, &s, 0, heads, nullptr, nullptr, 0, 0, 1.f, window, sinks, weights != 0, 1.f, 0}; }
};

static bool fits(const Given &g, size_t *bytes) {
    const lnh_kv_cache c = g.cache();
    const lnh_kv_seqs s = g.rows();
    const nh::AttnCall call = g.call(c, s);
    return g.select ? nh::attn_select_fits({call, nullptr, g.select, 1, 1, nullptr}, CUS, bytes) : nh::attn_fits(call, CUS, bytes);
}

static void print(const nh::AttnCall &call) {
    const nh::AttnPlan whole = nh::attn_plan(call, CUS);
    const size_t n = call.seqs->n_seqs, at_once = nh::attn_part_seqs(call, whole);
    const nh::AttnPlan p = at_once < n ? nh::attn_plan(nh::AttnPart(call, 0, at_once).call, CUS) : whole;
    std::printf("%s", p.chunk_rows ? "many" : p.joined ? "shares" : "whole");
    if (p.chunk_rows) std::printf(" rows=%u splits=%u", p.chunk_rows, p.splits);
    if (!p.chunk_rows && !p.joined) std::printf(" waves=%u", 1u << p.unit_waves);
    std::printf(" eight=%d parts=%zu\n", p.few_rows ? 1 : 0, (n + at_once - 1) / at_once);
}

static void sizes() {
    size_t bytes = 0;
    Given g;
    // lists of 4096 tiles for 2^19 units: whole units, whose tiles nobody counts together
    g = Given{};
    g.type = LNH_TYPE_F32, g.block = 256, g.tokens = g.max_new = 65536, g.max_len = 256 * 256, g.select = 256;
    CHECK(fits(g, &bytes) && bytes < (size_t)8 << 30);
    // a list of nearly 2^31 positions, rows for a workgroup a compute unit and more
    for (const size_t rows : {1, 31, 32, 33, 40, 1000}) {
        g = Given{};
        g.block = 1 << 16, g.tokens = g.max_new = rows, g.seqs = 1, g.max_len = ((size_t)1 << 31) - (1 << 17), g.select = ((size_t)1 << 15) - 3;
        CHECK(fits(g, &bytes));
        g.type = LNH_TYPE_F32;
        CHECK(fits(g, &bytes));
    }
    // all positions: as many workgroups as a launch has and no more, shares beyond what they count
    g = Given{};
    g.seqs = g.tokens = 400000, g.max_len = 500;
    g.heads = g.heads_kv = 10;
    CHECK(fits(g, &bytes));
    g.max_len = ((size_t)1 << 31) - (1 << 17);
    g.seqs = g.tokens = 32;
    CHECK(!fits(g, &bytes));
    g.seqs = g.tokens = (size_t)1 << 24;  // workgroups
    g.max_len = 500;
    CHECK(!fits(g, &bytes));
}

int main(int argc, char **argv) {
    if (argc > 1 && !std::strcmp(argv[1], "-")) {
        Given g;
        while (std::scanf("%u %u %u %u %u %zu %zu %zu %zu %zu %zu %d %zu", &g.type, &g.heads, &g.heads_kv, &g.dim, &g.block, &g.seqs, &g.tokens, &g.max_new, &g.max_len,
                          &g.window, &g.sinks, &g.weights, &g.select) == 13) {
            const lnh_kv_cache c = g.cache();
            const lnh_kv_seqs s = g.rows();
            const nh::AttnCall call = g.call(c, s);
            if (g.select) {
                const nh::AttnSelectCall chosen{call, nullptr, g.select, 1, 1, nullptr};
                const nh::SelectPlan p = nh::select_plan(chosen, CUS);
                print(nh::ChosenRows(chosen, p, 0, p.rows, nullptr, nullptr).call);
            } else {
                print(call);
            }
        }
        return 0;
    }
    sizes();
    if (failures) return 1;
    std::printf("OK\n");
    return 0;
}
