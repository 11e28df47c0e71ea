// The entry points of a step's index, rotary axes, page bounds and picked pages on the
// CPU: every refusal, with its text, on a context made by hand (a call that passes
// every check then fails on the device).
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "sage_cache.hpp"
#include "sage_internal.hpp"

static int failed = 0;
#define CHECK(x)                                                    \
    do {                                                            \
        if (!(x)) {                                                 \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);     \
            failed++;                                               \
        }                                                           \
    } while (0)

static bool refused(sage_status st, const char* text, sage_status want = SAGE_ERR_INVALID) {
    const bool ok = st == want && std::strstr(sage_last_error(), text);
    if (!ok) std::printf("  got %d: %s (wanted: %s)\n", st, sage_last_error(), text);
    return ok;
}
// Every check passed: the device of this context is not there.
static bool passed(sage_status st) {
    const bool ok = st == SAGE_ERR_DEVICE || (st == SAGE_ERR_INVALID && std::strstr(sage_last_error(), "device -2"));
    if (!ok) std::printf("  got %d: %s\n", st, sage_last_error());
    return ok;
}

alignas(256) static char mem[4096];
static int32_t* const n = reinterpret_cast<int32_t*>(mem);
static uint8_t* const u = reinterpret_cast<uint8_t*>(mem);
// Two sequences of four rows at most, 4 query heads over 2 KV heads, five pages of 16.
static const sage_cache_shape H{2, 4, 3, 4, 2, 5, 16, 3};
static const sage_cache_index INDEX{n, 3, n, 2, n, 6};

static void axes() {
    sage_attention ctx{nullptr, -2, 128, sage_config_for_head_dim(128)};
    const sage_shape shape{1, 4, 8, 0};
    const sage_strides st{4096, 512, 128};
    const sage_tensor x{mem, 4096, st, SAGE_BF16};
    const sage_tensor_mut o{mem, 4096, st, SAGE_BF16};
    const sage_rotary_axes r{reinterpret_cast<float*>(mem), 1024, {16, 24, 24, 0}, 3, SAGE_ROTARY_AXES_HALF, 0, n, 24, 8};
    CHECK(passed(sage_rotary_axes_apply(&ctx, &shape, &r, &x, &o, 0)));
    CHECK(refused(sage_rotary_axes_apply(&ctx, &shape, nullptr, &x, &o, 0), "null argument"));
    auto bad = [&](auto change, const char* text) {
        sage_rotary_axes q = r;
        change(q);
        CHECK(refused(sage_rotary_axes_apply(&ctx, &shape, &q, &x, &o, 0), text));
        const sage_tensor kv{mem, 8 * 256, {0, 256, 128}, SAGE_BF16};
        const sage_cache_shape h{1, 8, 8, 2, 2, 1, 16, 1};
        const sage_cache cache{u, u, u, u, 2 * 16 * 64, 2 * 16 * 4};
        CHECK(refused(sage_cache_append_axes(&ctx, &h, &cache, &INDEX, &kv, &kv, &q, nullptr, nullptr), text));
    };
    using R = sage_rotary_axes&;
    bad([](R q) { q.axes = 0; }, "0 axes (1 to 4 are supported)");
    bad([](R q) { q.axes = 5; }, "5 axes (1 to 4 are supported)");
    bad([](R q) { q.sections[1] = 0; }, "axis 1 of 0 pairs");
    bad([](R q) { q.sections[1] = 25; }, "130 rotated channels of head dim 128");
    bad([](R q) { q.sections[0] = ~0ull; }, "axis 0 of");
    bad([](R q) { q.layout = 3; }, "unknown layout 3");
    bad([](R q) { q.layout = SAGE_ROTARY_AXES_AXIS_HALF, q.dealt = 1; }, "need its pairs in one run");
    bad([](R q) { q.table_len = 127; }, "rotary table: buffer holds 127 elements, needs 128");
    bad([](R q) { q.table = nullptr; }, "rotary table");
    bad([](R q) { q.table++; }, "16-byte aligned");
    bad([](R q) { q.table_len = 1ull << 40; }, "does not fit in i32");
    bad([](R q) { q.positions = nullptr; }, "rotary positions: buffer holds 0");
    bad([](R q) { q.positions_len = 23; }, "rotary positions: buffer holds 23 elements, needs 24");
    bad([](R q) { q.positions_stride = 7; }, "7 entries from axis to axis, 8 rows");
    bad([](R q) { q.positions_stride = ~0ull; }, "from axis to axis");
    bad([](R q) { q.positions = (int*)(mem + 2); }, "4-byte aligned");
    const sage_tensor kv{mem, 4 * 256, {0, 256, 128}, SAGE_BF16};
    const sage_cache cache{u, u, u, u, 5 * 2 * 16 * 64, 5 * 2 * 16 * 4};
    CHECK(passed(sage_cache_append_axes(&ctx, &H, &cache, &INDEX, &kv, &kv, &r, nullptr, nullptr)));
    CHECK(refused(sage_cache_append_axes(&ctx, &H, &cache, &INDEX, &kv, &kv, nullptr, nullptr, nullptr), "null argument"));

    // The table, against its definition.
    std::vector<float> t(7 * 20), plain(7 * 20);
    const uint64_t sec[3] = {4, 3, 3};
    CHECK(sage_rotary_axes_table(sec, 3, 1, 0, 7, 1e4, nullptr, t.data(), t.size()) == SAGE_OK);
    CHECK(sage_rotary_table(20, 7, 1e4, nullptr, plain.data(), plain.size()) == SAGE_OK && t == plain);
    CHECK(sage_rotary_axes_table(sec, 3, 0, 1, 7, 1e4, nullptr, t.data(), t.size()) == SAGE_OK);
    for (int p = 0; p < 7; p++)
        for (int i = 0; i < 10; i++) {
            const int a = i < 4 ? 0 : i < 7 ? 1 : 2, j = i - (a == 0 ? 0 : a == 1 ? 4 : 7);
            const double angle = p * std::pow(1e4, -(double)j / (double)sec[a]);
            CHECK(t[(p * 10 + i) * 2] == (float)std::cos(angle) && t[(p * 10 + i) * 2 + 1] == (float)std::sin(angle));
        }
    float* f = t.data();
    CHECK(refused(sage_rotary_axes_table(sec, 3, 0, 0, 7, 1e4, nullptr, f, 139), "buffer holds 139 elements, needs 140"));
    CHECK(refused(sage_rotary_axes_table(sec, 5, 0, 0, 7, 1e4, nullptr, f, 140), "5 axes"));
    CHECK(refused(sage_rotary_axes_table(nullptr, 3, 0, 0, 7, 1e4, nullptr, f, 140), "null argument"));
    CHECK(refused(sage_rotary_axes_table(sec, 3, 0, 0, 7, 1.0, nullptr, f, 140), "base"));
    const uint64_t one[2] = {1, 3}, none[2] = {0, 3};
    const sage_rotary_scaling ntk{SAGE_ROTARY_NTK, 4, 0, 0, 0, 0};
    CHECK(sage_rotary_axes_table(one, 2, 0, 0, 7, 1e4, &ntk, f, 140) == SAGE_OK);
    CHECK(refused(sage_rotary_axes_table(one, 2, 0, 1, 7, 1e4, &ntk, f, 140), "NTK"));
    CHECK(refused(sage_rotary_axes_table(none, 2, 0, 1, 7, 1e4, nullptr, f, 140), "axis 0 of 0 pairs"));
}

static void tables() {
    sage_attention ctx{nullptr, -2, 128, sage_config_for_head_dim(128)};
    int64_t* slots = reinterpret_cast<int64_t*>(mem);
    const sage_cache_requests requests{n, 2, n, 2};
    const sage_cache_free ring{n, 5, n, 2};
    const sage_cache_step step{n, 3, n, 2, n, 6, n, 4, slots, 4, n, 4, n, 4, n, 4};
    CHECK(passed(sage_cache_tables(&ctx, &H, &requests, &ring, &step)));
    CHECK(refused(sage_cache_tables(nullptr, &H, &requests, &ring, &step), "null argument"));
    CHECK(refused(sage_cache_tables(&ctx, &H, &requests, &ring, nullptr), "null argument"));
    auto bad = [&](auto change, const char* text) {
        sage_cache_shape h = H;
        sage_cache_requests q = requests;
        sage_cache_free f = ring;
        sage_cache_step s = step;
        change(h, q, f, s);
        CHECK(text ? refused(sage_cache_tables(&ctx, &h, &q, &f, &s), text) : passed(sage_cache_tables(&ctx, &h, &q, &f, &s)));
    };
    using A = sage_cache_shape&;
    using Q = sage_cache_requests&;
    using F = sage_cache_free&;
    using S = sage_cache_step&;
    bad([](A h, Q, F, S) { h.page_tokens = 17; }, "pages of 17 tokens");
    bad([](A h, Q, F, S) { h.batch = 65536; }, "exceed the launch grid");
    bad([](A, Q q, F, S) { q.news_len = 1; }, "request rows: buffer holds 1 elements, needs 2");
    bad([](A, Q q, F, S) { q.past = nullptr; }, "request lengths: buffer holds 0");
    bad([](A, Q, F f, S) { f.pages_len = 0; }, "a ring of no places");
    bad([](A, Q, F f, S) { f.pages_len = 1ull << 31; }, "does not fit in i32");
    bad([](A, Q, F f, S) { f.pages = nullptr; }, "free pages: buffer holds 0");
    bad([](A, Q, F f, S) { f.state_len = 1; }, "free pages' state: buffer holds 1 elements, needs 2");
    bad([](A, Q, F, S s) { s.starts_len = 2; }, "cache starts: buffer holds 2 elements, needs 3");
    bad([](A, Q, F, S s) { s.lengths_len = 1; }, "cache lengths");
    bad([](A, Q, F, S s) { s.page_table_len = 5; }, "cache page table: buffer holds 5 elements, needs 6");
    bad([](A, Q, F, S s) { s.positions_len = 3; }, "step positions: buffer holds 3 elements, needs 4");
    bad([](A, Q, F, S s) { s.positions++; }, "step positions must start at a 16-byte aligned");
    bad([](A, Q, F, S s) { s.slots_len = 3; }, "step slots: buffer holds 3 elements, needs 4");
    bad([](A, Q, F, S s) { s.slots++; }, "step slots must start at a 16-byte aligned");
    bad([](A, Q, F, S s) { s.sequences_len = 3; }, "step sequences: buffer holds 3 elements, needs 4");
    bad([](A, Q, F, S s) { s.state_len = 3; }, "step state: buffer holds 3 elements, needs 4");
    bad([](A, Q, F, S s) { s.scratch_len = 3; }, "step scratch: buffer holds 3 elements, needs 4");
    bad([](A, Q, F, S s) { s.positions = nullptr, s.sequences = nullptr, s.slots = nullptr; }, nullptr);
    bad([](A h, Q q, F, S s) { h.batch = 0, q = {}, s.scratch = nullptr; }, nullptr);
}

struct Workspace {  // as sage_pick_workspace_new makes it, which needs the device
    sage_cache_shape shape;
    uint64_t head_dim, top, bytes;
    int device, window;
    sage::PickedPlan plan;
    void* buf;
};

static void picks() {
    sage_attention ctx{nullptr, -2, 128, sage_config_for_head_dim(128)};
    const sage_cache cache{u, u, u, u, 5 * 2 * 16 * 64, 5 * 2 * 16 * 4};
    const sage_cache_bounds bounds{reinterpret_cast<int8_t*>(mem), u, 5 * 2 * 256, 5 * 2};
    const sage_tensor q{mem, 4 * 512, {0, 512, 128}, SAGE_F16};
    const sage_tensor_mut o{mem, 4 * 512, {0, 512, 128}, SAGE_F16};
    const Workspace made{H, 128, 2, 0, -2, 4, {}, nullptr};
    auto update = [&](const sage_cache_shape& h, const sage_cache_bounds& b, const sage_cache_index& i) {
        return sage_cache_bounds_update(&ctx, &h, &cache, &i, &b);
    };
    auto pick = [&](Workspace w, const sage_cache_bounds& b, const sage_cache_index& i, const sage_pick_options& opts,
                    uint64_t len = 16) {
        return sage_cache_pick(&ctx, reinterpret_cast<sage_pick_workspace*>(&w), &b, &i, &q, n, len, &opts);
    };
    auto attend = [&](Workspace w, const sage_cache_index& i, uint64_t len = 16) {
        const sage_cache_options opts{0, 0, 1};
        return sage_cache_attend_picked(&ctx, reinterpret_cast<sage_pick_workspace*>(&w), &cache, &i, n, len, &q, &o, &opts);
    };
    const sage_pick_options opts{1, 1, 1};
    CHECK(passed(update(H, bounds, INDEX)));
    CHECK(passed(pick(made, bounds, INDEX, opts)));
    CHECK(passed(attend(made, INDEX)));
    CHECK(refused(sage_cache_bounds_update(&ctx, &H, nullptr, &INDEX, &bounds), "null argument"));
    CHECK(refused(sage_cache_pick(&ctx, nullptr, &bounds, &INDEX, &q, n, 16, &opts), "null argument"));
    const sage_cache_options causal{0, 0, 1};
    CHECK(refused(sage_cache_attend_picked(&ctx, nullptr, &cache, &INDEX, n, 16, &q, &o, &causal), "null argument"));

    sage_cache_bounds b = bounds;
    b.codes_len--;
    CHECK(refused(update(H, b, INDEX), "bounds codes: buffer holds 2559 elements, needs 2560"));
    CHECK(refused(pick(made, b, INDEX, opts), "bounds codes: buffer holds 2559 elements, needs 2560"));
    b = bounds, b.scales = nullptr;
    CHECK(refused(update(H, b, INDEX), "bounds scales: buffer holds 0"));
    CHECK(refused(pick(made, b, INDEX, opts), "bounds scales: buffer holds 0"));
    b = bounds, b.codes += 8;
    CHECK(refused(update(H, b, INDEX), "bounds codes must start at a 16-byte aligned"));
    sage_cache_index i = INDEX;
    i.page_table_len = 5;
    CHECK(refused(update(H, bounds, i), "cache page table"));
    CHECK(refused(pick(made, bounds, i, opts), "cache page table"));
    CHECK(refused(attend(made, i), "cache page table"));
    sage_cache_shape tall = H;
    tall.heads = tall.kv_heads = 21845, tall.max_new = 98000;
    const sage_cache big{u, u, u, u, 1ull << 40, 1ull << 40};
    const sage_cache_bounds wide{reinterpret_cast<int8_t*>(mem), u, 1ull << 40, 1ull << 40};
    CHECK(refused(sage_cache_bounds_update(&ctx, &tall, &big, &INDEX, &wide), "98000 new rows of 21845 KV heads"));
    tall.max_new = 9000;
    CHECK(passed(sage_cache_bounds_update(&ctx, &tall, &big, &INDEX, &wide)));

    CHECK(refused(pick(made, bounds, INDEX, {1, 0, 1}), "the last is always one"));
    CHECK(refused(pick(made, bounds, INDEX, {2, 1, 1}), "the first 2 and the last 1 of 2 pages"));
    CHECK(refused(pick(made, bounds, INDEX, {0, 3, 1}), "the first 0 and the last 3 of 2 pages"));
    CHECK(refused(pick(made, bounds, INDEX, {~0ull, ~0ull, 1}), "pages"));
    CHECK(refused(pick(made, bounds, INDEX, {~0ull, 2, 1}), "pages"));
    CHECK(refused(pick(made, bounds, INDEX, opts, 15), "picked pages: buffer holds 15 elements, needs 16"));
    CHECK(refused(attend(made, INDEX, 15), "picked pages: buffer holds 15 elements, needs 16"));
    Workspace w = made;
    w.head_dim = 64;
    CHECK(refused(pick(w, bounds, INDEX, opts), "workspace was made for head dim 64"));
    CHECK(refused(attend(w, INDEX), "workspace was made for head dim 64"));
    w = made, w.device = 3;
    CHECK(refused(pick(w, bounds, INDEX, opts), "workspace is of device 3"));
    CHECK(refused(attend(w, INDEX), "workspace is of device 3"));

    sage_pick_workspace* ws = nullptr;
    auto shaped = [&](uint64_t top, auto change, const char* text) {
        sage_cache_shape h = H;
        change(h);
        CHECK(refused(sage_pick_workspace_new(&ctx, &h, top, &ws), text) && !ws);
    };
    CHECK(passed(sage_pick_workspace_new(&ctx, &H, 2, &ws)) && !ws);
    CHECK(passed(sage_pick_workspace_new(&ctx, &H, SAGE_PICK_TOP, &ws)) && !ws);
    CHECK(refused(sage_pick_workspace_new(&ctx, nullptr, 2, &ws), "null argument"));
    using A = sage_cache_shape&;
    shaped(0, [](A) {}, "pick: 0 pages a row (1 to 256 are supported)");
    shaped(257, [](A) {}, "pick: 257 pages a row");
    shaped(2, [](A h) { h.max_pages = 32769; }, "pick: 32769 columns");
    shaped(2, [](A h) { h.kv_heads = 3; }, "KV heads");
    shaped(2, [](A h) { h.rows = 1 << 21; }, "pick: 2097152 rows");
    shaped(2, [](A h) { h.max_new = 1 << 21; }, "of a sequence, of 4 and 2 heads exceed the launch grid");
    shaped(2, [](A h) { h.kv_heads = 1, h.heads = 1024, h.max_new = 1 << 18; }, "exceed the launch grid");
    CHECK(sage_pick_workspace_bytes(nullptr) == 0);
    sage_pick_workspace_destroy(nullptr);
}

// What a unit of the attention keeps in LDS fits the 160 KB of a compute unit at every allowed shape.
static void plans() {
    for (int d : {64, 128})
        for (int group : {1, 2, 3, 4, 7, 8, 16, 40})
            for (int top : {1, 2, 32, 256})
                for (int cols : {1, 3, 256, 32768})
                    for (int rows : {1, 2, 5, 1000}) {
                        const sage::PickedPlan p = sage::picked_plan(d, 3, rows, 2 * group, 2, rows, cols, 16, top);
                        CHECK(p.lds <= 64u << 10 && p.lds >= 4u * (2 + 3 * std::min(top, cols)));
                        CHECK(p.splits >= 1 && p.splits <= 256 && p.parts >= 1 && p.parts <= 256);
                        CHECK(!p.chunks || (rows * group > 16 && group <= 8 && p.chunk_lds <= 40u << 10));
                        CHECK(p.part_rows >= (p.splits > 1 ? (uint64_t)p.splits * rows * 2 * group : 0));
                        CHECK(p.part_rows >= (p.chunks ? 512u * 32 : 0));
                    }
    CHECK(!sage::picked_plan(64, 65535, 100000, 8 * 4000, 4000, 9, 4, 16, 4).chunks);
    CHECK(sage::picked_plan(64, 100, 100000, 8 * 40, 40, 1000, 4, 16, 4).chunks);
    // One launch where it fits, and never more keys than LDS has.
    CHECK(sage::pick_tiles(64, 4, 8, 1, 256) == 1 && sage::pick_tiles(1, 4, 8, 1, 1024) == 0);
    CHECK(sage::pick_tiles(2, 4, 8, 1000, 954) == 4 && sage::pick_tiles(1, 17, 8, 1000, 954) == 0);
    for (int group : {1, 2, 5, 16})
        for (int rows : {1, 3, 40, 2000})
            for (int cols : {1, 100, 1024, 2048, 2049}) {
                const int tiles = sage::pick_tiles(9, group, 3, rows, cols);
                int slots = 1;
                while (slots < group) slots *= 2;
                CHECK(tiles * std::min(tiles * 16 / slots, rows) * cols <= tiles << 14 && (tiles == 0 || cols <= 2048));
            }
    for (int cols : {1, 256, 32768})
        for (int kv : {1, 8, 100}) {
            const int w = sage::pick_window(4000000, kv, cols);
            CHECK(w >= 1 && (long long)w * kv * cols <= std::max(1ll << 26, (long long)kv * cols));
            CHECK(sage::pick_window(3, kv, cols) == 3);
        }
}

int main() {
    axes();
    tables();
    picks();
    plans();
    if (failed) return std::printf("%d checks failed\n", failed), 1;
    std::printf("pick host tests passed\n");
    return 0;
}
