// The rotary and paged-cache entry points on the CPU: every refusal, in its
// order and with its text, on a context made by hand (a call that passes every
// check then fails on the device), and the kernels' index lookups on bad
// indexes, where each read has to stay inside its array.
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

static void index_lookups() {
    sage::CacheDev c{};
    // Arrays of exactly the sizes the entry points ask for (the build checks addresses).
    std::vector<int> starts, lengths, table;
    auto set = [&](std::vector<int> s, std::vector<int> l, std::vector<int> t, int cols, int pages) {
        starts = std::move(s), lengths = std::move(l), table = std::move(t);
        c.starts = starts.data(), c.lengths = lengths.data(), c.page_table = table.data();
        c.batch = (int)lengths.size(), c.max_pages = cols, c.pages = pages, c.page_shift = 4, c.kv_heads = 3;
        c.rows = 1000;
        CHECK((int)starts.size() == c.batch + 1 && (int)table.size() == c.batch * cols);
    };
    const int lo = -2147483647 - 1, hi = 2147483647;
    set({2, 5, 5, 9}, {3, 0, 40}, {0, 6, 7, -1, lo, hi, 1, 2, 3}, 3, 7);
    const int want[12] = {-1, -1, 0, 0, 0, 2, 2, 2, 2, -1, -1, -1};
    for (int r = 0; r < 12; r++) CHECK(sage::sequence_of(c, r) == want[r]);
    CHECK(sage::slot_of(c, 0, 2) == 0 && sage::slot_of(c, 0, 4) == 2 && sage::slot_of(c, 2, 5) == 36);
    CHECK(sage::cache_page(c, 0, 0) == 0 && sage::cache_page(c, 0, 31) == 6 && sage::cache_page(c, 0, 32) == -1);
    CHECK(sage::cache_page(c, 1, 0) == -1 && sage::cache_page(c, 1, 16) == -1 && sage::cache_page(c, 1, 47) == -1);
    CHECK(sage::cache_page(c, 2, 47) == 3 && sage::cache_page(c, 2, 48) == -1 && sage::cache_page(c, 2, -1) == -1);
    CHECK(sage::cache_page(c, 2, hi) == -1 && sage::cache_page(c, 2, lo) == -1);
    CHECK(sage::cache_row(c, 2147483646, 2, 15) == ((2147483646ll * 3 + 2) << 4) + 15);
    // Starts and lengths that make no sense: every answer is in range.
    const int bad[] = {lo, -5, 0, 3, 999, 1000, hi};
    for (int s0 : bad)
        for (int s1 : bad)
            for (int s2 : bad)
                for (int l : bad) {
                    set({s0, s1, s2}, {l, l}, {1, 2, 3, 4}, 2, 7);
                    for (int r = 0; r < 1000; r += 37) {
                        const int b = sage::sequence_of(c, r);
                        CHECK(b >= -1 && b < 2);
                        if (b >= 0) {
                            const int page = sage::cache_page(c, b, sage::slot_of(c, b, r));
                            CHECK(page >= -1 && page < 7);
                        }
                    }
                    for (int b = 0; b < 2; b++) {
                        const sage::SequenceIndex q = sage::sequence_index(c, b, 100);
                        CHECK(q.n >= 0 && q.n <= 100 && q.len >= 0 && q.len <= 32);
                        for (int j : {0, 50, 99, 100000})
                            for (int causal : {0, 1}) CHECK(q.limit(j, causal) >= 0 && q.limit(j, causal) <= q.len);
                    }
                }
}

static void refusals() {
    sage_attention ctx{nullptr, -2, 128, sage_config_for_head_dim(128)};
    alignas(256) static char mem[4096];
    float table[64 * 8];
    const sage_shape shape{1, 4, 8, 0};
    const sage_strides st{4096, 512, 128};
    sage_tensor x{mem, 4096, st, SAGE_BF16};
    sage_tensor_mut o{mem, 4096, st, SAGE_BF16};
    sage_rotary r{reinterpret_cast<float*>(mem), 64 * 8, 64, SAGE_ROTARY_HALF, nullptr, 0};
    CHECK(passed(sage_rotary_apply(&ctx, &shape, &r, &x, &o, 0)));
    CHECK(refused(sage_rotary_apply(nullptr, &shape, &r, &x, &o, 0), "null argument"));
    CHECK(refused(sage_rotary_apply(&ctx, &shape, nullptr, &x, &o, 0), "null argument"));
    const sage_shape none{1, 4, 0, 0}, wide{1ull << 20, 4, 1ull << 20, 0}, wraps{1ull << 40, 4, 1ull << 40, 0};
    CHECK(sage_rotary_apply(&ctx, &none, &r, &x, &o, 0) == SAGE_OK);
    CHECK(refused(sage_rotary_apply(&ctx, &wide, &r, &x, &o, 0), "do not fit in i32"));
    CHECK(refused(sage_rotary_apply(&ctx, &wraps, &r, &x, &o, 0), "do not fit in i32"));
    const sage_shape tall{1ull << 6, 1, 1ull << 20, 0}, broad{1, (1ull << 30) + 1, 1, 0};
    CHECK(refused(sage_rotary_apply(&ctx, &tall, &r, &x, &o, 0), "exceed the launch grid"));
    CHECK(refused(sage_rotary_apply(&ctx, &broad, &r, &x, &o, 0), "exceed the launch grid"));
    auto rot = [&](auto change, const char* text) {
        sage_rotary q = r;
        change(q);
        CHECK(refused(sage_rotary_apply(&ctx, &shape, &q, &x, &o, 0), text));
    };
    rot([](sage_rotary& q) { q.layout = 2; }, "unknown layout 2");
    rot([](sage_rotary& q) { q.rot = 0; }, "rotated channels");
    rot([](sage_rotary& q) { q.rot = 7; }, "rotated channels");
    rot([](sage_rotary& q) { q.rot = 130; }, "rotated channels");
    rot([](sage_rotary& q) { q.table_len = 63; }, "rotary table: buffer holds 63 elements, needs 64");
    rot([](sage_rotary& q) { q.table = nullptr; }, "rotary table");
    rot([](sage_rotary& q) { q.table++; }, "16-byte aligned");
    rot([](sage_rotary& q) { q.table_len = 1ull << 40; }, "does not fit in i32");
    rot([](sage_rotary& q) { q.positions = (int*)mem, q.positions_len = 7; }, "rotary positions: buffer holds 7 elements, needs 8");
    rot([](sage_rotary& q) { q.positions = (int*)(mem + 2), q.positions_len = 8; }, "4-byte aligned");
    auto tensor = [&](auto change, const char* text) {
        sage_tensor t = x;
        change(t);
        CHECK(refused(sage_rotary_apply(&ctx, &shape, &r, &t, &o, 0), text));
    };
    tensor([](sage_tensor& t) { t.strides.head = 4; }, "multiples of 8");
    tensor([](sage_tensor& t) { t.len = 4095; }, "buffer holds 4095 elements, needs 4096");
    tensor([](sage_tensor& t) { t.data = mem + 8; }, "16-byte aligned");
    tensor([](sage_tensor& t) { t.dtype = 2; }, "unknown dtype 2");
    tensor([](sage_tensor& t) { t.dtype = SAGE_F16; }, "one element type");
    tensor([](sage_tensor& t) { t.strides.token = 1ull << 63; }, "exceed 2^62");

    // The table.
    CHECK(sage_rotary_table(64, 8, 1e4, nullptr, table, 512) == SAGE_OK);
    CHECK(refused(sage_rotary_table(64, 8, 1e4, nullptr, table, 511), "buffer holds 511"));
    CHECK(refused(sage_rotary_table(63, 8, 1e4, nullptr, table, 512), "even number"));
    CHECK(refused(sage_rotary_table(64, 8, 1.0, nullptr, table, 512), "base"));
    CHECK(refused(sage_rotary_table(64, 1ull << 33, 1e4, nullptr, table, 512), "does not fit in i32"));
    CHECK(refused(sage_rotary_table(64, 8, 1e4, nullptr, nullptr, 512), "null argument"));
    sage_rotary_scaling sc{SAGE_ROTARY_YARN, 4, 4096, 0, 0, 0};
    CHECK(sage_rotary_table(64, 8, 1e4, &sc, table, 512) == SAGE_OK);
    sc.factor = 0.5;
    CHECK(refused(sage_rotary_table(64, 8, 1e4, &sc, table, 512), "scaling factor"));
    sc = {SAGE_ROTARY_YARN, 4, 0, 0, 0, 0};
    CHECK(refused(sage_rotary_table(64, 8, 1e4, &sc, table, 512), "YaRN"));
    sc = {SAGE_ROTARY_YARN, 4, 4096, 2, 3, 0};
    CHECK(refused(sage_rotary_table(64, 8, 1e4, &sc, table, 512), "YaRN"));
    sc = {SAGE_ROTARY_NTK, 4, 0, 0, 0, 0};
    CHECK(refused(sage_rotary_table(2, 8, 1e4, &sc, table, 512), "NTK"));
    sc.kind = 4;
    CHECK(refused(sage_rotary_table(64, 8, 1e4, &sc, table, 512), "unknown scaling 4"));

    // The cache: two sequences of three and one rows, 4 query heads over 2 KV heads.
    const sage_cache_shape h{2, 4, 3, 4, 2, 5, 16, 3};
    uint64_t codes = 0, scales = 0;
    CHECK(sage_cache_sizes(&h, 128, &codes, &scales) == SAGE_OK && codes == 5 * 2 * 16 * 64 && scales == 5 * 2 * 16 * 4);
    CHECK(sage_cache_sizes(&h, 64, &codes, &scales) == SAGE_OK && codes == 5 * 2 * 16 * 32 && scales == 5 * 2 * 16 * 2);
    CHECK(refused(sage_cache_sizes(&h, 96, &codes, &scales), "head dim 64 or 128"));
    CHECK(refused(sage_cache_sizes(nullptr, 64, &codes, &scales), "null argument"));
    uint8_t* u = reinterpret_cast<uint8_t*>(mem);
    int32_t* n = reinterpret_cast<int32_t*>(mem);
    const sage_cache cache{u, u, u, u, 5 * 2 * 16 * 64, 5 * 2 * 16 * 4};
    const sage_cache_index index{n, 3, n, 2, n, 6};
    const sage_tensor kv{mem, 4 * 256, {0, 256, 128}, SAGE_F16}, q{mem, 4 * 512, {0, 512, 128}, SAGE_F16};
    const sage_tensor_mut kvo{mem, 4 * 256, {0, 256, 128}, SAGE_F16}, qo{mem, 4 * 512, {0, 512, 128}, SAGE_F16};
    auto append = [&](const sage_cache_shape& h, const sage_cache& c, const sage_cache_index& i) {
        return sage_cache_append(&ctx, &h, &c, &i, &kv, &kv, &r, &q, &qo);
    };
    auto read = [&](const sage_cache_shape& h, const sage_cache& c, const sage_cache_index& i) {
        return sage_cache_read(&ctx, &h, &c, &i, &kvo, &kvo);
    };
    auto attend = [&](const sage_cache_shape& h, const sage_cache& c, const sage_cache_index& i) {
        // A workspace as sage_cache_workspace_new makes it needs the device: the same fields by hand.
        struct {
            sage_cache_shape shape;
            uint64_t head_dim, bytes;
            int device;
            sage::CachePlan plan;
            void* buf;
        } ws{h, 128, 0, -2, {false, true, 1, 0}, nullptr};
        const sage_cache_options o{0, 0, 1};
        return sage_cache_attend(&ctx, reinterpret_cast<sage_cache_workspace*>(&ws), &c, &i, &q, &qo, &o);
    };
    CHECK(passed(append(h, cache, index)));
    CHECK(passed(read(h, cache, index)));
    CHECK(passed(attend(h, cache, index)));
    CHECK(passed(sage_cache_append(&ctx, &h, &cache, &index, &kv, &kv, nullptr, nullptr, nullptr)));
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, &kv, &kv, &r, &q, nullptr), "queries need"));
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, &kv, &kv, &r, nullptr, &qo), "queries need"));
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, &kv, &kv, nullptr, &q, &qo), "queries need"));
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, nullptr, &kv, &r, &q, &qo), "null argument"));
    sage_tensor other = kv;
    other.dtype = SAGE_BF16;
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, &kv, &other, &r, &q, &qo), "one element type"));
    other = kv, other.len--;
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, &other, &kv, &r, &q, &qo), "cache append K: buffer holds"));
    CHECK(refused(sage_cache_append(&ctx, &h, &cache, &index, &kv, &other, &r, &q, &qo), "cache append V: buffer holds"));
    sage_cache_workspace* ws = nullptr;
    CHECK(passed(sage_cache_workspace_new(&ctx, &h, &ws)) && !ws);
    CHECK(refused(sage_cache_workspace_new(&ctx, nullptr, &ws), "null argument"));
    CHECK(sage_cache_workspace_bytes(nullptr) == 0);
    sage_cache_workspace_destroy(nullptr);

    auto all = [&](auto change, const char* text) {
        sage_cache_shape hh = h;
        sage_cache c = cache;
        sage_cache_index i = index;
        change(hh, c, i);
        CHECK(refused(append(hh, c, i), text));
        CHECK(refused(read(hh, c, i), text));
        CHECK(refused(attend(hh, c, i), text));
    };
    using H = sage_cache_shape&;
    using C = sage_cache&;
    using I = sage_cache_index&;
    all([](H h, C, I) { h.kv_heads = 3; }, "4 query heads are not a multiple of 3 KV heads");
    all([](H h, C, I) { h.kv_heads = 0; }, "KV heads");
    all([](H h, C, I) { h.heads = 0; }, "KV heads");
    all([](H h, C, I) { h.page_tokens = 8; }, "pages of 8 tokens");
    all([](H h, C, I) { h.page_tokens = 48; }, "pages of 48 tokens");
    all([](H h, C, I) { h.page_tokens = 512; }, "pages of 512 tokens");
    all([](H h, C, I) { h.pages = 0; }, "0 pages in the pool");
    all([](H h, C, I) { h.max_pages = 0; }, "0 columns in the page table");
    all([](H h, C, I) { h.pages = 1ull << 31; }, "does not fit in i32");
    all([](H h, C, I) { h.rows = 1ull << 31; }, "does not fit in i32");
    all([](H h, C, I) { h.rows = 1ull << 26; }, "exceed the launch grid");
    all([](H h, C, I) { h.max_pages = (1ull << 26) + 1; }, "exceed 2^30 tokens");
    all([](H h, C, I) { h.max_pages = ~0ull; }, "exceed 2^30 tokens");
    all([](H h, C, I) { h.batch = 65536; }, "exceed the launch grid");
    all([](H h, C, I) { h.heads = 65536, h.kv_heads = 1; }, "exceed the launch grid");
    all([](H h, C, I) { h.heads = h.kv_heads = 30000; }, "exceed the launch grid");
    all([](H h, C, I) { h.max_new = 1ull << 31; }, "exceed the launch grid");
    all([](H h, C, I) { h.heads = h.kv_heads = 64, h.max_new = (1ull << 25) - 1; }, "exceed the launch grid");
    all([](H h, C, I) { h.pages = 6; }, "cache K codes: buffer holds 10240 elements, needs 12288");
    all([](H, C c, I) { c.scales_len--; }, "cache K scales: buffer holds 639 elements, needs 640");
    all([](H, C c, I) { c.k_codes = nullptr; }, "cache K codes: buffer holds 0");
    all([](H, C c, I) { c.v_codes += 8; }, "cache V codes must start at a 16-byte aligned");
    all([](H, C c, I) { c.v_scales++; }, "cache V scales must start at a 16-byte aligned");
    all([](H, C, I i) { i.starts_len = 2; }, "cache starts: buffer holds 2 elements, needs 3");
    all([](H, C, I i) { i.lengths_len = 1; }, "cache lengths: buffer holds 1 elements, needs 2");
    all([](H, C, I i) { i.page_table_len = 5; }, "cache page table: buffer holds 5 elements, needs 6");
    all([](H, C, I i) { i.lengths = (int32_t*)(mem + 1); }, "cache lengths must start at a 4-byte aligned");
    all([](H h, C, I) { h.rows = 5; }, "buffer holds");
    // Nothing to do is no error, whatever the (empty) tensors' addresses are, once the device is there.
    const sage_tensor e{nullptr, 0, {0, 256, 128}, SAGE_F16};
    const sage_tensor_mut eo{nullptr, 0, {0, 256, 128}, SAGE_F16};
    sage_cache_shape zero = h;
    zero.rows = 0;
    CHECK(passed(sage_cache_append(&ctx, &zero, &cache, &index, &e, &e, nullptr, nullptr, nullptr)));
    CHECK(passed(sage_cache_read(&ctx, &zero, &cache, &index, &eo, &eo)));
}

// The most rows that a rotation takes: four to a workgroup of 256, so 2^26 - 4
// of them are the last below a launch's 2^32 threads.
static void row_limit() {
    sage_attention ctx{nullptr, -2, 128, sage_config_for_head_dim(128)};
    alignas(256) static char mem[256];
    const sage_strides st{0, 128, 128};
    const sage_tensor x{mem, 1ull << 40, st, SAGE_BF16};
    const sage_tensor_mut o{mem, 1ull << 40, st, SAGE_BF16};
    const sage_rotary r{reinterpret_cast<float*>(mem), 64, 64, SAGE_ROTARY_HALF, nullptr, 0};
    for (uint64_t more = 0; more <= 5; more++) {
        const sage_shape shape{1, 1, (1ull << 26) - 5 + more, 0};
        const sage_status s = sage_rotary_apply(&ctx, &shape, &r, &x, &o, 0);
        CHECK(more < 2 ? passed(s) : refused(s, "exceed the launch grid"));
    }
}

int main() {
    index_lookups();
    refusals();
    row_limit();
    if (failed) return std::printf("%d checks failed\n", failed), 1;
    std::printf("cache host tests passed\n");
    return 0;
}
