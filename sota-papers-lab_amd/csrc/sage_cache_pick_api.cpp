// C ABI of a step's index, of the pages' bounds and of the attention over picked
// pages (include/sage_hip.h): every check before any launch, then the launches on the
// context's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "sage_cache_checks.hpp"

using namespace sage::checks;
using sage::set_error;
using sage::succeeded;

struct sage_pick_workspace {
    sage_cache_shape shape;
    uint64_t head_dim, top, bytes;
    int device, window;
    sage::PickedPlan plan;
    void* buf;  // a pick's keys, or an attention's partial outputs
};

namespace {

// What the calls over picks ask of a shape beside shape_checked: lists that fit the
// kernels' LDS, and in a grid's x a workgroup a row and KV head, or 16 columns of one.
sage_status pick_shape_checked(const sage_cache_shape& h, uint64_t top) {
    const sage_status st = shape_checked(h);
    if (st != SAGE_OK) return st;
    if (top < 1 || top > SAGE_PICK_TOP)
        return set_error(SAGE_ERR_INVALID, "pick: %llu pages a row (1 to %d are supported)", (u64)top, SAGE_PICK_TOP);
    if (h.max_pages > SAGE_PICK_PAGES)
        return set_error(SAGE_ERR_INVALID, "pick: %llu columns in the page table (at most %d are supported)",
                         (u64)h.max_pages, SAGE_PICK_PAGES);
    if (std::max(h.rows, h.max_new) * h.kv_heads >= 1ull << 22 ||
        (h.max_new * (h.heads / h.kv_heads) + 15) / 16 * h.kv_heads >= 1ull << 24)
        return set_error(SAGE_ERR_INVALID, "pick: %llu rows, %llu of a sequence, of %llu and %llu heads exceed the launch grid",
                         (u64)h.rows, (u64)h.max_new, (u64)h.heads, (u64)h.kv_heads);
    return SAGE_OK;
}

sage_status bounds_checked(const sage_cache_shape& h, uint64_t d, const sage_cache_bounds& b, sage::BoundsDev* out) {
    const uint64_t cells = h.pages * h.kv_heads;
    sage_status st = buffer(b.codes, b.codes_len, cells * 2 * d, 16, "bounds codes");
    if (st == SAGE_OK) st = buffer(b.scales, b.scales_len, cells, 16, "bounds scales");
    if (st == SAGE_OK) *out = {b.codes, b.scales};
    return st;
}

sage_status workspace_fits(const sage_attention* s, const sage_pick_workspace* ws) {
    if (ws->head_dim != s->head_dim)
        return set_error(SAGE_ERR_INVALID, "workspace was made for head dim %llu, kernels are %llu", (u64)ws->head_dim,
                         (u64)s->head_dim);
    if (ws->device != s->device)
        return set_error(SAGE_ERR_INVALID, "workspace is of device %d, the context of %d", ws->device, s->device);
    return SAGE_OK;
}

}  // namespace

extern "C" {

sage_status sage_cache_tables(const sage_attention* s, const sage_cache_shape* shape,
                              const sage_cache_requests* requests, const sage_cache_free* free,
                              const sage_cache_step* step) {
    if (!s || !shape || !requests || !free || !step) return set_error(SAGE_ERR_INVALID, "null argument");
    const sage_cache_shape& h = *shape;
    sage_status st = shape_checked(h);
    if (st == SAGE_OK) st = buffer(requests->news, requests->news_len, h.batch, 4, "request rows");
    if (st == SAGE_OK) st = buffer(requests->past, requests->past_len, h.batch, 4, "request lengths");
    if (st == SAGE_OK && free->pages_len == 0) st = set_error(SAGE_ERR_INVALID, "free pages: a ring of no places");
    if (st == SAGE_OK) st = in_i32(free->pages_len, "free pages");
    if (st == SAGE_OK) st = buffer(free->pages, free->pages_len, 1, 4, "free pages");
    if (st == SAGE_OK) st = buffer(free->state, free->state_len, 2, 4, "free pages' state");
    if (st == SAGE_OK) st = buffer(step->starts, step->starts_len, h.batch + 1, 4, "cache starts");
    if (st == SAGE_OK) st = buffer(step->lengths, step->lengths_len, h.batch, 4, "cache lengths");
    if (st == SAGE_OK) st = buffer(step->page_table, step->page_table_len, h.batch * h.max_pages, 4, "cache page table");
    if (st == SAGE_OK && step->positions) st = buffer(step->positions, step->positions_len, h.rows, 16, "step positions");
    if (st == SAGE_OK && step->slots) st = buffer(step->slots, step->slots_len, h.rows, 16, "step slots");
    if (st == SAGE_OK && step->sequences) st = buffer(step->sequences, step->sequences_len, h.rows, 16, "step sequences");
    if (st == SAGE_OK) st = buffer(step->state, step->state_len, 4, 4, "step state");
    if (st == SAGE_OK) st = buffer(step->scratch, step->scratch_len, 2 * h.batch, 4, "step scratch");
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    int shift = 4;
    while ((1ull << shift) < h.page_tokens) shift++;
    const sage::StepArgs a{requests->news, requests->past, free->state,  free->pages,
                           step->starts,   step->lengths,  step->page_table, step->state,
                           step->scratch,  step->positions, step->sequences,
                           reinterpret_cast<long long*>(step->slots),
                           (int)h.batch,   (int)h.rows,    shift,        (int)h.max_pages,
                           (int)h.pages,   (int)free->pages_len};
    return done(sage::launch_cache_step(a, s->stream), "launch cache tables");
}

sage_status sage_cache_bounds_update(const sage_attention* s, const sage_cache_shape* shape, const sage_cache* cache,
                                     const sage_cache_index* index, const sage_cache_bounds* bounds) {
    if (!s || !shape || !cache || !index || !bounds) return set_error(SAGE_ERR_INVALID, "null argument");
    const sage_cache_shape& h = *shape;
    sage::BoundsArgs a{};
    sage_status st = cache_checked(h, s->head_dim, *cache, *index, &a.c);
    if (st == SAGE_OK) st = bounds_checked(h, s->head_dim, *bounds, &a.bounds);
    if (st == SAGE_OK && (h.max_new / h.page_tokens + 2) * h.kv_heads >= 1ull << 24)
        st = set_error(SAGE_ERR_INVALID, "bounds: %llu new rows of %llu KV heads exceed the launch grid", (u64)h.max_new,
                       (u64)h.kv_heads);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (h.batch == 0 || h.max_new == 0) return succeeded();
    a.max_new = (int)h.max_new;
    return done(sage::launch_cache_bounds((int)s->head_dim, a, s->stream), "launch cache bounds");
}

sage_status sage_pick_workspace_new(const sage_attention* s, const sage_cache_shape* shape, uint64_t top,
                                    sage_pick_workspace** out) {
    if (!out) return set_error(SAGE_ERR_INVALID, "null output");
    *out = nullptr;
    if (!s || !shape) return set_error(SAGE_ERR_INVALID, "null argument");
    const sage_cache_shape& h = *shape;
    sage_status st = pick_shape_checked(h, top);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    const int window = sage::pick_window((int)h.rows, (int)h.kv_heads, (int)h.max_pages);
    const sage::PickedPlan plan =
        sage::picked_plan((int)s->head_dim, (int)h.batch, (int)h.rows, (int)h.heads, (int)h.kv_heads, (int)h.max_new,
                          (int)h.max_pages, (int)h.page_tokens, (int)top);
    // A key is 4 bytes, where memory keeps them and not every page is picked anyway; a partial
    // row D floats, a maximum and a sum.
    const bool in_memory = h.max_pages > top && !sage::pick_tiles((int)h.batch, (int)(h.heads / h.kv_heads), (int)h.kv_heads,
                                                                  (int)h.max_new, (int)h.max_pages);
    const uint64_t keys = in_memory ? 4ull * window * h.kv_heads * h.max_pages : 0;
    uint64_t bytes = 0;
    if (__builtin_mul_overflow(plan.part_rows, (s->head_dim + 2) * 4, &bytes) || bytes > 1ull << 62)
        return set_error(SAGE_ERR_INVALID, "pick workspace needs more than 2^62 bytes");
    bytes = std::max(bytes, keys);
    sage_pick_workspace* w =
        new (std::nothrow) sage_pick_workspace{h, s->head_dim, top, bytes, s->device, window, plan, nullptr};
    if (!w) return set_error(SAGE_ERR_DEVICE, "out of host memory");
    if (bytes) {
        const hipError_t e = hipMalloc(&w->buf, bytes);
        if (e != hipSuccess) {
            delete w;
            return hip_failed(e, "allocate pick workspace");
        }
    }
    *out = w;
    return succeeded();
}

void sage_pick_workspace_destroy(sage_pick_workspace* ws) {
    if (!ws) return;
    if (ws->buf) (void)hipFree(ws->buf);
    delete ws;
}

uint64_t sage_pick_workspace_bytes(const sage_pick_workspace* ws) { return ws ? ws->bytes : 0; }

sage_status sage_cache_pick(const sage_attention* s, const sage_pick_workspace* ws, const sage_cache_bounds* bounds,
                            const sage_cache_index* index, const sage_tensor* q, int32_t* picked, uint64_t picked_len,
                            const sage_pick_options* opts) {
    if (!s || !ws || !bounds || !index || !q || !opts) return set_error(SAGE_ERR_INVALID, "null argument");
    sage_status st = workspace_fits(s, ws);
    if (st != SAGE_OK) return st;
    if (opts->last < 1 || opts->first > ws->top || opts->last > ws->top - opts->first)
        return set_error(SAGE_ERR_INVALID, "pick: the first %llu and the last %llu of %llu pages (the last is always one)",
                         (u64)opts->first, (u64)opts->last, (u64)ws->top);
    const sage_cache_shape& h = ws->shape;
    sage::PickArgs a{};
    st = index_checked(h, *index, &a.c);
    if (st == SAGE_OK) st = bounds_checked(h, s->head_dim, *bounds, &a.bounds);
    if (st == SAGE_OK) st = view(q, h.rows, h.heads, s->head_dim, "Q");
    if (st == SAGE_OK) st = buffer(picked, picked_len, h.rows * h.kv_heads * ws->top, 4, "picked pages");
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (h.rows == 0 || h.batch == 0 || h.max_new == 0) return succeeded();
    a.q = rows_of(q);
    a.keys = static_cast<uint32_t*>(ws->buf);
    a.picked = picked;
    a.heads = (int)h.heads;
    a.group = (int)(h.heads / h.kv_heads);
    a.max_new = (int)h.max_new;
    a.causal = opts->causal != 0;
    a.q_f16 = q->dtype == SAGE_F16;
    a.top = (int)ws->top;
    a.first = (int)opts->first;
    a.last = (int)opts->last;
    a.window = ws->window;
    a.key_cols = (int)h.max_pages;
    return done(sage::launch_cache_pick((int)s->head_dim, a, s->stream), "launch cache pick");
}

sage_status sage_cache_attend_picked(const sage_attention* s, const sage_pick_workspace* ws, const sage_cache* cache,
                                     const sage_cache_index* index, const int32_t* picked, uint64_t picked_len,
                                     const sage_tensor* q, const sage_tensor_mut* out, const sage_cache_options* opts) {
    if (!s || !ws || !cache || !index || !q || !out || !opts) return set_error(SAGE_ERR_INVALID, "null argument");
    sage_status st = workspace_fits(s, ws);
    if (st != SAGE_OK) return st;
    const sage_cache_shape& h = ws->shape;
    sage::CacheAttnArgs a{};
    st = cache_checked(h, s->head_dim, *cache, *index, &a.c);
    if (st == SAGE_OK) st = buffer(picked, picked_len, h.rows * h.kv_heads * ws->top, 4, "picked pages");
    if (st == SAGE_OK) st = attend_checked(h, s->head_dim, q, out, *opts, &a);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (h.rows == 0 || h.batch == 0 || h.max_new == 0) return succeeded();
    a.picked = picked;
    a.top = (int)ws->top;
    a.part_o = static_cast<float*>(ws->buf);
    a.part_ml = ws->buf ? a.part_o + ws->plan.part_rows * s->head_dim : nullptr;
    return done(sage::launch_cache_attend_picked((int)s->head_dim, a, ws->plan, s->stream),
                "launch attention over picked pages");
}

}  // extern "C"
