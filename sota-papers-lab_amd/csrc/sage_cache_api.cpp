// C ABI of the rotary and paged-cache entry points (include/sage_hip.h): every
// check before any launch, then the launch on the context's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "sage_cache_checks.hpp"

using namespace sage::checks;
using sage::set_error;
using sage::succeeded;

struct sage_cache_workspace {
    sage_cache_shape shape;
    uint64_t head_dim, bytes;
    int device;
    sage::CachePlan plan;
    void* buf;
};

namespace {

// The angles' speeds under a scaling: w_i of a table of rot channels.
struct Speeds {
    int kind = SAGE_ROTARY_NONE;
    double base = 0, f = 1, original = 0, fast = 0, slow = 0, attention = 1;

    sage_status checked(double base_, const sage_rotary_scaling* scaling, uint64_t least_rot) {
        base = base_;
        kind = scaling ? scaling->kind : SAGE_ROTARY_NONE;
        if (kind < SAGE_ROTARY_NONE || kind > SAGE_ROTARY_YARN)
            return set_error(SAGE_ERR_INVALID, "rotary: unknown scaling %d", kind);
        f = kind == SAGE_ROTARY_NONE ? 1.0 : scaling->factor;
        if (!(f >= 1.0) || !std::isfinite(f))
            return set_error(SAGE_ERR_INVALID, "rotary: scaling factor %g is not 1 or more", f);
        attention = scaling && scaling->attention != 0.0 ? scaling->attention : 1.0;
        if (!std::isfinite(attention)) return set_error(SAGE_ERR_INVALID, "rotary: attention factor %g", attention);
        if (kind == SAGE_ROTARY_NTK && least_rot < 4)
            return set_error(SAGE_ERR_INVALID, "rotary: NTK scaling needs 4 rotated channels or more");
        if (kind == SAGE_ROTARY_YARN) {
            original = scaling->original;
            fast = scaling->beta_fast != 0.0 ? scaling->beta_fast : 32.0;
            slow = scaling->beta_slow != 0.0 ? scaling->beta_slow : 1.0;
            if (!(original > 0.0) || !std::isfinite(original) || !(slow < fast) || !std::isfinite(fast))
                return set_error(SAGE_ERR_INVALID, "rotary: YaRN scaling of %g positions between %g and %g turns",
                                 original, slow, fast);
            if (scaling->attention == 0.0) attention = 0.1 * std::log(f) + 1.0;
        }
        return SAGE_OK;
    }

    double of(uint64_t i, uint64_t rot) const {
        const double b = kind == SAGE_ROTARY_NTK ? base * std::pow(f, (double)rot / (double)(rot - 2)) : base;
        double w = std::pow(b, -2.0 * (double)i / (double)rot);
        if (kind == SAGE_ROTARY_LINEAR) w /= f;
        if (kind == SAGE_ROTARY_YARN) {
            // Peng et al., "YaRN: Efficient Context Window Extension of Large Language
            // Models", 2023: pairs that turn often keep their angle, slow ones are interpolated.
            const double turns = original * w / (2.0 * 3.14159265358979323846);
            const double g = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            w = g * w + (1.0 - g) * w / f;
        }
        return w;
    }

    // One pair's column of a table of `pairs` pairs.
    void column(float* out, uint64_t pairs, uint64_t pair, uint64_t positions, double w) const {
        for (uint64_t p = 0; p < positions; p++) {
            const double a = (double)p * w;
            out[(p * pairs + pair) * 2] = (float)(attention * std::cos(a));
            out[(p * pairs + pair) * 2 + 1] = (float)(attention * std::sin(a));
        }
    }
};

sage_status table_room(uint64_t positions, uint64_t rot, uint64_t out_len) {
    const sage_status st = in_i32(positions, "rotary positions");
    if (st != SAGE_OK || out_len >= positions * rot) return st;
    return set_error(SAGE_ERR_INVALID, "rotary table: buffer holds %llu elements, needs %llu", (u64)out_len,
                     (u64)(positions * rot));
}

// The pairs of all axes together, at most `most`.
sage_status sections_checked(const uint64_t* sections, uint64_t axes, uint64_t most, uint64_t* pairs) {
    if (axes < 1 || axes > SAGE_ROTARY_AXES)
        return set_error(SAGE_ERR_INVALID, "rotary: %llu axes (1 to %d are supported)", (u64)axes, SAGE_ROTARY_AXES);
    *pairs = 0;
    for (uint64_t a = 0; a < axes; a++) {
        if (sections[a] < 1 || sections[a] > most)
            return set_error(SAGE_ERR_INVALID, "rotary: axis %llu of %llu pairs (1 to %llu)", (u64)a, (u64)sections[a],
                             (u64)most);
        *pairs += sections[a];
    }
    if (*pairs > most)
        return set_error(SAGE_ERR_INVALID, "rotary: %llu rotated channels of head dim %llu: an even number from 2 to it",
                         (u64)(2 * *pairs), (u64)(2 * most));
    return SAGE_OK;
}
// each(i, a, j): pair i is the j-th of axis a.
template <class Each>
void deal(const uint64_t* sections, uint64_t axes, uint64_t pairs, bool dealt, Each each) {
    uint64_t got[SAGE_ROTARY_AXES] = {}, a = 0;
    for (uint64_t i = 0; i < pairs; i++) {
        while (got[a] == sections[a]) a = (a + 1) % axes;
        each(i, a, got[a]++);
        if (dealt) a = (a + 1) % axes;
    }
}

sage_status checked(const sage_rotary* r, uint64_t d, uint64_t rows, int transpose, sage::RotaryDev* out) {
    if (r->layout != SAGE_ROTARY_HALF && r->layout != SAGE_ROTARY_PAIRS)
        return set_error(SAGE_ERR_INVALID, "rotary: unknown layout %d", r->layout);
    if (r->rot < 2 || r->rot % 2 || r->rot > d)
        return set_error(SAGE_ERR_INVALID,
                         "rotary: %llu rotated channels of head dim %llu: an even number from 2 to it", (u64)r->rot,
                         (u64)d);
    sage_status st = buffer(r->table, r->table_len, r->rot, 16, "rotary table");
    if (st == SAGE_OK) st = in_i32(r->table_len / r->rot, "rotary positions");
    if (st == SAGE_OK && r->positions) st = buffer(r->positions, r->positions_len, rows, 4, "rotary positions");
    if (st != SAGE_OK) return st;
    *out = {r->table, r->positions, (int)(r->table_len / r->rot), (int)r->rot, r->layout, transpose != 0};
    return SAGE_OK;
}

sage_status checked(const sage_rotary_axes* r, uint64_t d, uint64_t rows, int transpose, sage::RotaryDev* out) {
    if (r->layout < SAGE_ROTARY_AXES_HALF || r->layout > SAGE_ROTARY_AXES_AXIS_HALF)
        return set_error(SAGE_ERR_INVALID, "rotary: unknown layout %d", r->layout);
    uint64_t pairs = 0;
    sage_status st = sections_checked(r->sections, r->axes, d / 2, &pairs);
    if (st != SAGE_OK) return st;
    if (r->dealt && r->layout == SAGE_ROTARY_AXES_AXIS_HALF)
        return set_error(SAGE_ERR_INVALID, "rotary: the halves of an axis's channels need its pairs in one run");
    st = buffer(r->table, r->table_len, 2 * pairs, 16, "rotary table");
    if (st == SAGE_OK) st = in_i32(r->table_len / (2 * pairs), "rotary positions");
    if (st == SAGE_OK && (r->positions_stride < rows || r->positions_stride >= 1ull << 60))
        st = set_error(SAGE_ERR_INVALID, "rotary positions: %llu entries from axis to axis, %llu rows",
                       (u64)r->positions_stride, (u64)rows);
    if (st == SAGE_OK)
        st = buffer(r->positions, r->positions_len, (r->axes - 1) * r->positions_stride + rows, 4, "rotary positions");
    if (st != SAGE_OK) return st;
    *out = {r->table, r->positions, (int)(r->table_len / (2 * pairs)), (int)(2 * pairs), r->layout, transpose != 0};
    out->axes = (int)r->axes;
    out->positions_stride = (long long)r->positions_stride;
    deal(r->sections, r->axes, pairs, r->dealt != 0,
         [&](uint64_t i, uint64_t a, uint64_t) { out->axis_of[i / 16] |= (uint32_t)a << (i % 16 * 2); });
    for (uint64_t a = 0; a < r->axes; a++) out->sections[a] = (int)r->sections[a];
    return SAGE_OK;
}

template <class R>
sage_status apply(const sage_attention* s, const sage_shape* shape, const R* rotary, const sage_tensor* x,
                  const sage_tensor_mut* out, int32_t transpose) {
    if (!s || !shape || !rotary || !x || !out) return set_error(SAGE_ERR_INVALID, "null argument");
    if (shape->batch == 0 || shape->tokens == 0 || shape->heads == 0) return succeeded();
    uint64_t rows;
    if (__builtin_mul_overflow(shape->batch, shape->tokens, &rows) || rows > I32 || shape->heads > I32)
        return set_error(SAGE_ERR_INVALID, "rotary: %llu x %llu rows of %llu heads do not fit in i32",
                         (u64)shape->batch, (u64)shape->tokens, (u64)shape->heads);
    if (rows > ROWS - 4 || shape->heads > 1ull << 30)
        return set_error(SAGE_ERR_INVALID, "rotary: %llu rows of %llu heads exceed the launch grid", (u64)rows,
                         (u64)shape->heads);
    const uint64_t d = s->head_dim;
    const sage_shape& h = *shape;
    sage_status st = view(x->data, x->len, x->strides, x->dtype, h.batch, h.tokens, h.heads, d, "rotary input");
    if (st == SAGE_OK)
        st = view(out->data, out->len, out->strides, out->dtype, h.batch, h.tokens, h.heads, d, "rotary output");
    if (st == SAGE_OK && x->dtype != out->dtype)
        st = set_error(SAGE_ERR_INVALID, "rotary input and output must share one element type");
    sage::RotaryArgs a{};
    if (st == SAGE_OK) st = checked(rotary, d, rows, transpose, &a.r);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    a.x = rows_of(x);
    a.out = rows_of(out);
    a.batch = (int)shape->batch;
    a.tokens = (int)shape->tokens;
    a.heads = (int)shape->heads;
    a.f16 = x->dtype == SAGE_F16;
    return done(sage::launch_rotary((int)d, a, s->stream), "launch rotary");
}

template <class R>
sage_status append(const sage_attention* s, const sage_cache_shape* shape, const sage_cache* cache,
                   const sage_cache_index* index, const sage_tensor* k, const sage_tensor* v, const R* rotary,
                   const sage_tensor* q, const sage_tensor_mut* q_out) {
    if (!s || !shape || !cache || !index || !k || !v) return set_error(SAGE_ERR_INVALID, "null argument");
    if (!q != !q_out || (q && !rotary))
        return set_error(SAGE_ERR_INVALID, "cache append: queries need an output and a rotary");
    const uint64_t d = s->head_dim;
    sage::AppendArgs a{};
    sage_status st = cache_checked(*shape, d, *cache, *index, &a.c);
    if (st == SAGE_OK) st = view(k, shape->rows, shape->kv_heads, d, "cache append K");
    if (st == SAGE_OK) st = view(v, shape->rows, shape->kv_heads, d, "cache append V");
    if (st == SAGE_OK && q) st = view(q, shape->rows, shape->heads, d, "cache append Q");
    if (st == SAGE_OK && q) st = view(q_out, shape->rows, shape->heads, d, "cache append Q output");
    if (st == SAGE_OK && (k->dtype != v->dtype || (q && (q->dtype != k->dtype || q_out->dtype != k->dtype))))
        st = set_error(SAGE_ERR_INVALID, "Q, K and V must share one element type");
    if (st == SAGE_OK && rotary) st = checked(rotary, d, shape->rows, 0, &a.r);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (shape->rows == 0 || shape->batch == 0) return succeeded();
    a.k = rows_of(k);
    a.v = rows_of(v);
    if (q) {
        a.q = rows_of(q);
        a.q_out = rows_of(q_out);
    }
    a.heads = (int)shape->heads;
    a.f16 = k->dtype == SAGE_F16;
    return done(sage::launch_cache_append((int)d, a, s->stream), "launch cache append");
}

}  // namespace

extern "C" {

sage_status sage_rotary_table(uint64_t rot, uint64_t positions, double base, const sage_rotary_scaling* scaling,
                              float* out, uint64_t out_len) {
    if (!out) return set_error(SAGE_ERR_INVALID, "null argument");
    if (rot < 2 || rot % 2 || rot > 1u << 16)
        return set_error(SAGE_ERR_INVALID, "rotary: %llu rotated channels: an even number from 2", (u64)rot);
    if (!(base > 1.0) || !std::isfinite(base))
        return set_error(SAGE_ERR_INVALID, "rotary: base %g is not over 1", base);
    sage_status st = table_room(positions, rot, out_len);
    Speeds speeds;
    if (st == SAGE_OK) st = speeds.checked(base, scaling, rot);
    if (st != SAGE_OK) return st;
    for (uint64_t i = 0; i < rot / 2; i++) speeds.column(out, rot / 2, i, positions, speeds.of(i, rot));
    return succeeded();
}

sage_status sage_rotary_axes_table(const uint64_t* sections, uint64_t axes, int32_t dealt, int32_t per_axis,
                                   uint64_t positions, double base, const sage_rotary_scaling* scaling, float* out,
                                   uint64_t out_len) {
    if (!sections || !out) return set_error(SAGE_ERR_INVALID, "null argument");
    uint64_t pairs = 0, least = 1u << 15;
    sage_status st = sections_checked(sections, axes, 1u << 15, &pairs);
    if (st != SAGE_OK) return st;
    if (!(base > 1.0) || !std::isfinite(base))
        return set_error(SAGE_ERR_INVALID, "rotary: base %g is not over 1", base);
    for (uint64_t a = 0; a < axes; a++) least = std::min(least, sections[a]);
    st = table_room(positions, 2 * pairs, out_len);
    Speeds speeds;
    if (st == SAGE_OK) st = speeds.checked(base, scaling, 2 * (per_axis ? least : pairs));
    if (st != SAGE_OK) return st;
    deal(sections, axes, pairs, dealt != 0, [&](uint64_t i, uint64_t a, uint64_t j) {
        speeds.column(out, pairs, i, positions, per_axis ? speeds.of(j, 2 * sections[a]) : speeds.of(i, 2 * pairs));
    });
    return succeeded();
}

sage_status sage_rotary_apply(const sage_attention* s, const sage_shape* shape, const sage_rotary* rotary,
                              const sage_tensor* x, const sage_tensor_mut* out, int32_t transpose) {
    return apply(s, shape, rotary, x, out, transpose);
}

sage_status sage_rotary_axes_apply(const sage_attention* s, const sage_shape* shape, const sage_rotary_axes* rotary,
                                   const sage_tensor* x, const sage_tensor_mut* out, int32_t transpose) {
    return apply(s, shape, rotary, x, out, transpose);
}

sage_status sage_cache_sizes(const sage_cache_shape* shape, uint64_t head_dim, uint64_t* codes, uint64_t* scales) {
    if (!shape || !codes || !scales) return set_error(SAGE_ERR_INVALID, "null argument");
    if (head_dim != 64 && head_dim != 128)
        return set_error(SAGE_ERR_INVALID, "sage attention supports head dim 64 or 128, got %llu", (u64)head_dim);
    const sage_status st = shape_checked(*shape);
    if (st != SAGE_OK) return st;
    *codes = code_rows(*shape) * (head_dim / 2);
    *scales = code_rows(*shape) * (head_dim / sage::CACHE_BLOCK);
    return succeeded();
}

sage_status sage_cache_append(const sage_attention* s, const sage_cache_shape* shape, const sage_cache* cache,
                              const sage_cache_index* index, const sage_tensor* k, const sage_tensor* v,
                              const sage_rotary* rotary, const sage_tensor* q, const sage_tensor_mut* q_out) {
    return append(s, shape, cache, index, k, v, rotary, q, q_out);
}

sage_status sage_cache_append_axes(const sage_attention* s, const sage_cache_shape* shape, const sage_cache* cache,
                                   const sage_cache_index* index, const sage_tensor* k, const sage_tensor* v,
                                   const sage_rotary_axes* rotary, const sage_tensor* q, const sage_tensor_mut* q_out) {
    if (!rotary) return set_error(SAGE_ERR_INVALID, "null argument");
    return append(s, shape, cache, index, k, v, rotary, q, q_out);
}

sage_status sage_cache_read(const sage_attention* s, const sage_cache_shape* shape, const sage_cache* cache,
                            const sage_cache_index* index, const sage_tensor_mut* k, const sage_tensor_mut* v) {
    if (!s || !shape || !cache || !index || !k || !v) return set_error(SAGE_ERR_INVALID, "null argument");
    const uint64_t d = s->head_dim;
    sage::ReadArgs a{};
    sage_status st = cache_checked(*shape, d, *cache, *index, &a.c);
    if (st == SAGE_OK) st = view(k, shape->rows, shape->kv_heads, d, "cache read K");
    if (st == SAGE_OK) st = view(v, shape->rows, shape->kv_heads, d, "cache read V");
    if (st == SAGE_OK && k->dtype != v->dtype) st = set_error(SAGE_ERR_INVALID, "K and V must share one element type");
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (shape->rows == 0 || shape->batch == 0) return succeeded();
    a.k = rows_of(k);
    a.v = rows_of(v);
    a.f16 = k->dtype == SAGE_F16;
    return done(sage::launch_cache_read((int)d, a, s->stream), "launch cache read");
}

sage_status sage_cache_workspace_new(const sage_attention* s, const sage_cache_shape* shape,
                                     sage_cache_workspace** out) {
    if (!out) return set_error(SAGE_ERR_INVALID, "null output");
    *out = nullptr;
    if (!s || !shape) return set_error(SAGE_ERR_INVALID, "null argument");
    sage_status st = shape_checked(*shape);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    const sage_cache_shape& h = *shape;
    const sage::CachePlan plan = sage::cache_plan((int)s->head_dim, (int)h.batch, (int)h.rows, (int)h.heads,
                                                  (int)h.kv_heads, (int)h.max_new, (int)(h.max_pages * h.page_tokens));
    // A partial row: D floats, a maximum and a sum.
    uint64_t bytes = 0;
    if (__builtin_mul_overflow(plan.part_rows, (s->head_dim + 2) * 4, &bytes) || bytes > 1ull << 62)
        return set_error(SAGE_ERR_INVALID, "cache workspace needs more than 2^62 bytes");
    sage_cache_workspace* w = new (std::nothrow) sage_cache_workspace{h, s->head_dim, bytes, s->device, plan, nullptr};
    if (!w) return set_error(SAGE_ERR_DEVICE, "out of host memory");
    if (bytes) {
        const hipError_t e = hipMalloc(&w->buf, bytes);
        if (e != hipSuccess) {
            delete w;
            return hip_failed(e, "allocate cache workspace");
        }
    }
    *out = w;
    return succeeded();
}

void sage_cache_workspace_destroy(sage_cache_workspace* ws) {
    if (!ws) return;
    if (ws->buf) (void)hipFree(ws->buf);
    delete ws;
}

uint64_t sage_cache_workspace_bytes(const sage_cache_workspace* ws) { return ws ? ws->bytes : 0; }

sage_status sage_cache_attend(const sage_attention* s, const sage_cache_workspace* ws, const sage_cache* cache,
                              const sage_cache_index* index, const sage_tensor* q, const sage_tensor_mut* out,
                              const sage_cache_options* opts) {
    if (!s || !ws || !cache || !index || !q || !out || !opts) return set_error(SAGE_ERR_INVALID, "null argument");
    if (ws->head_dim != s->head_dim)
        return set_error(SAGE_ERR_INVALID, "workspace was made for head dim %llu, kernels are %llu", (u64)ws->head_dim,
                         (u64)s->head_dim);
    if (ws->device != s->device)
        return set_error(SAGE_ERR_INVALID, "workspace is of device %d, the context of %d", ws->device, s->device);
    const sage_cache_shape& h = ws->shape;
    const uint64_t d = s->head_dim;
    sage::CacheAttnArgs a{};
    sage_status st = cache_checked(h, d, *cache, *index, &a.c);
    if (st == SAGE_OK) st = attend_checked(h, d, q, out, *opts, &a);
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (h.rows == 0 || h.batch == 0 || h.max_new == 0) return succeeded();
    a.splits = ws->plan.chunks ? ws->plan.wgs : 1;
    a.whole = ws->plan.whole;
    a.part_o = static_cast<float*>(ws->buf);
    a.part_ml = ws->buf ? a.part_o + ws->plan.part_rows * d : nullptr;
    return done(sage::launch_cache_attend((int)d, a, ws->plan, s->stream), "launch cache attention");
}

}  // extern "C"
