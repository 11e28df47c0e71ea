// C ABI of the rotary and paged-cache entry points (include/sage_hip.h): every
// check before any launch, then the launch on the context's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "sage_cache.hpp"
#include "sage_internal.hpp"

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

using u64 = unsigned long long;
constexpr uint64_t I32 = 2147483647ull;
// Rows below it: at most 64 threads a row in a grid's x, of which a launch takes
// less than 2^32. The rotation's workgroups take four rows each: 2^26 - 4 at most.
constexpr uint64_t ROWS = 1ull << 26;

sage_status hip_failed(hipError_t e, const char* what) {
    return set_error(SAGE_ERR_DEVICE, "%s: %s (%s)", what, hipGetErrorName(e), hipGetErrorString(e));
}

sage_status done(hipError_t e, const char* what) {
    if (e != hipSuccess) return hip_failed(e, what);
    return succeeded();
}

// The kernels run on the current device; the context's stream and the memory
// it was made for are its own device's.
sage_status on_device(const sage_attention* s) {
    int dev = -1;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_failed(e, "current device");
    if (dev != s->device)
        return set_error(SAGE_ERR_INVALID, "the context is of device %d, the current device is %d", s->device, dev);
    return SAGE_OK;
}

sage_status in_i32(uint64_t v, const char* what) {
    return v <= I32 ? SAGE_OK : set_error(SAGE_ERR_INVALID, "%s = %llu does not fit in i32", what, (u64)v);
}

sage_status buffer(const void* p, uint64_t have, uint64_t need, uintptr_t align, const char* what) {
    if (need == 0) return SAGE_OK;
    if (!p || have < need)
        return set_error(SAGE_ERR_INVALID, "%s: buffer holds %llu elements, needs %llu", what, (u64)(p ? have : 0),
                         (u64)need);
    if (reinterpret_cast<uintptr_t>(p) % align)
        return set_error(SAGE_ERR_INVALID, "%s must start at a %u-byte aligned device address", what, (unsigned)align);
    return SAGE_OK;
}

// A 16-bit view of batch x tokens rows of heads.
sage_status view(const void* data, uint64_t len, const sage_strides& st, int32_t dtype, uint64_t batch, uint64_t tokens,
                 uint64_t heads, uint64_t d, const char* what) {
    sage_status r = sage_strides_check(&st, what);
    if (r != SAGE_OK) return r;
    if (dtype != SAGE_BF16 && dtype != SAGE_F16)
        return set_error(SAGE_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
    if (st.token >= 1ull << 62 || st.head >= 1ull << 62 || (batch > 1 && st.batch >= 1ull << 62))
        return set_error(SAGE_ERR_INVALID, "%s: strides exceed 2^62 elements", what);
    return buffer(data, len, sage_strides_extent(&st, batch, tokens, heads, d), 16, what);
}
sage_status view(const sage_tensor* t, uint64_t rows, uint64_t heads, uint64_t d, const char* what) {
    const sage_strides st{0, t->strides.token, t->strides.head};
    return view(t->data, t->len, st, t->dtype, 1, rows, heads, d, what);
}
sage_status view(const sage_tensor_mut* t, uint64_t rows, uint64_t heads, uint64_t d, const char* what) {
    const sage_strides st{0, t->strides.token, t->strides.head};
    return view(t->data, t->len, st, t->dtype, 1, rows, heads, d, what);
}

template <class T>
sage::RowView rows_of(const T* t) {
    return {static_cast<uint16_t*>(const_cast<void*>(static_cast<const void*>(t->data))), (long long)t->strides.batch,
            (long long)t->strides.token, (long long)t->strides.head};
}

sage_status rotary_checked(const sage_rotary* r, uint64_t d, uint64_t rows, int transpose, sage::RotaryDev* out) {
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

sage_status shape_checked(const sage_cache_shape& h) {
    if (h.kv_heads == 0 || h.heads == 0 || h.heads % h.kv_heads)
        return set_error(SAGE_ERR_INVALID, "%llu query heads are not a multiple of %llu KV heads", (u64)h.heads,
                         (u64)h.kv_heads);
    if (h.page_tokens < 16 || h.page_tokens > 256 || (h.page_tokens & (h.page_tokens - 1)))
        return set_error(SAGE_ERR_INVALID, "cache: pages of %llu tokens (16, 32, 64, 128 or 256 are supported)",
                         (u64)h.page_tokens);
    if (h.pages == 0 || h.max_pages == 0)
        return set_error(SAGE_ERR_INVALID, "cache: %llu pages in the pool, %llu columns in the page table",
                         (u64)h.pages, (u64)h.max_pages);
    sage_status st = in_i32(h.pages, "cache pages");
    if (st == SAGE_OK) st = in_i32(h.rows, "cache rows");
    if (st != SAGE_OK) return st;
    if (h.max_pages > (1ull << 30) / h.page_tokens)
        return set_error(SAGE_ERR_INVALID, "cache: %llu pages of %llu tokens exceed 2^30 tokens a sequence",
                         (u64)h.max_pages, (u64)h.page_tokens);
    if (h.rows >= ROWS)
        return set_error(SAGE_ERR_INVALID, "cache: %llu rows exceed the launch grid", (u64)h.rows);
    // Launch grids: x below 2^24 workgroups, append's K, V and query heads and the
    // joins' KV heads in y, the batch in z.
    if (h.batch > 65535 || h.heads > 65535 || 2 * h.kv_heads + h.heads > 65535)
        return set_error(SAGE_ERR_INVALID, "cache: %llu sequences of %llu and %llu heads exceed the launch grid",
                         (u64)h.batch, (u64)h.heads, (u64)h.kv_heads);
    // A tile is 16 columns or more; 128 where there are many.
    const uint64_t group = h.heads / h.kv_heads;
    if (h.max_new > I32 / 64 / group || (h.max_new * group + 127) / 128 * h.kv_heads >= 1ull << 24)
        return set_error(SAGE_ERR_INVALID, "cache: %llu new rows of %llu heads a KV head exceed the launch grid",
                         (u64)h.max_new, (u64)group);
    return SAGE_OK;
}

// Code rows of a pool, at most 2^31 pages x 65535 heads x 256 tokens: no wrap.
uint64_t code_rows(const sage_cache_shape& h) { return h.pages * h.kv_heads * h.page_tokens; }

sage_status cache_checked(const sage_cache_shape& h, uint64_t d, const sage_cache& c, const sage_cache_index& i,
                          sage::CacheDev* out) {
    sage_status st = shape_checked(h);
    const uint64_t codes = st == SAGE_OK ? code_rows(h) * (d / 2) : 0, scales = codes / (sage::CACHE_BLOCK / 2);
    if (st == SAGE_OK) st = buffer(c.k_codes, c.codes_len, codes, 16, "cache K codes");
    if (st == SAGE_OK) st = buffer(c.k_scales, c.scales_len, scales, 16, "cache K scales");
    if (st == SAGE_OK) st = buffer(c.v_codes, c.codes_len, codes, 16, "cache V codes");
    if (st == SAGE_OK) st = buffer(c.v_scales, c.scales_len, scales, 16, "cache V scales");
    if (st == SAGE_OK) st = buffer(i.starts, i.starts_len, h.batch + 1, 4, "cache starts");
    if (st == SAGE_OK) st = buffer(i.lengths, i.lengths_len, h.batch, 4, "cache lengths");
    if (st == SAGE_OK) st = buffer(i.page_table, i.page_table_len, h.batch * h.max_pages, 4, "cache page table");
    if (st != SAGE_OK) return st;
    int shift = 4;
    while ((1ull << shift) < h.page_tokens) shift++;
    *out = {c.k_codes, c.k_scales, c.v_codes, c.v_scales, i.starts, i.lengths, i.page_table, (int)h.batch,
            (int)h.rows, (int)h.kv_heads, (int)h.pages, shift, (int)h.max_pages};
    return SAGE_OK;
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
    sage_status st = in_i32(positions, "rotary positions");
    if (st == SAGE_OK && out_len < positions * rot)
        st = set_error(SAGE_ERR_INVALID, "rotary table: buffer holds %llu elements, needs %llu", (u64)out_len,
                       (u64)(positions * rot));
    if (st != SAGE_OK) return st;
    const int kind = scaling ? scaling->kind : SAGE_ROTARY_NONE;
    const double f = kind == SAGE_ROTARY_NONE ? 1.0 : scaling->factor, pi = 3.14159265358979323846;
    if (kind < SAGE_ROTARY_NONE || kind > SAGE_ROTARY_YARN)
        return set_error(SAGE_ERR_INVALID, "rotary: unknown scaling %d", kind);
    if (!(f >= 1.0) || !std::isfinite(f))
        return set_error(SAGE_ERR_INVALID, "rotary: scaling factor %g is not 1 or more", f);
    double attention = scaling && scaling->attention != 0.0 ? scaling->attention : 1.0, fast = 0, slow = 0;
    if (!std::isfinite(attention)) return set_error(SAGE_ERR_INVALID, "rotary: attention factor %g", attention);
    if (kind == SAGE_ROTARY_NTK) {
        if (rot < 4) return set_error(SAGE_ERR_INVALID, "rotary: NTK scaling needs 4 rotated channels or more");
        base *= std::pow(f, (double)rot / (double)(rot - 2));
    }
    if (kind == SAGE_ROTARY_YARN) {
        fast = scaling->beta_fast != 0.0 ? scaling->beta_fast : 32.0;
        slow = scaling->beta_slow != 0.0 ? scaling->beta_slow : 1.0;
        if (!(scaling->original > 0.0) || !std::isfinite(scaling->original) || !(slow < fast) || !std::isfinite(fast))
            return set_error(SAGE_ERR_INVALID, "rotary: YaRN scaling of %g positions between %g and %g turns",
                             scaling->original, slow, fast);
        if (scaling->attention == 0.0) attention = 0.1 * std::log(f) + 1.0;
    }
    for (uint64_t i = 0; i < rot / 2; i++) {
        double w = std::pow(base, -2.0 * (double)i / (double)rot);
        if (kind == SAGE_ROTARY_LINEAR) w /= f;
        if (kind == SAGE_ROTARY_YARN) {
            // Peng et al., "YaRN: Efficient Context Window Extension of Large Language
            // Models", 2023: pairs that turn often keep their angle, slow ones are interpolated.
            const double turns = scaling->original * w / (2.0 * pi);
            const double g = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            w = g * w + (1.0 - g) * w / f;
        }
        for (uint64_t p = 0; p < positions; p++) {
            const double a = (double)p * w;
            out[(p * (rot / 2) + i) * 2] = (float)(attention * std::cos(a));
            out[(p * (rot / 2) + i) * 2 + 1] = (float)(attention * std::sin(a));
        }
    }
    return succeeded();
}

sage_status sage_rotary_apply(const sage_attention* s, const sage_shape* shape, const sage_rotary* rotary,
                              const sage_tensor* x, const sage_tensor_mut* out, int32_t transpose) {
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
    if (st == SAGE_OK) st = rotary_checked(rotary, d, rows, transpose, &a.r);
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
    if (st == SAGE_OK && rotary) st = rotary_checked(rotary, d, shape->rows, 0, &a.r);
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
    if (st == SAGE_OK) st = view(q, h.rows, h.heads, d, "Q");
    if (st == SAGE_OK) st = view(out, h.rows, h.heads, d, "output");
    if (st == SAGE_OK) st = on_device(s);
    if (st != SAGE_OK) return st;
    if (h.rows == 0 || h.batch == 0 || h.max_new == 0) return succeeded();
    a.q = rows_of(q);
    a.out = rows_of(out);
    a.heads = (int)h.heads;
    a.group = (int)(h.heads / h.kv_heads);
    a.max_new = (int)h.max_new;
    a.causal = opts->causal != 0;
    a.q_f16 = q->dtype == SAGE_F16;
    a.out_f16 = out->dtype == SAGE_F16;
    const float scale = opts->has_softmax_scale ? opts->softmax_scale : (float)(1.0 / std::sqrt((double)d));
    // A scale of 0 becomes the least normal float: every weight is 1 still, and
    // the -infinity of a masked logit stays what it is.
    a.qk_mul = std::max(std::fabs(scale) * 1.44269504088896340736f, 1.17549435e-38f);
    if (scale != scale) a.qk_mul = scale;
    a.q_sign = std::signbit(scale) ? 0x80008000u : 0u;
    a.splits = ws->plan.chunks ? ws->plan.wgs : 1;
    a.whole = ws->plan.whole;
    a.part_o = static_cast<float*>(ws->buf);
    a.part_ml = ws->buf ? a.part_o + ws->plan.part_rows * d : nullptr;
    return done(sage::launch_cache_attend((int)d, a, ws->plan, s->stream), "launch cache attention");
}

}  // extern "C"
