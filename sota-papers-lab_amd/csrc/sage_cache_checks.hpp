// Checks that the rotary and cache entry points share: views, buffers, shapes,
// indexes and rotary positions, with the refusals' texts.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "sage_cache.hpp"
#include "sage_internal.hpp"

namespace sage {
namespace checks {

using u64 = unsigned long long;
constexpr uint64_t I32 = 2147483647ull;
// Rows below it: at most 64 threads a row in a grid's x, of which a launch takes
// less than 2^32. The rotation's workgroups take four rows each: 2^26 - 4 at most.
constexpr uint64_t ROWS = 1ull << 26;

inline sage_status hip_failed(hipError_t e, const char* what) {
    (void)hipGetLastError();  // reported here, not by the next launch as well
    return set_error(SAGE_ERR_DEVICE, "%s: %s (%s)", what, hipGetErrorName(e), hipGetErrorString(e));
}

inline sage_status done(hipError_t e, const char* what) {
    if (e != hipSuccess) return hip_failed(e, what);
    return succeeded();
}

// The kernels run on the current device; the context's stream and the memory
// it was made for are its own device's.
inline sage_status on_device(const sage_attention* s) {
    int dev = -1;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_failed(e, "current device");
    if (dev != s->device)
        return set_error(SAGE_ERR_INVALID, "the context is of device %d, the current device is %d", s->device, dev);
    return SAGE_OK;
}

inline sage_status in_i32(uint64_t v, const char* what) {
    return v <= I32 ? SAGE_OK : set_error(SAGE_ERR_INVALID, "%s = %llu does not fit in i32", what, (u64)v);
}

inline sage_status buffer(const void* p, uint64_t have, uint64_t need, uintptr_t align, const char* what) {
    if (need == 0) return SAGE_OK;
    if (!p || have < need)
        return set_error(SAGE_ERR_INVALID, "%s: buffer holds %llu elements, needs %llu", what, (u64)(p ? have : 0),
                         (u64)need);
    if (reinterpret_cast<uintptr_t>(p) % align)
        return set_error(SAGE_ERR_INVALID, "%s must start at a %u-byte aligned device address", what, (unsigned)align);
    return SAGE_OK;
}

// A 16-bit view of batch x tokens rows of heads.
inline sage_status view(const void* data, uint64_t len, const sage_strides& st, int32_t dtype, uint64_t batch, uint64_t tokens,
                 uint64_t heads, uint64_t d, const char* what) {
    sage_status r = sage_strides_check(&st, what);
    if (r != SAGE_OK) return r;
    if (dtype != SAGE_BF16 && dtype != SAGE_F16)
        return set_error(SAGE_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
    if (st.token >= 1ull << 62 || st.head >= 1ull << 62 || (batch > 1 && st.batch >= 1ull << 62))
        return set_error(SAGE_ERR_INVALID, "%s: strides exceed 2^62 elements", what);
    return buffer(data, len, sage_strides_extent(&st, batch, tokens, heads, d), 16, what);
}
inline sage_status view(const sage_tensor* t, uint64_t rows, uint64_t heads, uint64_t d, const char* what) {
    const sage_strides st{0, t->strides.token, t->strides.head};
    return view(t->data, t->len, st, t->dtype, 1, rows, heads, d, what);
}
inline sage_status view(const sage_tensor_mut* t, uint64_t rows, uint64_t heads, uint64_t d, const char* what) {
    const sage_strides st{0, t->strides.token, t->strides.head};
    return view(t->data, t->len, st, t->dtype, 1, rows, heads, d, what);
}

template <class T>
RowView rows_of(const T* t) {
    return {static_cast<uint16_t*>(const_cast<void*>(static_cast<const void*>(t->data))), (long long)t->strides.batch,
            (long long)t->strides.token, (long long)t->strides.head};
}

inline sage_status shape_checked(const sage_cache_shape& h) {
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
inline uint64_t code_rows(const sage_cache_shape& h) { return h.pages * h.kv_heads * h.page_tokens; }

// The index of a checked shape, and the sizes in out; the pool's buffers stay null.
inline sage_status index_checked(const sage_cache_shape& h, const sage_cache_index& i, CacheDev* out) {
    sage_status st = buffer(i.starts, i.starts_len, h.batch + 1, 4, "cache starts");
    if (st == SAGE_OK) st = buffer(i.lengths, i.lengths_len, h.batch, 4, "cache lengths");
    if (st == SAGE_OK) st = buffer(i.page_table, i.page_table_len, h.batch * h.max_pages, 4, "cache page table");
    if (st != SAGE_OK) return st;
    int shift = 4;
    while ((1ull << shift) < h.page_tokens) shift++;
    *out = {nullptr, nullptr, nullptr, nullptr, i.starts, i.lengths, i.page_table, (int)h.batch,
            (int)h.rows, (int)h.kv_heads, (int)h.pages, shift, (int)h.max_pages};
    return SAGE_OK;
}

inline sage_status cache_checked(const sage_cache_shape& h, uint64_t d, const sage_cache& c, const sage_cache_index& i,
                                 CacheDev* out) {
    sage_status st = shape_checked(h);
    const uint64_t codes = st == SAGE_OK ? code_rows(h) * (d / 2) : 0, scales = codes / (CACHE_BLOCK / 2);
    if (st == SAGE_OK) st = buffer(c.k_codes, c.codes_len, codes, 16, "cache K codes");
    if (st == SAGE_OK) st = buffer(c.k_scales, c.scales_len, scales, 16, "cache K scales");
    if (st == SAGE_OK) st = buffer(c.v_codes, c.codes_len, codes, 16, "cache V codes");
    if (st == SAGE_OK) st = buffer(c.v_scales, c.scales_len, scales, 16, "cache V scales");
    if (st == SAGE_OK) st = index_checked(h, i, out);
    if (st != SAGE_OK) return st;
    out->k_codes = c.k_codes, out->k_scales = c.k_scales, out->v_codes = c.v_codes, out->v_scales = c.v_scales;
    return SAGE_OK;
}

// An attention's queries, output and options, into `a`.
inline sage_status attend_checked(const sage_cache_shape& h, uint64_t d, const sage_tensor* q, const sage_tensor_mut* out,
                                  const sage_cache_options& opts, CacheAttnArgs* a) {
    sage_status st = view(q, h.rows, h.heads, d, "Q");
    if (st == SAGE_OK) st = view(out, h.rows, h.heads, d, "output");
    if (st != SAGE_OK) return st;
    a->q = rows_of(q);
    a->out = rows_of(out);
    a->heads = (int)h.heads;
    a->group = (int)(h.heads / h.kv_heads);
    a->max_new = (int)h.max_new;
    a->causal = opts.causal != 0;
    a->q_f16 = q->dtype == SAGE_F16;
    a->out_f16 = out->dtype == SAGE_F16;
    const float scale = opts.has_softmax_scale ? opts.softmax_scale : (float)(1.0 / std::sqrt((double)d));
    // A scale of 0 becomes the least normal float: every weight is 1 still, and
    // the -infinity of a masked logit stays what it is.
    a->qk_mul = std::max(std::fabs(scale) * 1.44269504088896340736f, 1.17549435e-38f);
    if (scale != scale) a->qk_mul = scale;
    a->q_sign = std::signbit(scale) ? 0x80008000u : 0u;
    return SAGE_OK;
}

}  // namespace checks
}  // namespace sage
