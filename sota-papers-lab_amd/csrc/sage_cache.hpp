// Parameter blocks of the rotary and paged-cache kernels, and what they share:
// the row -> sequence lookup, the page lookup and the 4-bit codec.
//
// Cache layout (include/sage_hip.h): for each page and KV head, page_tokens
// rows of D / 2 code bytes and, apart, of D / 32 scale bytes. One head's page is
// contiguous, so that the attention of one KV head streams it in whole lines.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sage_device.hpp"

namespace sage {

constexpr int CACHE_BLOCK = 32;  // channels a scale (E8M0 block of the OCP MX formats)

// A [row][head][dim] view; batch strides where the entry point has a batch.
struct RowView {
    uint16_t* p;
    long long sb, st, sh;
};

struct RotaryDev {
    const float* table;  // [table_rows][rot / 2][2]
    const int* positions;
    int table_rows, rot, layout, transpose;
};

// Device view of sage_cache, sage_cache_index and sage_cache_shape.
struct CacheDev {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    const int *starts, *lengths, *page_table;
    int batch, rows, kv_heads, pages, page_shift, max_pages;
};

struct RotaryArgs {
    RowView x, out;
    RotaryDev r;
    int batch, tokens, heads, f16;
};

struct AppendArgs {
    RowView k, v, q, q_out;  // q.p null: no queries
    RotaryDev r;             // table null: no rotation
    CacheDev c;
    int heads, f16;
};

struct ReadArgs {
    RowView k, v;
    CacheDev c;
    int f16;
};

// One attention call. part_o, part_ml: the partial outputs of split sequences,
// D floats and a (maximum, sum) pair each.
struct CacheAttnArgs {
    RowView q, out;
    CacheDev c;
    float* part_o;
    float* part_ml;
    float qk_mul;     // |softmax scale| * log2(e), over 0
    uint32_t q_sign;  // 0x80008000 under a negative scale: the queries' signs
    int heads, group, max_new, causal, q_f16, out_f16;
    int splits;  // chunks: workgroups that a sequence's keys are split over, at most
    int whole;   // few rows: a workgroup a unit
};

hipError_t launch_rotary(int head_dim, const RotaryArgs& a, hipStream_t s);
hipError_t launch_cache_append(int head_dim, const AppendArgs& a, hipStream_t s);
hipError_t launch_cache_read(int head_dim, const ReadArgs& a, hipStream_t s);
// How an attention call of these sizes runs: the chunk kernel, its keys split
// over wgs workgroups at most, or the one for few rows, in whole units (wide:
// of eight waves) or on wgs workgroups; and the partial outputs that the
// workspace holds. max_tokens: most tokens that the page table holds.
struct CachePlan {
    bool chunks, whole;
    int wgs;
    uint64_t part_rows;
    bool wide;
};
CachePlan cache_plan(int head_dim, int batch, int rows, int heads, int kv_heads, int max_new, int max_tokens);
hipError_t launch_cache_attend(int head_dim, const CacheAttnArgs& a, const CachePlan& plan, hipStream_t s);

// The index lookups, host and device: tests/cpp/cache_host.cpp runs them on bad
// indexes on the CPU.

// The code row of a token of (page, KV head): byte offset / (D / 2) of its
// codes and / (D / 32) of its scales.
__host__ __device__ __forceinline__ long long cache_row(const CacheDev& c, int page, int head, int token) {
    return (((long long)page * c.kv_heads + head) << c.page_shift) + token;
}

// The page of slot t of sequence b, or -1 where the slot holds nothing.
__host__ __device__ __forceinline__ int cache_page(const CacheDev& c, int b, int t) {
    const int col = t >> c.page_shift;
    if (t < 0 || col >= c.max_pages) return -1;
    const int page = c.page_table[(long long)b * c.max_pages + col];
    return (unsigned)page < (unsigned)c.pages ? page : -1;
}

// The sequence of a row: the last b with starts[b] <= row; -1 for rows outside
// all sequences.
__host__ __device__ __forceinline__ int sequence_of(const CacheDev& c, int row) {
    int lo = 0, hi = c.batch + 1;  // starts[< lo] <= row < starts[>= hi]
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (c.starts[mid] <= row)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo == 0 || lo > c.batch ? -1 : lo - 1;
}

// The slot of a row of sequence b, or -1 where it lies before slot 0 or past
// 31 bits.
__host__ __device__ __forceinline__ int slot_of(const CacheDev& c, int b, int row) {
    const long long n = (long long)c.starts[b + 1] - c.starts[b];
    const long long t = c.lengths[b] - n + ((long long)row - c.starts[b]);
    return t < 0 || t > 0x7fffffff ? -1 : (int)t;
}

// What one sequence's index says, in range: n rows from `start` on, of which
// row j sees slots up to diff + j under a causal mask, and len slots at all.
struct SequenceIndex {
    long long start, diff;
    int n, len;
    // Slots that row j sees: all below the limit.
    __host__ __device__ __forceinline__ int limit(int j, int causal) const {
        const long long v = diff + j + 1;
        return causal && v < len ? (v < 0 ? 0 : (int)v) : len;
    }
};
__host__ __device__ __forceinline__ SequenceIndex sequence_index(const CacheDev& c, int b, int max_new) {
    SequenceIndex s;
    s.start = c.starts[b];
    const long long n = c.starts[b + 1] - s.start, raw = c.lengths[b], most = (long long)c.max_pages << c.page_shift;
    s.diff = raw - n;
    s.n = (int)(n < 0 ? 0 : n < max_new ? n : max_new);
    s.len = (int)(raw < 0 ? 0 : raw < most ? raw : most);
    return s;
}

}  // namespace sage
