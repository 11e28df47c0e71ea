// What the attention kernels over the paged cache share (gfx950): conversions, the
// layout of V in LDS, page lookups, the joins of split keys, and the lists of
// picked pages.
#pragma once

#include <type_traits>

#include "sage_cache.hpp"

namespace sage {

namespace {

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int TOKENS = 64;  // tokens of a wave's step
constexpr int MAX_SPLITS = 256;
// The reference m of the softmax follows the maximum only where that is 2^8
// past it: the fp32 sums have room for that, and rescaling them becomes rare.
constexpr float SLACK = 8.0f;
constexpr float NEG_INF = -__builtin_inff();
// V's blocks from this scale on (2^126: a code of 4 is past every 16- and 32-bit
// type) are NaN as 255 is: an infinity of a masked token would reach the
// rows that do not see it as 0 * inf.
constexpr uint32_t V_NAN = 253;

// Codes 2 which and 2 which + 1 of a dword times s, as bf16 or fp16 (H16).
template <bool H16>
__device__ __forceinline__ uint32_t cvt2(uint32_t codes, float s, int which) {
    if constexpr (H16) {
        h2 r;
        switch (which) {
            case 0: r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 0); break;
            case 1: r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 1); break;
            case 2: r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 2); break;
            default: r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 3);
        }
        return __builtin_bit_cast(uint32_t, r);
    }
    bf2 r;
    switch (which) {
        case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0); break;
        case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1); break;
        case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2); break;
        default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
    }
    return __builtin_bit_cast(uint32_t, r);
}

// Eight channels of one code dword.
template <bool H16 = false>
__device__ __forceinline__ uint4 decode8(uint32_t codes, float s) {
    return make_uint4(cvt2<H16>(codes, s, 0), cvt2<H16>(codes, s, 1), cvt2<H16>(codes, s, 2),
                      cvt2<H16>(codes, s, 3));
}

// Eight values as bf16, or as two bf16 parts: the nearest and the rest's.
template <int PARTS>
__device__ __forceinline__ void parts_of(const float* f, bf8 (&p)[PARTS]) {
    uint32_t w[PARTS][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[0][i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        if (PARTS == 2)
            w[PARTS - 1][i] = pack_bf16x2(f[2 * i] - __uint_as_float(w[0][i] << 16),
                                          f[2 * i + 1] - __uint_as_float(w[0][i] & 0xffff0000u));
    }
#pragma unroll
    for (int k = 0; k < PARTS; k++) p[k] = __builtin_bit_cast(bf8, make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]));
}

// Eight channels of a query, negated under a negative softmax scale (so that
// the greatest logit is the greatest product).
__device__ __forceinline__ uint4 signed_q(uint4 x, uint32_t sign) {
    return make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
}
__device__ __forceinline__ uint4 load_q(const uint16_t* p, uint32_t sign) {
    return signed_q(*reinterpret_cast<const uint4*>(p), sign);
}

// Maximum and sum over the four lanes of a column (lanes 16 apart).
__device__ __forceinline__ float col_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Maximum over the aligned LANES (8 or 16) lanes of a row, in each of them.
template <int LANES>
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    return LANES > 8 ? fmaxf(v, dpp<0x140>(v)) : v;
}
__device__ __forceinline__ uint32_t col_or(uint32_t v) {
    auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = r[0] | r[1];
    r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return r[0] | r[1];
}

// A lane's value, scalar.
__device__ __forceinline__ long long uniform(long long v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
    return (long long)((uint64_t)hi << 32 | lo);
}

// A sequence's pages as a wave walks it: 64 columns of the page table, one a
// lane, loaded at once and read by lane index. Looked up one by one, each id is
// a load in front of the loads that need it, and waiting for it waits for
// all that are in flight (64 ragged sequences of up to 16384 tokens, 32/8 heads
// of 128: 173 us, with the window 152).
struct Pages {
    const int* table;  // the sequence's row
    int cols, pages, shift, lane;
    int base, ids;
    __device__ __forceinline__ Pages(const CacheDev& c, int b, int lane_, int t)
        : table(c.page_table + (long long)b * c.max_pages), cols(c.max_pages), pages(c.pages), shift(c.page_shift),
          lane(lane_) {
        fill(t >> shift);
    }
    __device__ __forceinline__ void fill(int col) {
        base = col;
        const int at = col + lane;
        const int id = at < cols ? table[at] : -1;
        ids = (unsigned)id < (unsigned)pages ? id : -1;
        asm volatile("" : "+v"(ids));  // waited for here, once a window, not at every use
    }
    // The page of slot t (of the window's first column or behind it), or -1.
    __device__ __forceinline__ int of(int t) {
        const int col = t >> shift;
        if (col - base >= 64) fill(col);
        return __builtin_amdgcn_readlane(ids, col - base);
    }
};

// Tokens of one of the chunk kernel's splits of a sequence of len tokens: whole tiles.
__device__ __forceinline__ int split_tokens(int len, int splits) {
    return ((len + splits - 1) / splits + TOKENS - 1) / TOKENS * TOKENS;
}

// Byte of half h (eight channels) of 16-channel unit u of a token's bf16 V row
// in LDS. LDS serves 128 bytes a clock: the units of a row are permuted by the
// token, so that the four tokens that 16 lanes of a transposing read take meet
// all of them, and the halves of some are swapped, so that what eight lanes
// write at once does too.
template <int D>
__device__ __forceinline__ int unit_at(int tok, int u, int h) {
    const int f = D == 128 ? tok & 7 : tok & 3, s = D == 128 ? u >> 2 & 1 : (tok ^ tok >> 1) & 1;
    return tok * (D * 2) + ((u ^ f) << 5) + ((h ^ s) << 4);
}

// Eight tokens of a lane's channel from two transposing reads, of four tokens
// each, at v and `on` bytes behind it.
__device__ __forceinline__ bf8 read_v(const uint8_t* v, int on) {
    typedef __attribute__((address_space(3))) s4* lds_ptr;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(v));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(v + on));
    return __builtin_bit_cast(bf8, (s8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Eight channels of an output row: the sums over the softmax's.
__device__ __forceinline__ void store_row(const CacheAttnArgs& a, long long row, int head, int ch, const float* f,
                                          float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = f[2 * i] * inv, y = f[2 * i + 1] * inv;
        w[i] = a.out_f16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
    }
    *reinterpret_cast<uint4*>(a.out.p + row * a.out.st + head * a.out.sh + ch) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Parts first .. first + parts - 1 of one column joined by a group of D / 8
// lanes, eight channels a lane (ch); or, with SHARE, by all the groups of a
// workgroup together (the first has the result): each sums the parts that fall
// to it in their order and the groups' sums are added in theirs, so the same
// call gives the same bits. at(p): part p's place. Returns the softmax's sum.
template <int D, bool SHARE, class At>
__device__ __forceinline__ float join_parts(const CacheAttnArgs& a, int parts, int ch, At at, float (&out)[8]) {
    constexpr int LANES = D / 8, GROUPS = 256 / LANES;
    __shared__ float sums[SHARE ? GROUPS : 1][D + 4], ls[GROUPS];
    const f2* ml = reinterpret_cast<const f2*>(a.part_ml);
    const int grp = threadIdx.x / LANES;
    // The maximum over all parts, then this group's share of the sums.
    float m = NEG_INF, l = 0.0f;
    for (int p = threadIdx.x % LANES; p < parts; p += LANES) m = fmaxf(m, ml[at(p)].x);
    m = row_max<LANES>(m);
    const float base = m == NEG_INF ? 0.0f : m;
    f4 f[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
#pragma unroll 4
    for (int p = SHARE ? grp : 0; p < parts; p += SHARE ? GROUPS : 1) {
        const f2 s = ml[at(p)];
        const f4* o = reinterpret_cast<const f4*>(a.part_o + at(p) * D + ch);
        const float w = __builtin_amdgcn_exp2f(s.x - base);
        l += w * s.y;
        f[0] += o[0] * w;
        f[1] += o[1] * w;
    }
    if (SHARE) {
        *reinterpret_cast<f4*>(&sums[SHARE ? grp : 0][ch]) = f[0];
        *reinterpret_cast<f4*>(&sums[SHARE ? grp : 0][ch + 4]) = f[1];
        ls[grp] = l;
        __syncthreads();
        l = 0.0f, f[0] = f[1] = f4{0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            l += ls[g];
            f[0] += *reinterpret_cast<const f4*>(&sums[SHARE ? g : 0][ch]);
            f[1] += *reinterpret_cast<const f4*>(&sums[SHARE ? g : 0][ch + 4]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) out[i] = f[i / 4][i % 4];
    return l;
}

// ---- Picked pages ----
//
// The pages that a unit's rows have picked (sage_cache_attend_picked), one behind
// the other, in place of a sequence's own: the tokens of a unit are those of the
// pages that any of its rows picked, ascending, and each page carries the rows that
// did. 16 columns of a group of four heads are four rows, whose picks share much: a
// page is read and converted once for all of them, and never costs more than the
// rows' own would, whose columns would fill a tile as wide.
struct Entries {
    uint32_t *col, *rows;  // the page table's column, and the rows of the unit that picked it, a bit each
    int* page;             // the pool's page, or -1
    int count;
};

// LDS of a unit of `cols` columns: the table's columns as bits, how many are set before each word,
// and the entries. rows: of a unit, at most.
__host__ __device__ __forceinline__ int unit_rows(int cols, int group, int max_new) {
    const int rows = (cols + group - 2) / group + 1;
    return rows < max_new ? rows : max_new;
}
__host__ __device__ __forceinline__ int pick_words(int max_pages) { return (max_pages + 31) / 32; }
__host__ __device__ __forceinline__ int pick_entries(int cols, int top, int group, int max_new, int max_pages) {
    const int most = unit_rows(cols, group, max_new) * top;
    return most < max_pages ? most : max_pages;
}
__host__ __device__ __forceinline__ unsigned pick_lds_bytes(int cols, int top, int group, int max_new, int max_pages) {
    return 4u * (2 * pick_words(max_pages) + 3 * pick_entries(cols, top, group, max_new, max_pages));
}

// The entries of rows j0 .. j0 + rows - 1 of sequence b, whose columns are below `pages`.
// All W waves of the workgroup together; COLS columns a unit.
template <int W, int COLS>
__device__ __forceinline__ Entries entries_of(const CacheAttnArgs& a, const SequenceIndex& seq, int b, int kvh, int j0,
                                              int rows, int pages, uint32_t* lds) {
    const CacheDev& c = a.c;
    const int words = pick_words(pages), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int most = pick_entries(COLS, a.top, a.group, a.max_new, c.max_pages);
    uint32_t *bits = lds, *before = bits + pick_words(c.max_pages);
    Entries e{before + pick_words(c.max_pages), nullptr, nullptr, 0};
    e.rows = e.col + most;
    e.page = reinterpret_cast<int*>(e.rows + most);
    __shared__ int found[W], odd[W];
    const int* table = c.page_table + (long long)b * c.max_pages;
    auto page_at = [&](int col) {
        const int id = table[col];
        return (unsigned)id < (unsigned)c.pages ? id : -1;
    };
    // Row r's i-th column, or -1.
    auto picked = [&](int r, int i) {
        const long long row = seq.start + j0 + r;
        if (row < 0 || row >= c.rows) return -1;
        const int col = a.picked[(row * c.kv_heads + kvh) * a.top + i];
        return (unsigned)col < (unsigned)pages ? col : -1;
    };
    if (rows == 1) {
        // One row's list as it is, if it ascends, with nothing behind a -1.
        int n = 0;
        bool out_of_order = false;
        for (int i0 = 0; i0 < a.top; i0 += 64 * W) {
            const int i = i0 + (int)threadIdx.x, col = i < a.top ? picked(0, i) : -1;
            const int last = i > 0 && i < a.top ? picked(0, i - 1) : -1;
            if (col >= 0) {
                out_of_order |= i > 0 && last >= col;
                out_of_order |= i > 0 && last < 0;
                const int at = min(i, pages - 1);
                e.col[at] = col;
                e.rows[at] = 1;
                e.page[at] = page_at(col);
            }
            n += __builtin_popcountll(__ballot(col >= 0));
        }
        const bool wrong = __any(out_of_order);
        if (lane == 0) found[wave] = n, odd[wave] = wrong;
        __syncthreads();
        bool any = false;
#pragma unroll
        for (int w = 0; w < W; w++) e.count += found[w], any = any || odd[w];
        if (!any) return e;
        __syncthreads();
        e.count = 0;
    }
    // A thread's first KEEP columns and their pages stay in registers from the first look to the last.
    constexpr int KEEP = 2;
    int kept[KEEP], ids[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const int i = threadIdx.x + k * 64 * W;
        kept[k] = i < rows * a.top ? picked(i / a.top, i % a.top) : -1;
    }
    for (int i = threadIdx.x; i < words; i += 64 * W) bits[i] = 0;
    __syncthreads();
    auto mark = [&](int col) {
        if (col >= 0) atomicOr(&bits[col >> 5], 1u << (col & 31));
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        mark(kept[k]);
        ids[k] = kept[k] >= 0 ? page_at(kept[k]) : -1;
    }
    for (int i = threadIdx.x + KEEP * 64 * W; i < rows * a.top; i += 64 * W) mark(picked(i / a.top, i % a.top));
    __syncthreads();
    // A run of words a thread.
    const int run = (words + 64 * W - 1) / (64 * W), w0 = min(words, (int)threadIdx.x * run), w1 = min(words, w0 + run);
    int mine = 0;
    for (int w = w0; w < w1; w++) mine += __builtin_popcount(bits[w]);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(upto, d);
        if (lane >= d) upto += x;
    }
    if (lane == 63) found[wave] = upto;
    __syncthreads();
    int at = upto - mine;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w < wave) at += found[w];
        e.count += found[w];
    }
    for (int w = w0; w < w1; w++) {
        before[w] = at;
        for (uint32_t x = bits[w]; x; x &= x - 1, at++) {
            e.col[at] = (uint32_t)(w * 32 + __builtin_ctz(x));
            e.rows[at] = 0;
        }
    }
    __syncthreads();
    auto note = [&](int r, int col, int id) {
        if (col < 0) return;
        const int place = before[col >> 5] + __builtin_popcount(bits[col >> 5] & ((1u << (col & 31)) - 1));
        atomicOr(&e.rows[place], 1u << r);
        e.page[place] = id;  // (every row that picked it writes the same)
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) note((threadIdx.x + k * 64 * W) / a.top, kept[k], ids[k]);
    for (int i = threadIdx.x + KEEP * 64 * W; i < rows * a.top; i += 64 * W) {
        const int col = picked(i / a.top, i % a.top);
        note(i / a.top, col, col >= 0 ? page_at(col) : -1);
    }
    __syncthreads();
    return e;
}

// The entries as a wave walks them, 64 at a time, as Pages does a table's columns.
struct Walk {
    Entries e;
    int shift, lane, base, ids;
    uint32_t cols, rows;
    __device__ __forceinline__ Walk(const Entries& e_, int shift_, int lane_, int t) : e(e_), shift(shift_), lane(lane_) {
        fill(t >> shift);
    }
    __device__ __forceinline__ void fill(int i) {
        base = i;
        const int at = i + lane;
        const bool in = at < e.count;
        ids = in ? e.page[at] : -1;
        cols = in ? e.col[at] : 0;
        rows = in ? e.rows[at] : 0;
        asm volatile("" : "+v"(ids), "+v"(cols), "+v"(rows));  // waited for here, once a window
    }
    // The page of token t of the list, or -1, its slot and the rows that see its page.
    __device__ __forceinline__ int of(int t, int& slot, uint32_t& rows_of) {
        const int i = t >> shift;
        if (i - base >= 64) fill(i);
        slot = (int)((__builtin_amdgcn_readlane(cols, i - base) << shift) + (t & ((1 << shift) - 1)));
        rows_of = __builtin_amdgcn_readlane(rows, i - base);
        return __builtin_amdgcn_readlane(ids, i - base);
    }
};

}  // namespace

}  // namespace sage
