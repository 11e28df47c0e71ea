// Bounds of the pages' keys, and the pick of pages by them (gfx950).
//
// Within a page every key of channel c lies between unit * lo_c and unit * hi_c,
// so a query's product with any of them is at most unit * sum_c max(q_c lo_c, q_c hi_c):
// a matrix product of [max(q, 0), min(q, 0)] with [hi, lo]. Both sides are
// whole numbers of 8 bits, their products and sums exact in 32 on the int8 MFMA and
// in fp32 (under 2^21), and a unit is a power of two, so the scores of a row's codes have no rounding, and
// their order does not depend on how they are summed. The codes do: a query has 8 bits beside the
// greatest channel of its group.
#include <algorithm>

#include "sage_cache.hpp"

namespace sage {

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int CHUNK_TILES = 4;  // of a wave's columns, in chunks of rows
constexpr uint32_t SCALE_NAN = 255;
constexpr uint32_t SCALE_MOST = 228;  // 2^21 * 2^(228 - 127) is an fp32 number

// The greatest of a wave's values.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));   // lane ^ 1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));   // lane ^ 2
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // the other quad of 8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));  // the other 8 of 16
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane(max(r[0], r[1]));
}

// ---- Bounds ----
//
// A wave takes a page's KV heads one by one, `heads` of them, each head's bytes on
// their way while the one before is at work: a lane has 16 channels of every
// TOK-th token, LOADS of them at a time: the page's, eight at most. With the
// greatest scale byte known, the codes become fp16 sixteenths of that scale (exact:
// 96 at most, what is under 2^-20 of the scale counts as if it were that much),
// of which two channels of two tokens take part in one maximum or minimum. The
// chain index -> page id -> codes bounds it, and the work of a (page, head) that does not
// depend on its tokens (190 VALU instructions at pages of 32 and 64 channels, of which 32 are
// conversions, maxima and minima of codes; the VALU is 39% busy), so the lanes' meet by
// halves: of two registers, each half of the lanes goes on with one.
// Reads 17/32 of a byte a key's channel and writes two a page's: 44628 tokens of 16
// heads of 64, pages of 32, 27 MB, in 11.3 us (13.8 with maxima of one token, and
// eight loads' registers for pages of every size).

constexpr uint32_t H2_INF = 0x7c007c00u, H2_SIGNS = 0x80008000u;
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b)));
}
__device__ __forceinline__ uint32_t pk_max3(uint32_t a, uint32_t b, uint32_t c) {
    const h2 x = __builtin_elementwise_maximum(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_maximum(x, __builtin_bit_cast(h2, c)));
}
__device__ __forceinline__ uint32_t pk_min3(uint32_t a, uint32_t b, uint32_t c) {
    const h2 x = __builtin_elementwise_minimum(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_minimum(x, __builtin_bit_cast(h2, c)));
}

template <int D, int LOADS>
struct BoundsPart {
    static constexpr int G = D / CACHE_BLOCK, LANES = D / 16, TOK = 64 / LANES;  // lanes a token, tokens a load
    uint2 w[LOADS];
    uint32_t sc[LOADS];
    // Tokens t0 .. of a page and head of code row `row`, `held` of which hold something;
    // the others count as the last of them.
    __device__ __forceinline__ void load(const CacheDev& c, long long row, int t0, int held) {
        const int lane = threadIdx.x & 63, part = lane % LANES;
        const uint8_t* codes = c.k_codes + row * (D / 2);
        const uint8_t* scales = c.k_scales + row * G;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (t0 + i * TOK >= held) break;
            const uint32_t t = min(t0 + i * TOK + lane / LANES, held - 1);
            w[i] = *reinterpret_cast<const uint2*>(codes + t * (uint32_t)(D / 2) + part * 8);
            sc[i] = scales[t * (uint32_t)G + part / 2];
        }
    }
    // The greatest scale byte, and whether any block is NaN.
    __device__ __forceinline__ uint32_t top(int t0, int held, bool& nan) const {
        uint32_t top = 1, most = 0;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (t0 + i * TOK >= held) break;
            most = max(most, sc[i]);
            top = max(top, sc[i] == SCALE_NAN ? 0u : sc[i]);
        }
        nan = nan || __any(most == SCALE_NAN);
        return top;
    }
    // Two loads at a time, whose codes take part in one maximum and minimum of three.
    __device__ __forceinline__ void take(int t0, int held, uint32_t top, bool nan, uint32_t (&hi)[8], uint32_t (&lo)[8]) const {
#pragma unroll
        for (int i = 0; i < LOADS; i += 2) {
            if (t0 + i * TOK >= held) break;
            uint32_t x[2][8];
            const bool both = LOADS > 1 && t0 + (i + 1) * TOK < held;
            constexpr int NEXT = LOADS > 1 ? 1 : 0;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const uint32_t scale = n && !both ? sc[i] : sc[i + n * NEXT];
                const float s = __uint_as_float((uint32_t)(127 + max((int)scale - (int)top + 4, -20)) << 23);
                const uint2 c = n && !both ? w[i] : w[i + n * NEXT];
                const h2 y[8] = {
                    __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.x, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.x, s, 1),
                    __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.x, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.x, s, 3),
                    __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.y, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.y, s, 1),
                    __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.y, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.y, s, 3)};
#pragma unroll
                for (int k = 0; k < 8; k++) x[n][k] = __builtin_bit_cast(uint32_t, y[k]);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) hi[k] = pk_max3(hi[k], x[0][k], x[1][k]), lo[k] = pk_min3(lo[k], x[0][k], x[1][k]);
            if (nan && (sc[i] == SCALE_NAN || (both && sc[i + NEXT] == SCALE_NAN)))
#pragma unroll
                for (int k = 0; k < 8; k++) hi[k] = H2_INF, lo[k] = H2_INF | H2_SIGNS;
        }
    }
};

// The maxima over all the lanes that have the same channels of 16 registers hi, -lo (8 each): the
// lanes above 32 go on with lo, those of odd rows of 16 with registers 4 .. 7, those above 8 of
// a row with two of four, and where four lanes have a token, those above 4 of 8 with
// one of two. out: the lane's registers, D / 64 of them.
template <int D>
__device__ __forceinline__ void over_tokens(uint32_t (&hi)[8], uint32_t (&lo)[8], uint32_t (&out)[D / 64]) {
    const int lane = threadIdx.x & 63;
    uint32_t four[4];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const auto r = __builtin_amdgcn_permlane32_swap(hi[k], lo[k] ^ H2_SIGNS, false, false);
        hi[k] = pk_max(r[0], r[1]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const auto r = __builtin_amdgcn_permlane16_swap(hi[k], hi[k + 4], false, false);
        four[k] = pk_max(r[0], r[1]);
    }
    uint32_t two[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        uint32_t y = __builtin_amdgcn_update_dpp(0, four[k], 0x128, 0xf, 0x3, false);  // row_ror:8
        y = __builtin_amdgcn_update_dpp(y, four[k + 2], 0x128, 0xf, 0xc, false);
        two[k] = pk_max(lane & 8 ? four[k + 2] : four[k], y);
    }
    if constexpr (D == 64) {
        uint32_t y = __builtin_amdgcn_update_dpp(0, two[0], 0x104, 0xf, 0x5, false);  // row_shl:4
        y = __builtin_amdgcn_update_dpp(y, two[1], 0x114, 0xf, 0xa, false);           // row_shr:4
        out[0] = pk_max(lane & 4 ? two[1] : two[0], y);
    } else {
        out[0] = two[0], out[1] = two[1];
    }
}

template <int D, int LOADS>
__global__ __launch_bounds__(256) void bounds_kernel(BoundsArgs a, int heads) {
    using Part = BoundsPart<D, LOADS>;
    constexpr int SPAN = LOADS * Part::TOK;
    const CacheDev& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t runs = (c.kv_heads + heads - 1) / heads;
    const int b = blockIdx.y;
    const uint32_t unit = blockIdx.x * 4 + wave, place = unit / runs;  // of the step's pages
    const int h0 = (int)(unit - place * runs) * heads, h1 = min(h0 + heads, c.kv_heads);
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    if (seq.n == 0 || seq.diff + seq.n <= 0) return;
    const long long col = (max(seq.diff, 0ll) >> c.page_shift) + place;
    if (col > (seq.diff + seq.n - 1) >> c.page_shift || col >= c.max_pages) return;
    const int page = __builtin_amdgcn_readfirstlane(cache_page(c, b, (int)col << c.page_shift));
    const int held = min(seq.len - ((int)col << c.page_shift), 1 << c.page_shift);
    if (page < 0 || held <= 0) return;
    Part next;
    next.load(c, cache_row(c, page, h0, 0), 0, held);
    for (int h = h0; h < h1; h++) {
        const long long row = cache_row(c, page, h, 0);
        Part now = next;
        if (h + 1 < h1) next.load(c, cache_row(c, page, h + 1, 0), 0, held);
        bool nan = false;
        uint32_t top = now.top(0, held, nan);
        for (int t0 = SPAN; t0 < held; t0 += SPAN) {
            Part more;
            more.load(c, row, t0, held);
            top = max(top, more.top(t0, held, nan));
        }
        top = wave_max(top);
        uint32_t hi[8], lo[8], best[D / 64];
#pragma unroll
        for (int i = 0; i < 8; i++) hi[i] = H2_INF | H2_SIGNS, lo[i] = H2_INF;
        now.take(0, held, top, nan, hi, lo);
        for (int t0 = SPAN; t0 < held; t0 += SPAN) {
            now.load(c, row, t0, held);
            now.take(t0, held, top, nan, hi, lo);
        }
        over_tokens<D>(hi, lo, best);
        const bool low = lane >= 32;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            const h2 x = __builtin_bit_cast(h2, best[i / 2]);
            const int y = (int)fminf(__builtin_ceilf((float)x[i % 2]), 127.0f);
            w |= (uint32_t)((low ? -y : y) & 255) << (8 * i);
        }
        const long long cell = (long long)page * c.kv_heads + h;
        const int part = lane % Part::LANES, first = part * 16 + (lane >> 4 & 1) * 8 + (lane >> 3 & 1) * 4;
        int8_t* out = a.bounds.codes + cell * (2 * D) + low * D;
        if constexpr (D == 64)
            *reinterpret_cast<uint16_t*>(out + first + (lane >> 2 & 1) * 2) = (uint16_t)w;
        else
            *reinterpret_cast<uint32_t*>(out + first) = w;
        if (lane == 0) a.bounds.scales[cell] = (uint8_t)top;
    }
}

// ---- Scores ----
//
// A tile is 16 (row, head of the group) columns of one KV head; a row's heads
// fill a power of two of them, 2^slots, the last head again where the group is smaller
// (a maximum does not mind), so that a row's maximum over its heads stays in a lane's
// four results or between lanes 16 and 32 apart. Groups over 16 take several
// turns of one row. Pages run along the lanes, 16 a step.
//
// A step of a batch reads 2 D + 1 bytes a page once (63 rows over up to 256 pages each, 8 KV
// heads of 128: 17 MB in 9.2 us), and is bound by a chain: index, page ids, bounds,
// scores, list. Chunks meet the same pages again and again, in the L2: 20 GFLOP of
// whole numbers for 1563 rows over up to 954 pages in 49 us; the VALU is 42% busy
// with keys, codes and lists, the MFMA pipe 7%.

// Eight channels' codes, a byte each: rint(x * up) of x kept within lo .. hi. The sum
// with 1.5 * 2^23 has units of 1, so its low byte is the nearest whole number, ties to even.
__device__ __forceinline__ uint2 codes_of(uint4 raw, bool f16, float up, float lo, float hi) {
    float f[8];
    unpack8(raw, f, f16);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            u[k] = __float_as_uint(__builtin_fmaf(__builtin_amdgcn_fmed3f(f[4 * i + k], lo, hi), up, 12582912.0f));
        w[i] = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400) | __builtin_amdgcn_perm(u[3], u[2], 0x04000c0c);
    }
    return up == 0.0f ? make_uint2(0, 0) : make_uint2(w[0], w[1]);
}

// The greatest magnitude of eight channels, as its 16 bits.
__device__ __forceinline__ uint32_t greatest(uint4 raw) {
    typedef uint16_t u2 __attribute__((ext_vector_type(2)));
    const auto mag = [](uint32_t w) { return __builtin_bit_cast(u2, w & 0x7fff7fffu); };
    const u2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(raw.x), mag(raw.y)),
                                           __builtin_elementwise_max(mag(raw.z), mag(raw.w)));
    return max((uint32_t)m.x, (uint32_t)m.y);
}

// The greatest power of two 2^e, |e| <= 126, with top * 2^e <= 127, of a magnitude's
// bits; 0 where it is 0 or not finite.
__device__ __forceinline__ float power_for(uint32_t top, bool f16) {
    if (top == 0 || top >= (f16 ? 0x7c00u : 0x7f80u)) return 0.0f;
    int e;
    const float m = __builtin_frexpf(f16 ? f16_to_f32((uint16_t)top) : __uint_as_float(top << 16), &e);
    e = m <= 127.0f / 128 ? 7 - e : 6 - e;
    return __uint_as_float((uint32_t)(127 + min(max(e, -126), 126)) << 23);
}

// Ascending with the score; 0 is no page's and 1 a page's that is not there.
__device__ __forceinline__ uint32_t key_of(float score) {
    const uint32_t u = __float_as_uint(score);
    return (int)u < 0 ? ~u : u | 0x80000000u;
}

constexpr float INF = __builtin_inff();

// What a wave holds of 16 pages: lane (page, quarter of its bounds' bytes), so that a lane's loads
// are of one line (1563 rows of 8 KV heads over up to 954 columns: 49 us; 58 where each
// load took 64 bytes of every page).
template <int D>
struct PageStep {
    i4 w[2 * D / 64];
    uint32_t scale;
    bool there;
    __device__ __forceinline__ void load(const PickArgs& a, int kvh, int id) {
        there = (unsigned)id < (unsigned)a.c.pages;
        const long long cell = (long long)(there ? id : 0) * a.c.kv_heads + kvh;
        const int8_t* at = a.bounds.codes + cell * (2 * D) + (threadIdx.x >> 4 & 3) * (D / 2);
#pragma unroll
        for (int s = 0; s < 2 * D / 64; s++) w[s] = *reinterpret_cast<const i4*>(at + 16 * s);
        scale = a.bounds.scales[cell];
    }
};

// Pages first, first + step, ... (16 at a time) below `pages`, each step's on their
// way while the one before is at work: the first are asked for when this is made.
template <int D>
struct PageWalk {
    const int* table;
    int first, step, pages, id;
    PageStep<D> next;
    __device__ __forceinline__ PageWalk(const PickArgs& a, int b, int kvh, int first_, int step_, int pages_)
        : table(a.c.page_table + (long long)b * a.c.max_pages), first(first_), step(step_), pages(pages_) {
        next.load(a, kvh, id_at(first));
        id = id_at(first + step);
    }
    __device__ __forceinline__ int id_at(int p0) const {
        const int col = p0 + (threadIdx.x & 15);
        return col < pages ? table[col] : -1;
    }
    // The queries' codes against the pages: store(t, r, col, key) has the key of row t << (4 - slots) |
    // (4 (lane / 16) + r) >> slots, where that is the row's first result.
    template <int TILES, class Store>
    __device__ __forceinline__ void run(const PickArgs& a, int kvh, int slots, const i4 (&q)[TILES][2 * D / 64],
                                        Store store) {
        const int g = threadIdx.x >> 4 & 3, n = threadIdx.x & 15;
        for (int p0 = first; p0 < pages; p0 += step) {
            const PageStep<D> now = next;
            next.load(a, kvh, id);
            id = id_at(p0 + 2 * step);
            const int col = p0 + n;
            const float unit = __uint_as_float(max(min(now.scale, SCALE_MOST), 1u) << 23);
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                i4 x{};
#pragma unroll
                for (int s = 0; s < 2 * D / 64; s++)
                    x = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[t][s], now.w[s], x, 0, 0, 0);
                // Result r is column 4 g + r.
                if (slots >= 1) x[0] = max(x[0], x[1]), x[2] = max(x[2], x[3]);
                if (slots >= 2) x[0] = max(x[0], x[2]);
                if (slots >= 3) x[0] = max(x[0], __shfl_xor(x[0], 16));
                if (slots >= 4) x[0] = max(x[0], __shfl_xor(x[0], 32));
                if (col < pages) {
                    auto key = [&](int r) { return now.there ? key_of((float)x[r] * unit) : 1u; };
                    if (slots < 3 || (g & ((1 << slots) / 4 - 1)) == 0) store(t, 0, col, key(0));
                    if (slots < 2) store(t, 2, col, key(2));
                    if (slots < 1) store(t, 1, col, key(1)), store(t, 3, col, key(3));
                }
            }
        }
    }
};

// Where a tile's column n finds its query: the row's head of that place (from 16 * turn on).
__device__ __forceinline__ const uint16_t* query_of(const PickArgs& a, const SequenceIndex& seq, int kvh, int j0, int n,
                                                    int slots, int turn) {
    const int j = j0 + (n >> slots), head = kvh * a.group + min(turn * 16 + (n & ((1 << slots) - 1)), a.group - 1);
    const long long row = seq.start + j;
    return j < seq.n && row >= 0 && row < a.c.rows ? a.q.p + row * a.q.st + head * a.q.sh : nullptr;
}

// A tile's codes in LDS, column by column: those of the channels above 0, which meet
// the greatest keys, then those below.
template <int D>
struct TileLds {
    static constexpr int STRIDE = 2 * D + 16;
    uint32_t top[16];
    alignas(16) uint8_t codes[16 * STRIDE];
    __device__ __forceinline__ void put(int n, int part, uint4 raw, bool f16, float up) {
        uint8_t* at = codes + n * STRIDE + 8 * part;
        *reinterpret_cast<uint2*>(at) = codes_of(raw, f16, up, 0.0f, INF);
        *reinterpret_cast<uint2*>(at + D) = codes_of(raw, f16, up, -INF, 0.0f);
    }
    __device__ __forceinline__ void get(i4 (&q)[2 * D / 64]) const {
        const uint8_t* at = codes + (threadIdx.x & 15) * STRIDE + (threadIdx.x >> 4 & 3) * (D / 2);
#pragma unroll
        for (int s = 0; s < 2 * D / 64; s++) q[s] = *reinterpret_cast<const i4*>(at + 16 * s);
    }
};

// A tile's queries, eight channels a lane, a few columns a turn.
template <int D>
struct TileQueries {
    static constexpr int PARTS = D / 8, COLS = 64 / PARTS, TURNS = 16 / COLS;  // columns a turn
    uint4 raw[TURNS];
    __device__ __forceinline__ TileQueries(const PickArgs& a, const SequenceIndex& seq, int kvh, int j0, int slots) {
        const int lane = threadIdx.x & 63, n = lane / PARTS, part = lane % PARTS;
#pragma unroll
        for (int i = 0; i < TURNS; i++) {
            const uint16_t* p = query_of(a, seq, kvh, j0, i * COLS + n, slots, 0);
            raw[i] = p ? *reinterpret_cast<const uint4*>(p + 8 * part) : make_uint4(0, 0, 0, 0);
        }
    }
    // The codes of turns first, first + step, ... into LDS.
    __device__ __forceinline__ void encode(const PickArgs& a, int slots, TileLds<D>& lds, int first, int step) const {
        const int lane = threadIdx.x & 63, n = lane / PARTS, part = lane % PARTS;
        // Over a column's channels and a row's columns.
        uint32_t top[TURNS];
#pragma unroll
        for (int i = 0; i < TURNS; i++) {
            top[i] = greatest(raw[i]);
#pragma unroll
            for (int d = 1; d < 64; d *= 2)
                if (d < PARTS << slots) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], d));
        }
#pragma unroll
        for (int d = 1; d < TURNS; d *= 2) {
            if (1 << slots <= COLS * d) continue;
            uint32_t other[TURNS];
#pragma unroll
            for (int i = 0; i < TURNS; i++) other[i] = top[i ^ d];
#pragma unroll
            for (int i = 0; i < TURNS; i++) top[i] = max(top[i], other[i]);
        }
#pragma unroll
        for (int i = 0; i < TURNS; i++)
            if (i % step == first) lds.put(i * COLS + n, part, raw[i], a.q_f16, power_for(top[i], a.q_f16));
    }
};

// By a wave for itself.
template <int D>
__device__ __forceinline__ void encode_tile(const PickArgs& a, const SequenceIndex& seq, int kvh, int j0, int slots,
                                            TileLds<D>& lds, i4 (&q)[2 * D / 64]) {
    const TileQueries<D> x(a, seq, kvh, j0, slots);
    __builtin_amdgcn_wave_barrier();  // the tile before is read
    x.encode(a, slots, lds, 0, 1);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    lds.get(q);
}

// By a workgroup for all its waves, eight channels a thread; raw: those of this
// turn's head (raw_part), asked for before the pages.
template <int D>
__device__ __forceinline__ uint4 raw_part(const PickArgs& a, const SequenceIndex& seq, int kvh, int j0, int slots, int turn) {
    constexpr int PARTS = D / 8;
    const int n = threadIdx.x / PARTS, part = threadIdx.x % PARTS;
    const uint16_t* p = n < 16 ? query_of(a, seq, kvh, j0, n, slots, turn) : nullptr;
    return p ? *reinterpret_cast<const uint4*>(p + 8 * part) : make_uint4(0, 0, 0, 0);
}
template <int D>
__device__ __forceinline__ void encode_shared(const PickArgs& a, const SequenceIndex& seq, int kvh, int j0, int slots,
                                              int turn, uint4 raw, TileLds<D>& lds, i4 (&q)[2 * D / 64]) {
    constexpr int PARTS = D / 8;
    const int n = threadIdx.x / PARTS, part = threadIdx.x % PARTS, turns = (a.group + 15) / 16;
    if (n < 16) {  // (whole waves)
        uint32_t top = greatest(raw);
        for (int i = 0; i < turns; i++)
            if (i != turn) top = max(top, greatest(raw_part<D>(a, seq, kvh, j0, slots, i)));
#pragma unroll
        for (int d = 1; d < PARTS; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if (part == 0) lds.top[n] = top;
    }
    __syncthreads();
    if (n < 16) {
        const int first = n >> slots << slots;
        uint32_t top = 0;
        for (int i = 0; i < 1 << slots; i++) top = max(top, lds.top[first + i]);
        lds.put(n, part, raw, a.q_f16, power_for(top, a.q_f16));
    }
    __syncthreads();
    lds.get(q);
}

// Chunks of rows: TILES tiles of columns a wave, all waves of a workgroup over the
// same pages. Grid: x = KV heads, `parts` parts of the pages, row tiles; z = sequences.
template <int D, int TILES>
__global__ __launch_bounds__(256, 2) void score_kernel(PickArgs a, int slots, int parts) {
    const CacheDev& c = a.c;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = threadIdx.x >> 4 & 3;
    const int b = blockIdx.z, kvh = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
    const int part = rest % parts, tile = rest / parts, rows = TILES << (4 - slots), j0 = (tile * 4 + wave) * rows;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int count = min(seq.n - j0, rows);
    const long long row0 = seq.start + j0 - a.row0;  // within the window
    if (count <= 0 || row0 >= a.window || row0 + count <= 0) return;
    const int pages = (seq.limit(j0 + count - 1, a.causal) + (1 << c.page_shift) - 1) >> c.page_shift;
    if (pages <= a.top) return;  // every page is picked
    PageWalk<D> walk(a, b, kvh, part * 16, parts * 16, pages);
    __shared__ TileLds<D> lds[4];
    i4 q[TILES][2 * D / 64];
#pragma unroll
    for (int t = 0; t < TILES; t++)
        encode_tile<D>(a, seq, kvh, j0 + (t << (4 - slots)), slots, lds[wave], q[t]);
    walk.template run<TILES>(a, kvh, slots, q, [&](int t, int r, int col, uint32_t key) {
        const int j = (t << (4 - slots)) + ((4 * g + r) >> slots);
        const long long row = row0 + j;
        if (j < count && row >= 0 && row < a.window) a.keys[(row * c.kv_heads + kvh) * a.key_cols + col] = key;
    });
}

// One tile a workgroup, its waves over pages of their own; groups over 16 heads in
// turns, of which each keeps the greater key.
template <int D>
__global__ __launch_bounds__(256, 2) void score_tile_kernel(PickArgs a, int slots, int parts) {
    __shared__ TileLds<D> lds;
    const CacheDev& c = a.c;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = threadIdx.x >> 4 & 3;
    const int b = blockIdx.z, kvh = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
    const int part = rest % parts, tile = rest / parts, rows = 16 >> slots, j0 = tile * rows;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int count = min(seq.n - j0, rows);
    const long long row0 = seq.start + j0 - a.row0;  // within the window
    if (count <= 0 || row0 >= a.window || row0 + count <= 0) return;
    const int pages = (seq.limit(j0 + count - 1, a.causal) + (1 << c.page_shift) - 1) >> c.page_shift;
    if (pages <= a.top) return;  // every page is picked
    for (int turn = 0; turn < (a.group + 15) / 16; turn++) {
        const uint4 raw = raw_part<D>(a, seq, kvh, j0, slots, turn);
        PageWalk<D> walk(a, b, kvh, (part * 4 + wave) * 16, parts * 64, pages);
        i4 q[1][2 * D / 64];
        encode_shared<D>(a, seq, kvh, j0, slots, turn, raw, lds, q[0]);
        walk.template run<1>(a, kvh, slots, q, [&](int, int r, int col, uint32_t key) {
            const int j = (4 * g + r) >> slots;
            const long long row = row0 + j;
            if (j >= count || row < 0 || row >= a.window) return;
            uint32_t& at = a.keys[(row * c.kv_heads + kvh) * a.key_cols + col];
            at = turn ? max(at, key) : key;
        });
    }
}

// ---- The greatest ----
//
// The least key that is picked is found bit by bit: a count for each bit of how many
// of a row's keys, which stay in registers, reach it, over WAVES waves together. Then the keys above it, and of those equal to it the
// first ones, go out in the columns' order.
struct Counts {
    int* lds;  // [2][WAVES]
    int turn;
    // Sum over the waves, and over those before this one.
    template <int WAVES>
    __device__ __forceinline__ int total(int mine, int wave, int& before) {
        before = 0;
        if (WAVES == 1) return mine;
        int* at = lds + turn * WAVES;
        if ((threadIdx.x & 63) == 0) at[wave] = mine;
        __syncthreads();
        int sum = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const int x = at[w];
            if (w < wave) before += x;
            sum += x;
        }
        turn ^= 1;
        return sum;
    }
};

// Where a search for the top-th greatest key begins: the bits from `bit` on, on `least`,
// which top keys reach.
struct Search {
    uint32_t least = 0;
    int bit = 31;
    // The top-th greatest is within lo .. hi, or any key over hi is.
    static __device__ __forceinline__ Search between(uint32_t lo, uint32_t hi) {
        const int n = lo == hi ? 0 : 32 - __builtin_clz(lo ^ hi);  // bits in which they differ
        return {n == 32 ? 0 : lo >> n << n, n - 1};
    }
};

// The list from a row's keys, all more than 0 of which are more than top: key[i] is of
// the i-th of the wave's columns that col(i) gives, in their order.
template <int WAVES, int KEYS, class Col>
__device__ __forceinline__ void write_greatest(const uint32_t (&key)[KEYS], int top, int wave, int* out, int* lds, Col col,
                                               Search from = Search{}) {
    const int lane = threadIdx.x & 63;
    Counts counts{lds, 0};
    int before;
    uint32_t least = from.least;
    for (int bit = from.bit; bit >= 0; bit--) {
        const uint32_t t = least | 1u << bit;
        int mine = 0;
#pragma unroll
        for (int i = 0; i < KEYS; i++) mine += __builtin_popcountll(__ballot(key[i] >= t));
        const int sum = counts.total<WAVES>(mine, wave, before);
        if (sum >= top) least = t;
        if (sum == top) break;
    }
    int above = 0, equal = 0, above_before, equal_before;
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        above += __builtin_popcountll(__ballot(key[i] > least));
        equal += __builtin_popcountll(__ballot(key[i] == least));
    }
    const int room = top - counts.total<WAVES>(above, wave, above_before);  // of the keys equal to the least
    counts.total<WAVES>(equal, wave, equal_before);
    const uint64_t lower = (1ull << lane) - 1;
    int seen = equal_before, place = above_before + min(equal_before, room);
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        const uint64_t eq = __ballot(key[i] == least);
        const bool in = key[i] > least || (key[i] == least && seen + __builtin_popcountll(eq & lower) < room);
        const uint64_t ins = __ballot(in);
        if (in) out[place + __builtin_popcountll(ins & lower)] = col(i);
        place += __builtin_popcountll(ins);
        seen += __builtin_popcountll(eq);
    }
}

// A wave's writes to LDS before its reads behind this.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A row's list by one wave; key[i]: of column i * 64 + lane. For lists of at most
// 64, the top-th greatest of the lanes' greatest keys is no more than the list's least, and
// few keys reach it: the counts go over those, two a lane (1563 rows of 8 KV heads over
// up to 954 columns, lists of 32: 49 us, 61 with counts over all keys). `few`: LDS of the wave.
struct Few {
    uint32_t key[128];
    int col[128];
};
template <int KEYS>
__device__ __forceinline__ void write_greatest_of_wave(const uint32_t (&key)[KEYS], int top, int* out, Few& few) {
    const int lane = threadIdx.x & 63;
    uint32_t most = 0, highest = 0;
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        most = max(most, key[i]);
        highest = max(highest, key[i] + 1 ? key[i] : 0);  // of those that are not always picked
    }
    highest = wave_max(highest);
    // (top is at most the lanes that have a key: the least of their greatest bounds the list's.)
    const Search from = top > 64 ? Search{} : Search::between(min(~wave_max(~most), highest), highest);
    auto plain = [&] { write_greatest<1, KEYS>(key, top, 0, out, nullptr, [&](int i) { return i * 64 + lane; }, from); };
    if (KEYS <= 4 || top > 64) return plain();
    uint32_t bound = from.least;
    for (int bit = from.bit; bit >= 0; bit--) {
        const uint32_t t = bound | 1u << bit;
        const int sum = __builtin_popcountll(__ballot(most >= t));
        if (sum >= top) bound = t;
        if (sum == top) break;
    }
    const uint64_t lower = (1ull << lane) - 1;
    int n = 0;
#pragma unroll
    for (int i = 0; i < KEYS; i++) n += __builtin_popcountll(__ballot(key[i] >= bound));
    if (n > 128) return plain();
    wave_sync();  // the row before is read
    n = 0;
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        const uint64_t in = __ballot(key[i] >= bound);
        const int at = n + __builtin_popcountll(in & lower);
        if (key[i] >= bound) few.key[at] = key[i], few.col[at] = i * 64 + lane;
        n += __builtin_popcountll(in);
    }
    wave_sync();
    const uint32_t two[2] = {lane < n ? few.key[lane] : 0, 64 + lane < n ? few.key[64 + lane] : 0};
    write_greatest<1, 2>(two, top, 0, out, nullptr, [&](int i) { return few.col[i * 64 + lane]; },
                         Search::between(min(bound, highest), highest));
}

// A row's list where all its pages are picked.
__device__ __forceinline__ void write_all(int* out, int pages, int top, int first, int step) {
    for (int i = first; i < top; i += step) out[i] = i < pages ? i : -1;
}

// From the keys in memory. Grid: x = rows and KV heads, z = sequences.
template <int WAVES, int KEYS>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void pick_kernel(PickArgs a) {
    const CacheDev& c = a.c;
    const int lane = threadIdx.x & 63, wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = WAVES == 1 ? 0 : wave_id;
    const long long unit = WAVES == 1 ? (long long)blockIdx.x * 4 + wave_id : blockIdx.x;
    const int b = blockIdx.z, kvh = (int)(unit % c.kv_heads), j = (int)(unit / c.kv_heads);
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const long long row = seq.start + j;
    if (j >= seq.n || row < a.row0 || row >= (long long)a.row0 + a.window) return;
    const int pages = (seq.limit(j, a.causal) + (1 << c.page_shift) - 1) >> c.page_shift;
    int* out = a.picked + (row * c.kv_heads + kvh) * a.top;
    if (pages <= a.top) return write_all(out, pages, a.top, WAVES == 1 ? lane : (int)threadIdx.x, WAVES * 64);
    const uint32_t* keys = a.keys + ((row - a.row0) * c.kv_heads + kvh) * a.key_cols;
    uint32_t key[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        const int col = (wave * KEYS + i) * 64 + lane;
        key[i] = col >= pages ? 0 : col < a.first || col >= pages - a.last ? 0xffffffffu : keys[col];
    }
    if constexpr (WAVES == 1) {
        __shared__ Few few[4];
        write_greatest_of_wave<KEYS>(key, a.top, out, few[wave_id]);
    } else {
        __shared__ int lds[2 * WAVES];
        write_greatest<WAVES, KEYS>(key, a.top, wave, out, lds, [&](int i) { return (wave * KEYS + i) * 64 + lane; });
    }
}

// Rows whose keys fit LDS: both in one launch, eight waves over the pages of TILES
// tiles of rows, then over the rows. Grid: x = KV heads, row tiles; z = sequences.
// The masks of 16 and 32 keys a lane are more than the scalar registers hold: 18 and some 91 of
// them wait in lanes of a vector register (pick_kernel<16, 32>: 81), and <128, 4, 32> keeps two vector
// registers in memory.
template <int D, int TILES, int KEYS>
__global__ __launch_bounds__(512, TILES == 1 ? 2 : 4) void row_pick_kernel(PickArgs a, int slots) {
    extern __shared__ uint32_t row_keys[];  // [rows][key_cols]
    __shared__ union {
        TileLds<D> tile[TILES];
        Few few[8];
    } lds;
    const CacheDev& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int b = blockIdx.z, kvh = blockIdx.x % c.kv_heads, rows = TILES << (4 - slots);
    const int j0 = blockIdx.x / c.kv_heads * rows;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int count = min(seq.n - j0, rows);
    if (count <= 0) return;
    auto pages_of = [&](int j) { return (seq.limit(j0 + j, a.causal) + (1 << c.page_shift) - 1) >> c.page_shift; };
    const int pages = pages_of(count - 1);
    auto score = [&](PageWalk<D>& walk, const i4 (&q)[TILES][2 * D / 64]) {
        walk.template run<TILES>(a, kvh, slots, q, [&](int t, int r, int col, uint32_t key) {
            const int j = (t << (4 - slots)) + ((4 * g + r) >> slots);
            if (j < count) row_keys[j * a.key_cols + col] = key;
        });
    };
    if (pages > a.top) {
        i4 q[TILES][2 * D / 64];
        // (The queries are asked for in front of the pages, whose loads wait for their ids.)
        if constexpr (TILES == 1) {
            const uint4 raw = raw_part<D>(a, seq, kvh, j0, slots, 0);
            PageWalk<D> walk(a, b, kvh, wave * 16, 128, pages);
            encode_shared<D>(a, seq, kvh, j0, slots, 0, raw, lds.tile[0], q[0]);
            score(walk, q);
        } else {
            const int t = wave % TILES;
            const TileQueries<D> x(a, seq, kvh, j0 + (t << (4 - slots)), slots);
            PageWalk<D> walk(a, b, kvh, wave * 16, 128, pages);
            x.encode(a, slots, lds.tile[t], wave / TILES, 8 / TILES);
            __syncthreads();
#pragma unroll
            for (int t = 0; t < TILES; t++) lds.tile[t].get(q[t]);
            score(walk, q);
        }
    }
    __syncthreads();  // (the tiles are read, too)
    for (int j = wave; j < count; j += 8) {
        const long long row = seq.start + j0 + j;
        if (row < 0 || row >= c.rows) continue;
        const int mine = pages_of(j);
        int* out = a.picked + (row * c.kv_heads + kvh) * a.top;
        if (mine <= a.top) {
            write_all(out, mine, a.top, lane, 64);
            continue;
        }
        uint32_t key[KEYS];
#pragma unroll
        for (int i = 0; i < KEYS; i++) {
            const int col = i * 64 + lane;
            key[i] = col >= mine ? 0 : col < a.first || col >= mine - a.last ? 0xffffffffu : row_keys[j * a.key_cols + col];
        }
        write_greatest_of_wave<KEYS>(key, a.top, out, lds.few[wave]);
    }
}

}  // namespace

hipError_t launch_cache_bounds(int head_dim, const BoundsArgs& a, hipStream_t s) {
    const long long pages = std::min<long long>(((long long)a.max_new + (1 << a.c.page_shift) - 1) >> a.c.page_shift, a.c.max_pages) + 1;
    // Heads of a page by one wave, where that leaves waves enough to fill the chip. Replayed from a
    // graph, us, 1, 2 and 4 heads, 3 x 15000 tokens:
    //   16 heads of 64, pages of 16      19.5  15.7  14.0
    //                   pages of 32      12.7  11.3  11.1 (ragged, 44628 tokens: 11.3 with 2, 11.9 with 4)
    //   8 heads of 128, pages of 16      12.7  11.4  11.6
    //                   pages of 64       8.3   8.5   8.3
    //                   pages of 256      9.7   9.5  10.2
    const int loads = (head_dim << a.c.page_shift) / 1024;  // of a page of one head, 1024 channels each
    const int heads = (int)std::max(1ll, std::min<long long>({loads == 1 ? 4 : 2, a.c.kv_heads, pages * a.c.batch * a.c.kv_heads / 4096}));
    const long long units = pages * ((a.c.kv_heads + heads - 1) / heads);
    const dim3 grid((unsigned)((units + 3) / 4), a.c.batch);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, heads); };
    if (head_dim == 64)
        go(loads == 1 ? bounds_kernel<64, 1> : loads == 2 ? bounds_kernel<64, 2> : loads == 4 ? bounds_kernel<64, 4> : bounds_kernel<64, 8>);
    else
        go(loads == 2 ? bounds_kernel<128, 2> : loads == 4 ? bounds_kernel<128, 4> : bounds_kernel<128, 8>);
    return hipGetLastError();
}

// Columns of a tile that a row takes, as a power of two.
static int slots_of(int group) {
    int slots = 0;
    while (slots < 4 && 1 << slots < group) slots++;
    return slots;
}

int pick_window(int rows, int kv_heads, int max_pages) {
    const long long most = 1 << 26;  // keys: 256 MB
    return (int)std::min<long long>(rows, std::max(1ll, most / ((long long)kv_heads * max_pages)));
}

// The pages are cut into as many parts as fill 512 workgroups with chunks and 1024 with single
// tiles. Half of both, these and twice of both, us, 32/8 heads of 128: 1 x 1000 rows over 4096 columns
// 207, 177, 188, over 8192 1068, 991, 964, 1 x 128 rows over 4096 49, 48, 60; 64/2 heads, 64 rows over
// 1024 columns 24.5, 24.0, 27.4.
template <int D>
static void score(const PickArgs& a, hipStream_t s) {
    const int slots = slots_of(a.group);
    const bool chunks = a.group <= 16 && (long long)a.max_new << slots > 16;
    const long long rows = (chunks ? 4 * CHUNK_TILES : 1) << (4 - slots), row_tiles = (a.max_new + rows - 1) / rows;
    const long long units = row_tiles * a.c.kv_heads * a.c.batch, most = chunks ? 512 : 1024, each = 64;
    const int parts = (int)std::max(1ll, std::min(most / units, (a.c.max_pages + each - 1) / each));
    hipLaunchKernelGGL((chunks ? score_kernel<D, CHUNK_TILES> : score_tile_kernel<D>),
                       dim3((unsigned)(row_tiles * parts * a.c.kv_heads), 1, a.c.batch), dim3(256), 0, s, a, slots, parts);
}

// One launch, where the keys of a workgroup's rows fit 64 KB of LDS: as many tiles a
// workgroup as leave 256 of them. But where a sequence's rows are one tile, under 128 workgroups
// and over 512 columns take two launches, which spread the pages over more workgroups; the
// rows of several tiles do not, as their scores come from waves of four tiles each
// (score_kernel). Replayed from a graph, us, one launch and two, lists of 32, pages of 16:
//                           512 columns  1024       2048
//   32/8 heads of 128
//   1 row                   9.0  8.9     13.8 9.3   23.3 13.1
//   4 rows                  10.3 8.6     14.3 9.4   24.2 13.9
//   5 rows (two tiles)      9.5  22.2    14.2 22.6  24.0 27.0
//   16                      9.6  23.3    14.5 24.4  24.3 28.7
//   64                      9.8  25.6    17.1 26.3  24.8 32.8
//   128                     10.2 25.8    15.4 28.2  25.5 41.8
//   16 x 1                  9.5  11.4    16.7 16.0  28.3 27.2
//   64 x 1                  17.3 20.6    29.0 32.7  58.4 69.6
//   8/8 heads, 16 rows      12.7 9.2     18.4 9.9   14.5 13.8 (2048: in two launches both)
//              32 (two)     12.3 22.3    18.4 23.1  28.6 27.5
//   4/1 heads, 4 rows       8.9  8.3     14.0 9.2   23.3 13.1
//              5 and 64     9.1  21.7    14.2 22.6  23.5 26.6;  9.3 24.7  14.1 25.3  23.9 31.5
// and at 256 columns 6.7 and 8.1 for 1 row, 7.5 and 24.4 for 64 (with four tiles a workgroup
// 13.1). The tiles of a workgroup, or 0.
int pick_tiles(int batch, int group, int kv_heads, int max_new, int max_pages) {
    const int slots = slots_of(group);
    if (group > 16 || max_pages > 2048) return 0;
    for (int tiles = 4; tiles; tiles /= 2) {
        const int rows = tiles << (4 - slots);
        if (std::min(rows, max_new) * max_pages > 1 << 14) continue;
        const long long units = ((long long)max_new + rows - 1) / rows * kv_heads * batch;
        if (tiles > 1 && (rows / 2 >= max_new || units < 256)) continue;  // fewer rows a workgroup
        return units >= 128 || max_pages <= 512 || rows < max_new ? tiles : 0;
    }
    return 0;
}

template <int D, int KEYS>
static bool row_pick(const PickArgs& a, hipStream_t s) {
    const int tiles = pick_tiles(a.c.batch, a.group, a.c.kv_heads, a.max_new, a.c.max_pages);
    const int slots = slots_of(a.group), rows = tiles << (4 - slots);
    if (!tiles) return false;
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.max_new + rows - 1) / rows * a.c.kv_heads), 1, a.c.batch), dim3(512),
                           std::min(rows, a.max_new) * a.c.max_pages * 4, s, a, slots);
    };
    if (tiles == 4)
        go(row_pick_kernel<D, 4, KEYS>);
    else if (tiles == 2)
        go(row_pick_kernel<D, 2, KEYS>);
    else
        go(row_pick_kernel<D, 1, KEYS>);
    return true;
}

template <int D>
static bool rows_in_one(const PickArgs& a, hipStream_t s) {
    if (a.c.max_pages <= 256) return row_pick<D, 4>(a, s);
    if (a.c.max_pages <= 512) return row_pick<D, 8>(a, s);
    if (a.c.max_pages <= 1024) return row_pick<D, 16>(a, s);
    return row_pick<D, 32>(a, s);
}

hipError_t launch_cache_pick(int head_dim, const PickArgs& a_, hipStream_t s) {
    PickArgs a = a_;
    if (head_dim == 64 ? rows_in_one<64>(a, s) : rows_in_one<128>(a, s)) return hipGetLastError();
    const int window = a.window;
    for (a.row0 = 0; a.row0 < a.c.rows; a.row0 += window) {
        a.window = std::min(window, a.c.rows - a.row0);
        if (a.c.max_pages > a.top) head_dim == 64 ? score<64>(a, s) : score<128>(a, s);
        const long long units = (long long)a.max_new * a.c.kv_heads;
        const auto pick = [&](auto kernel, int waves) {
            const long long wgs = waves == 1 ? (units + 3) / 4 : units;
            hipLaunchKernelGGL(kernel, dim3((unsigned)wgs, 1, a.c.batch), dim3(waves == 1 ? 256 : waves * 64), 0, s, a);
        };
        // As few waves a row as hold its keys, 16 a lane at most, but for the widest. With the next
        // kernel one step earlier, us, both launches, 64/2 heads of 128, 1 and 1000 rows: 1024 columns
        // 11.9 to 15.9 and 140 to 160; 4096 columns 16.7 to 32.8 and 538 to 716.
        if (a.c.max_pages <= 256)
            pick(pick_kernel<1, 4>, 1);
        else if (a.c.max_pages <= 512)
            pick(pick_kernel<1, 8>, 1);
        else if (a.c.max_pages <= 1024)
            pick(pick_kernel<1, 16>, 1);
        else if (a.c.max_pages <= 4096)
            pick(pick_kernel<4, 16>, 4);
        else
            pick(pick_kernel<16, 32>, 16);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace sage
