// Bounds of the pages' keys, and the pick of pages by them (gfx950).
//
// Within a page every key of channel c lies between unit * lo_c and unit * hi_c,
// so a query's product with any of them is at most unit * sum_c max(q_c lo_c, q_c hi_c):
// a matrix product of [max(q, 0), min(q, 0)] with [hi, lo]. Both sides are
// whole numbers of 8 bits, their products and sums exact in 32 on the int8 MFMA and
// in fp32 (under 2^21), and a unit is a power of two, so the scores have no rounding, and their
// order does not depend on how they are summed.
#include <algorithm>

#include "sage_cache.hpp"

namespace sage {

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr uint32_t SCALE_NAN = 255;
constexpr uint32_t SCALE_MOST = 228;  // 2^21 * 2^(228 - 127) is an fp32 number

// ---- Bounds ----
//
// A wave a (page, KV head): the greatest scale byte first, then the codes as fp16
// sixteenths of that scale (exact: 96 at most, what is under 2^-20 of the scale
// counts as if it were that much), of which two take part in one maximum or minimum.
// Reads 17/32 of a byte a key's channel and writes two a page's.
template <int D>
__global__ __launch_bounds__(256) void bounds_kernel(BoundsArgs a) {
    constexpr int G = D / CACHE_BLOCK, LANES = D / 16, TOK = 64 / LANES;  // lanes a token (16 channels each), tokens a load
    const CacheDev& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.y;
    const long long unit = (long long)blockIdx.x * 4 + wave;
    const int kvh = (int)(unit % c.kv_heads), at = (int)(unit / c.kv_heads);
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    if (seq.n == 0 || seq.diff + seq.n <= 0) return;
    const int page_tokens = 1 << c.page_shift;
    const long long col = (max(seq.diff, 0ll) >> c.page_shift) + at;
    if (col > (seq.diff + seq.n - 1) >> c.page_shift || col >= c.max_pages) return;
    const int page = cache_page(c, b, (int)col << c.page_shift);
    const int held = min(seq.len - ((int)col << c.page_shift), page_tokens);
    if (page < 0 || held <= 0) return;
    const long long row = cache_row(c, page, kvh, 0);
    const uint8_t* scales = c.k_scales + row * G;
    uint32_t top = 1;
    for (int t = lane; t < held; t += 64)
#pragma unroll
        for (int g = 0; g < G; g++) {
            const uint32_t s = scales[t * G + g];
            if (s != SCALE_NAN) top = max(top, s);
        }
#pragma unroll
    for (int d = 32; d; d /= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    const uint8_t* codes = c.k_codes + row * (D / 2);
    const _Float16 inf = (_Float16)__builtin_inff();
    h2 hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; i++) hi[i] = h2{-inf, -inf}, lo[i] = h2{inf, inf};
    const int part = lane % LANES;
#pragma unroll 4
    for (int t = lane / LANES; t < held; t += TOK) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes + t * (D / 2) + part * 8);
        const uint32_t sc = scales[t * G + part / 2];
        const float s = __uint_as_float((uint32_t)(127 + max((int)sc - (int)top + 4, -20)) << 23);
        h2 x[8] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.x, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.x, s, 1),
                   __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.x, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.x, s, 3),
                   __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.y, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.y, s, 1),
                   __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.y, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w.y, s, 3)};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            hi[i] = __builtin_elementwise_max(hi[i], sc == SCALE_NAN ? h2{inf, inf} : x[i]);
            lo[i] = __builtin_elementwise_min(lo[i], sc == SCALE_NAN ? h2{-inf, -inf} : x[i]);
        }
    }
#pragma unroll
    for (int d = LANES; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            hi[i] = __builtin_elementwise_max(hi[i], __builtin_bit_cast(h2, __shfl_xor(__builtin_bit_cast(int, hi[i]), d)));
            lo[i] = __builtin_elementwise_min(lo[i], __builtin_bit_cast(h2, __shfl_xor(__builtin_bit_cast(int, lo[i]), d)));
        }
    if (lane >= LANES) return;
    uint32_t w[2][4];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float up = __builtin_ceilf((float)hi[i / 2][i % 2]), down = __builtin_floorf((float)lo[i / 2][i % 2]);
        const uint32_t u = (uint32_t)(int)fminf(up, 127.0f) & 255, v = (uint32_t)(int)fmaxf(down, -127.0f) & 255;
        w[0][i / 4] = i % 4 ? w[0][i / 4] | u << (i % 4 * 8) : u;
        w[1][i / 4] = i % 4 ? w[1][i / 4] | v << (i % 4 * 8) : v;
    }
    const long long cell = (long long)page * c.kv_heads + kvh;
    int8_t* out = a.bounds.codes + cell * (2 * D) + part * 16;
    *reinterpret_cast<uint4*>(out) = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
    *reinterpret_cast<uint4*>(out + D) = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
    if (lane == 0) a.bounds.scales[cell] = (uint8_t)top;
}

// ---- Scores ----
//
// A tile is 16 (row, head of the group) columns of one KV head; a row's heads
// fill a power of two of them, `slots`, the last head again where the group is smaller
// (a maximum does not mind), so that a row's maximum over its heads stays in a lane's
// four results or between lanes 16 and 32 apart. Groups over 16 take several
// tiles of one row. Pages run along the lanes, 16 a step.

// Eight channels' codes, u = rint(x * up): max(u, 0) or, under `neg`, min(u, 0), a byte each.
__device__ __forceinline__ uint2 codes_of(uint4 raw, bool f16, float up, bool neg) {
    float f[8];
    unpack8(raw, f, f16);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int u = (int)__builtin_rintf(f[i] * up), v = neg ? min(u, 0) : max(u, 0);
        w[i / 4] |= (uint32_t)(v & 255) << (i % 4 * 8);
    }
    return make_uint2(w[0], w[1]);
}

// The greatest power of two 2^e, |e| <= 126, with top * 2^e <= 127 (top: fp32 bits, 0 or finite).
__device__ __forceinline__ float power_for(uint32_t top) {
    if (top == 0) return 0.0f;
    int e;
    const float m = __builtin_frexpf(__uint_as_float(top), &e);
    e = m <= 127.0f / 128 ? 7 - e : 6 - e;
    return __uint_as_float((uint32_t)(127 + min(max(e, -126), 126)) << 23);
}

__device__ __forceinline__ uint32_t greatest(uint4 raw, bool f16) {
    float f[8];
    unpack8(raw, f, f16);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    return top;
}

// Ascending with the score; 0 is no page's and 1 a page's that is not there.
__device__ __forceinline__ uint32_t key_of(float score) {
    const uint32_t u = __float_as_uint(score);
    return (int)u < 0 ? ~u : u | 0x80000000u;
}

// TILES: column tiles of a wave, over which a page's bounds are loaded once.
// Grid: x = KV heads, `parts` parts of the pages, row tiles; z = sequences.
template <int D, int TILES>
__global__ __launch_bounds__(256, 2) void score_kernel(PickArgs a, int slots, int parts) {
    constexpr int KS = 2 * D / 64, RAW = D / 16;  // MFMA steps; loads of 8 channels a lane, D / 2 channels in all
    const CacheDev& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int b = blockIdx.z, kvh = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads;
    const int part = rest % parts, tile = rest / parts, tile_rows = 16 / slots * TILES, j0 = tile * tile_rows;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int count = min(seq.n - j0, tile_rows);
    if (count <= 0 || seq.start + j0 >= (long long)a.row0 + a.window || seq.start + j0 + count <= a.row0) return;
    const int page_tokens = 1 << c.page_shift;
    const int pages = (seq.limit(j0 + count - 1, a.causal) + page_tokens - 1) >> c.page_shift;
    if (pages <= a.top) return;  // every page is picked

    // Where this lane's results belong: rows j0 + ... of tile t, see below.
    const int heads_tiles = (a.group + 15) / 16;
    i4 q[TILES][KS];
    auto load = [&](int t, int ht, auto each) {
        const int j = j0 + t * (16 / slots) + n / slots;
        const int head = kvh * a.group + min(ht * 16 + n % slots, a.group - 1);
        const long long row = seq.start + j;
        const bool have = j < seq.n && row >= 0 && row < c.rows;
        const uint16_t* p = a.q.p + row * a.q.st + head * a.q.sh + (g & 1) * (D / 2);
#pragma unroll
        for (int i = 0; i < RAW; i++)
            each(i, have ? *reinterpret_cast<const uint4*>(p + 8 * i) : make_uint4(0, 0, 0, 0));
    };
    float up[TILES];
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        uint32_t top = 0;
        for (int ht = 0; ht < heads_tiles; ht++) load(t, ht, [&](int, uint4 x) { top = max(top, greatest(x, a.q_f16)); });
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        for (int d = 1; d < slots; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        up[t] = top < 0x7f800000u ? power_for(top) : 0.0f;
    }
    auto encode = [&](int t, int ht) {
        load(t, ht, [&](int i, uint4 x) {
            const uint2 w = up[t] == 0.0f ? make_uint2(0, 0) : codes_of(x, a.q_f16, up[t], g >= 2);
            q[t][i / 2][i % 2 * 2] = (int)w.x;
            q[t][i / 2][i % 2 * 2 + 1] = (int)w.y;
        });
    };
    if (heads_tiles == 1)
#pragma unroll
        for (int t = 0; t < TILES; t++) encode(t, 0);

    for (int p0 = (part * 4 + wave) * 16; p0 < pages; p0 += parts * 64) {
        const int col = p0 + n, id = col < pages ? c.page_table[(long long)b * c.max_pages + col] : -1;
        const bool there = (unsigned)id < (unsigned)c.pages;
        const long long cell = (long long)(there ? id : 0) * c.kv_heads + kvh;
        const int8_t* at = a.bounds.codes + cell * (2 * D) + g * (D / 2);
        i4 w[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) w[s] = *reinterpret_cast<const i4*>(at + 16 * s);
        const uint32_t sc = min((uint32_t)a.bounds.scales[cell], SCALE_MOST);
        const float unit = __uint_as_float(max(sc, 1u) << 23);
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            i4 x{};
            for (int ht = 0; ht < heads_tiles; ht++) {
                if (heads_tiles > 1) encode(t, ht);
                i4 y{};
#pragma unroll
                for (int s = 0; s < KS; s++) y = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[t][s], w[s], y, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) x[r] = ht ? max(x[r], y[r]) : y[r];
            }
            // Result r is column 4 g + r: row (4 g + r) / slots of the tile.
            if (slots >= 2) x[0] = max(x[0], x[1]), x[2] = max(x[2], x[3]);
            if (slots >= 4) x[0] = max(x[0], x[2]);
            if (slots >= 8) x[0] = max(x[0], __shfl_xor(x[0], 16));
            if (slots >= 16) x[0] = max(x[0], __shfl_xor(x[0], 32));
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int j = j0 + t * (16 / slots) + (4 * g + r) / slots;
                const long long row = seq.start + j;
                if ((4 * g + r) % slots || j >= seq.n || col >= pages || row < a.row0 ||
                    row >= (long long)a.row0 + a.window)
                    continue;
                a.keys[((row - a.row0) * c.kv_heads + kvh) * a.key_cols + col] = there ? key_of((float)x[r] * unit) : 1;
            }
        }
    }
}

// ---- The greatest ----
//
// The least key that is picked is found bit by bit: 32 counts at most of how many
// of a row's keys, which stay in registers, reach it, over WAVES waves together;
// then the keys above it, and of those equal to it the first ones, go out in the
// columns' order. Grid: x = rows and KV heads, z = sequences.
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
    if (pages <= a.top) {
        for (int i = WAVES == 1 ? lane : (int)threadIdx.x; i < a.top; i += WAVES * 64) out[i] = i < pages ? i : -1;
        return;
    }
    const uint32_t* keys = a.keys + ((row - a.row0) * c.kv_heads + kvh) * a.key_cols;
    uint32_t key[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        const int col = (wave * KEYS + i) * 64 + lane;
        key[i] = col >= pages ? 0 : col < a.first || col >= pages - a.last ? 0xffffffffu : keys[col];
    }
    __shared__ int counts[2][WAVES];
    int turn = 0;
    // Sum over the waves, and over those before this one.
    auto total = [&](int mine, int& before) {
        before = 0;
        if (WAVES == 1) return mine;
        if (lane == 0) counts[turn][wave] = mine;
        __syncthreads();
        int sum = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const int x = counts[turn][w];
            if (w < wave) before += x;
            sum += x;
        }
        turn ^= 1;
        return sum;
    };
    int before;
    uint32_t least = 0;
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t t = least | 1u << bit;
        int mine = 0;
#pragma unroll
        for (int i = 0; i < KEYS; i++) mine += __builtin_popcountll(__ballot(key[i] >= t));
        const int sum = total(mine, before);
        if (sum >= a.top) least = t;
        if (sum == a.top) break;
    }
    int above = 0, equal = 0, above_before, equal_before;
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        above += __builtin_popcountll(__ballot(key[i] > least));
        equal += __builtin_popcountll(__ballot(key[i] == least));
    }
    const int room = a.top - total(above, above_before);  // of the keys equal to the least
    total(equal, equal_before);
    const uint64_t lower = (1ull << lane) - 1;
    int seen = equal_before, place = above_before + min(equal_before, room);
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        const uint64_t eq = __ballot(key[i] == least);
        const bool in = key[i] > least || (key[i] == least && seen + __builtin_popcountll(eq & lower) < room);
        const uint64_t ins = __ballot(in);
        if (in) out[place + __builtin_popcountll(ins & lower)] = (wave * KEYS + i) * 64 + lane;
        place += __builtin_popcountll(ins);
        seen += __builtin_popcountll(eq);
    }
}

}  // namespace

hipError_t launch_cache_bounds(int head_dim, const BoundsArgs& a, hipStream_t s) {
    const long long pages = std::min<long long>(((long long)a.max_new + (1 << a.c.page_shift) - 1) >> a.c.page_shift, a.c.max_pages) + 1;
    const dim3 grid((unsigned)((pages * a.c.kv_heads + 3) / 4), a.c.batch);
    if (head_dim == 64)
        hipLaunchKernelGGL(bounds_kernel<64>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(bounds_kernel<128>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

int pick_window(int rows, int kv_heads, int max_pages) {
    const long long most = 1 << 26;  // keys: 256 MB
    return (int)std::min<long long>(rows, std::max(1ll, most / ((long long)kv_heads * max_pages)));
}

template <int D>
static void score(const PickArgs& a, hipStream_t s) {
    int slots = 1;
    while (slots < 16 && slots < a.group) slots *= 2;
    const auto go = [&](auto kernel, int tiles) {
        const long long rows = 16 / slots * tiles, row_tiles = (a.max_new + rows - 1) / rows;
        const long long units = row_tiles * a.c.kv_heads * a.c.batch;
        const long long parts = std::max(1ll, std::min<long long>(1024 / units, (a.c.max_pages + 63) / 64));
        hipLaunchKernelGGL(kernel, dim3((unsigned)(row_tiles * parts * a.c.kv_heads), 1, a.c.batch), dim3(256), 0, s, a,
                           slots, (int)parts);
    };
    if (a.max_new * slots <= 16 || a.group > 16)
        go(score_kernel<D, 1>, 1);
    else
        go(score_kernel<D, 4>, 4);
}

hipError_t launch_cache_pick(int head_dim, const PickArgs& a_, hipStream_t s) {
    PickArgs a = a_;
    const int window = a.window;
    for (a.row0 = 0; a.row0 < a.c.rows; a.row0 += window) {
        a.window = std::min(window, a.c.rows - a.row0);
        if (a.c.max_pages > a.top) head_dim == 64 ? score<64>(a, s) : score<128>(a, s);
        const long long units = (long long)a.max_new * a.c.kv_heads;
        const auto pick = [&](auto kernel, int waves) {
            const long long wgs = waves == 1 ? (units + 3) / 4 : units;
            hipLaunchKernelGGL(kernel, dim3((unsigned)wgs, 1, a.c.batch), dim3(waves == 1 ? 256 : waves * 64), 0, s, a);
        };
        if (a.c.max_pages <= 256)
            pick(pick_kernel<1, 4>, 1);
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
