// Attention over picked pages (gfx950): chunks of rows, and how a call runs.
//
// Steps and other few rows run the few-rows kernel over their lists
// (sage_cache_attn.hip). Chunks take 32 columns a unit: a page that any of the unit's
// rows picked is read and converted once for all of them, so that wider units convert less
// and multiply more for rows that have not picked it. 32 is the width of the larger
// MFMA, whose operands a wave's registers hold beside the outputs of its own tokens.
#include <algorithm>

#include "sage_cache_attn.hpp"

namespace sage {

namespace {

constexpr int UCOLS = 32;        // columns of a unit
constexpr int USTEP = 4 * TOKENS;
constexpr uint32_t SLOTS = 512;       // workgroups that the chip holds at once

// The call's units in a line: sequence by sequence its tiles, KV heads fastest. As many
// rounds of SLOTS as there are whole run a workgroup a unit; the units over, `rest`, are cut
// into as many parts each as fill one more round, so that the chip does not wait for a
// few (1563 rows behind 30000 tokens, 32/8 heads of 128, 32 pages of 64 each, 1568 units:
// 267 us with all of them whole, 252 so).
struct Plot {
    uint32_t whole, rest, parts;  // units that run whole, units over, parts of each of those
    uint32_t cut;                 // the workgroup's: of which unit over,
    int part;                     // which part, or -1: a whole unit;
    int b, kvh, tile;             // its sequence (-1: none), KV head and tile
    SequenceIndex seq;

    // By every wave for itself; at: the place in the line of workgroups, or among the units over.
    __device__ __forceinline__ Plot(const CacheAttnArgs& a, uint32_t at, bool over) {
        const CacheDev& c = a.c;
        const int lane = threadIdx.x & 63, run = (c.batch + 63) / 64;
        const int b0 = min(c.batch, lane * run), b1 = min(c.batch, b0 + run);
        uint32_t mine = 0;
        for (int i = b0; i < b1; i++) mine += tiles_of(a, index_of(a, i));
        uint32_t upto = mine;
        for (int d = 1; d < min(64, c.batch); d *= 2) {
            const uint32_t v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        const uint32_t units = __builtin_amdgcn_readlane(upto, (c.batch - 1) / run) * c.kv_heads;
        whole = units / SLOTS * SLOTS;
        rest = units - whole;
        parts = rest ? min(SLOTS / rest, (uint32_t)a.splits) : 0;
        if (parts == 1) whole = units, rest = 0;
        b = -1, part = -1, cut = 0;
        uint32_t unit = at;
        if (over) {
            if (at >= rest) return;
            cut = at, unit = whole + at, part = 0;
        } else if (at >= whole) {
            if (at - whole >= rest * parts) return;
            part = (int)((at - whole) / rest), cut = at - whole - part * rest, unit = whole + cut;
        }
        const uint32_t place = unit / c.kv_heads;  // among the tiles
        kvh = (int)(unit - place * c.kv_heads);
        const int from = 63 - __builtin_clzll(__ballot(upto - mine <= place && lane * run < c.batch));
        uint32_t first = __builtin_amdgcn_readlane(upto - mine, from);
        b = from * run;
        while (true) {
            seq = index_of(a, b);
            const uint32_t n = tiles_of(a, seq);
            tile = (int)(place - first);
            if (place < first + n) return;
            if (b >= c.batch - 1) break;
            first += n;
            b++;
        }
        b = -1;  // (starts that make no sense)
    }
    // Of the rows that the tensors have: their units are no more than the launch counts.
    static __device__ __forceinline__ SequenceIndex index_of(const CacheAttnArgs& a, int b) {
        SequenceIndex s = sequence_index(a.c, b, a.max_new);
        s.n = (int)max(0ll, min((long long)s.n, a.c.rows - s.start));
        return s;
    }
    static __device__ __forceinline__ uint32_t tiles_of(const CacheAttnArgs& a, const SequenceIndex& s) {
        return ((uint32_t)s.n * a.group + UCOLS - 1) / UCOLS;
    }
};

// Four waves take 64 tokens of the list each in turn; their outputs meet in LDS in the
// end. K's codes go from memory to the MFMA's rows (a lane: a token, half of its channels)
// and are converted there; V's through the wave's own part of LDS, 32 tokens at a time,
// for the transposing read. A step's keys are asked for once the one before has its
// logits, its values once the one before has its sums.
// QP: bf16 parts of a query. BIG: pages of 64 tokens or more, so that a step is of one
// page, its place and rows scalar (the chunks above: 264 us without it, 252 with). The
// weights are two bf16 parts (2^-16 of each), as in the few-rows kernel, so that a row's
// bits do not depend on how many rows share its call: fp16 ones for bf16 outputs took those
// chunks 208 us, but are off by up to 2^-11 of each, which is more than the output's own rounding
// where values cancel, and lose weights below 2^-32 of the row's greatest.
// They are 52 GFLOP of pairs that were picked, a third of those that the units multiply. A wave's step
// of 64 tokens is 48 MFMAs and 486 other VALU instructions, of which 128 are conversions, 32
// exponentials and some 100 the weights' parts; the VALU is 56% busy, the MFMA pipe 38%. Two waves a
// SIMD is what 256 registers leave, which they need (255, none in memory).
template <int D, int QP, bool BIG>
__global__ __launch_bounds__(256, 2) void picked_chunk(CacheAttnArgs a) {
    static_assert(QP == 1 || D == 64, "two parts of 128 channels do not fit the registers");
    constexpr int G = D / 32, KS = D / 16, CT = D / 32;  // scale blocks, MFMA steps over the channels, channel tiles
    constexpr int VT = 64 / G, HALF = TOKENS / 2;        // tokens of a V load; of V in LDS at a time
    constexpr int PAD = D / 2 + 4;                       // floats of a column where half the outputs meet
    constexpr int PART = HALF * D * 2 > UCOLS * PAD * 4 ? HALF * D * 2 : UCOLS * PAD * 4;
    __shared__ __align__(16) uint8_t lds[4 * PART];
    __shared__ float wm[4][UCOLS], wl[4][UCOLS];
    extern __shared__ uint32_t pick_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const CacheDev& c = a.c;
    const Plot plot(a, blockIdx.x, false);
    if (plot.b < 0) return;
    const int b = plot.b, kvh = plot.kvh, c0 = plot.tile * UCOLS;
    const SequenceIndex seq = plot.seq;
    const int cols = seq.n * a.group;
    const int j0 = c0 / a.group, j1 = (min(c0 + UCOLS, cols) - 1) / a.group;
    const int j = (c0 + col) / a.group, head = kvh * a.group + (c0 + col) - j * a.group;
    const long long row = seq.start + j;
    const bool have = c0 + col < cols && row >= 0 && row < c.rows;
    const int limit = seq.limit(j, a.causal), least = seq.limit(j0, a.causal);
    uint4 raw[KS];  // the column's query, on its way while the list is made
    {
        const uint16_t* p = a.q.p + row * a.q.st + head * a.q.sh + half * (D / 2);
#pragma unroll
        for (int s = 0; s < KS; s++) raw[s] = have ? *reinterpret_cast<const uint4*>(p + 8 * s) : make_uint4(0, 0, 0, 0);
    }
    const int in_page = (1 << c.page_shift) - 1;
    const int pages = (seq.limit(j1, a.causal) + in_page) >> c.page_shift;
    const Entries entries = entries_of<4, UCOLS>(a, seq, b, kvh, j0, j1 - j0 + 1, pages, pick_lds);
    bf8 q[QP][KS];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const uint4 x = signed_q(raw[s], a.q_sign);
        if (QP == 2) {
            float f[8];
            unpack8(x, f, true);
            bf8 two[2];
            parts_of<2>(f, two);
            q[0][s] = two[0], q[QP - 1][s] = two[1];
        } else {
            q[0][s] = __builtin_bit_cast(bf8, x);
        }
    }
    const int tokens = entries.count << c.page_shift, steps = (tokens + USTEP - 1) / USTEP;
    const int parts = (int)plot.parts;
    const int s0 = plot.part < 0 ? 0 : steps * plot.part / parts, s1 = plot.part < 0 ? steps : steps * (plot.part + 1) / parts;
    const int t_first = s0 * USTEP + wave * TOKENS, end = min(s1 * USTEP, tokens);

    // A step's 16-token tiles: code row, slot of the first token, the rows that see it.
    constexpr int TILES = BIG ? 1 : 4;
    struct Tiles {
        long long at[TILES];
        int slot[TILES];
        uint32_t rows[TILES];
    };
    Walk walk(entries, c.page_shift, lane, t_first);
    auto look_up = [&](int t, Tiles& x) {
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const int page = walk.of(t + 16 * i, x.slot[i], x.rows[i]);
            if (page < 0) x.rows[i] = 0;
            x.at[i] = cache_row(c, max(page, 0), kvh, (t + 16 * i) & in_page);
        }
    };
    // The code row of the lane's token k of the step, of its tiles i (and i + 1, for `second`): a scalar and an
    // offset that never changes, where the step is of one page.
    auto row_at = [&](const Tiles& x, int i, int second) {
        if constexpr (BIG)
            return x.at[0];
        else
            return x.at[i] + ((x.at[i + 1 < 4 ? i + 1 : i] - x.at[i]) & -(long long)second);
    };
    uint32_t kw[2][KS], ks[2];
    auto load_k = [&](const Tiles& x) {
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            const long long r = row_at(x, 2 * sub, col >> 4);
            const uint32_t k = BIG ? 32 * sub + col : col & 15;
            const uint8_t* p = c.k_codes + r * (D / 2);
#pragma unroll
            for (int n = 0; n < KS / 4; n++) {
                const uint4 z = *reinterpret_cast<const uint4*>(p + (k * (D / 2) + half * (D / 4) + 16 * n));
                kw[sub][4 * n] = z.x, kw[sub][4 * n + 1] = z.y, kw[sub][4 * n + 2] = z.z, kw[sub][4 * n + 3] = z.w;
            }
            const uint8_t* z = c.k_scales + r * G;
            const uint32_t at = k * G + half * (G / 2);
            ks[sub] = D == 128 ? *reinterpret_cast<const uint16_t*>(z + at) : z[at];
        }
    };
    uint4 v[G];
    uint32_t vs[G];
    auto load_v = [&](const Tiles& x) {
#pragma unroll
        for (int i = 0; i < G; i++) {
            const long long r = row_at(x, i * VT / 16, VT == 32 && lane >= 32);
            const uint32_t k = BIG ? i * VT + lane / G : lane / G & 15;
            v[i] = *reinterpret_cast<const uint4*>(c.v_codes + r * (D / 2) + (k * (D / 2) + lane % G * 16));
            vs[i] = (c.v_scales + r * G)[k * G + lane % G];
        }
    };

    f16v o[CT];
#pragma unroll
    for (int u = 0; u < CT; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[u][i] = 0.0f;
    float m = NEG_INF, l = 0.0f;
    uint8_t* vl = lds + wave * PART;
    const int vtok = 4 * half + (lane >> 2 & 3), vunit = lane >> 4 & 1;
    Tiles next;
    if (t_first < end) {
        look_up(t_first, next);
        load_k(next);
        load_v(next);
    }
    for (int t = t_first; t < end; t += USTEP) {
        const Tiles now = next;
        const bool more = t + USTEP < end;
        f16v x[2];
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[sub][i] = 0.0f;
            const float sf[2] = {__uint_as_float((ks[sub] & 255) << 23), __uint_as_float((ks[sub] >> 8) << 23)};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const bf8 kk = __builtin_bit_cast(bf8, decode8(kw[sub][s], sf[s / 4]));
#pragma unroll
                for (int p = 0; p < QP; p++) x[sub] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kk, q[p][s], x[sub], 0, 0, 0);
            }
        }
        if (more) {
            look_up(t + USTEP, next);
            load_k(next);
        }
        // Register i of sub is token 8 (i / 4) + 4 half + i % 4 of its 32: of 16-token tile 2 sub + i / 8.
        auto slot_of = [&](int tile) { return BIG ? now.slot[0] + 16 * tile : now.slot[BIG ? 0 : tile]; };
        auto picked = [&](int tile) { return (now.rows[BIG ? 0 : tile] >> (j - j0) & 1) != 0; };
        auto sees = [&](int sub, int i) {
            const int tile = 2 * sub + i / 8;
            return picked(tile) && slot_of(tile) + ((8 * (i / 4) + i % 4) & 15) + 4 * half < limit;
        };
        float mx = NEG_INF;
        if (slot_of(0) + 16 > least || slot_of(1) + 16 > least || slot_of(2) + 16 > least || slot_of(3) + 16 > least) {
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!sees(sub, i)) x[sub][i] = NEG_INF;
        } else {
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[sub][i] = picked(2 * sub + i / 8) ? x[sub][i] : NEG_INF;
        }
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, x[sub][i]);
        {
            auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(m, fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
        }
        if (__any((mx - m) * a.qk_mul > SLACK)) {
            const float scale = __builtin_amdgcn_exp2f((m - (mx == NEG_INF ? 0.0f : mx)) * a.qk_mul);
            m = mx;
            l *= scale;
#pragma unroll
            for (int u = 0; u < CT; u++) o[u] *= scale;
        }
        const float base = m == NEG_INF ? 0.0f : m * a.qk_mul;
#pragma unroll
        for (int sub = 0; sub < 2; sub++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                x[sub][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[sub][i], a.qk_mul, -base));
                l += x[sub][i];
            }
        // 32 tokens of V into LDS as bf16, then O^T += V^T P^T.
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
#pragma unroll
            for (int n = sub * G / 2; n < (sub + 1) * G / 2; n++) {
                const float s = __uint_as_float(vs[n] >= V_NAN ? 0 : vs[n] << 23);
                const uint32_t w[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
#pragma unroll
                for (int d = 0; d < 4; d++)
                    *reinterpret_cast<uint4*>(vl + unit_at<D>((lane / G + n * VT) % HALF, (lane % G) * 2 + d / 2, d & 1)) =
                        decode8(w[d], s);
            }
#pragma unroll
            for (int st = 0; st < 2; st++) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] = x[sub][8 * st + i];
                bf8 p[2];
                parts_of<2>(e, p);
#pragma unroll
                for (int u = 0; u < CT; u++) {
                    const uint8_t* at = vl + 16 * st * (D * 2) + unit_at<D>(vtok, 2 * u + vunit, lane >> 1 & 1) + (lane & 1) * 8;
                    const bf8 vv = read_v(at, 8 * (D * 2));
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        o[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv, p[k], o[u], 0, 0, 0);
                }
            }
        }
        // Blocks of NaN, bit (token % VT) * G + block of each load.
        uint64_t bad[G], any_bad = 0;
#pragma unroll
        for (int i = 0; i < G; i++) bad[i] = __ballot(vs[i] >= V_NAN), any_bad |= bad[i];
        if (any_bad) {
            uint32_t hit = 0;  // blocks of NaN that this lane's tokens bring to its column
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int tok = 32 * sub + 8 * (i / 4) + 4 * half + i % 4;
                    const uint32_t blocks = (uint32_t)(bad[(32 * sub + 8 * (i / 4)) / VT] >> (tok % VT * G)) & ((1u << G) - 1);
                    if (sees(sub, i)) hit |= blocks;
                }
            auto r = __builtin_amdgcn_permlane32_swap(hit, hit, false, false);
            hit = r[0] | r[1];
#pragma unroll
            for (int u = 0; u < CT; u++)
                if (hit >> u & 1)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[u][i] = __builtin_nanf("");
        }
        if (more) load_v(next);
    }
    {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }

    // The waves' parts meet in LDS, half of the channels at a time: a thread sums N of a column.
    constexpr int N = D / 16;
    float* ol = reinterpret_cast<float*>(lds);  // [4][UCOLS][PAD]
    const int oc = threadIdx.x / 8, ch = threadIdx.x % 8 * N;
    const int oj = (c0 + oc) / a.group, oh = kvh * a.group + (c0 + oc) - oj * a.group;
    const long long orow = seq.start + oj;
    const bool out = c0 + oc < cols && orow >= 0 && orow < c.rows;
    if (half == 0) wm[wave][col] = m * a.qk_mul, wl[wave][col] = l;
#pragma unroll
    for (int pass = 0; pass < 2; pass++) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < CT / 2; u++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f16v& x = o[pass * (CT / 2) + u];
                *reinterpret_cast<f4*>(ol + (wave * UCOLS + col) * PAD + 32 * u + 2 * i + 4 * half) =
                    f4{x[i], x[i + 1], x[i + 2], x[i + 3]};
            }
        __syncthreads();
        if (!out) continue;
        float top = NEG_INF, sum = 0.0f, f[N] = {};
#pragma unroll
        for (int w = 0; w < 4; w++) top = fmaxf(top, wm[w][oc]);
        const float base = top == NEG_INF ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float s = __builtin_amdgcn_exp2f(wm[w][oc] - base);
            sum += wl[w][oc] * s;
            const float* p = ol + (w * UCOLS + oc) * PAD + ch;
#pragma unroll
            for (int i = 0; i < N; i++) f[i] += p[i] * s;
        }
        const int channel = pass * (D / 2) + ch;
        if (plot.part >= 0) {
            const long long at = (long long)(plot.part * plot.rest + plot.cut) * UCOLS + oc;
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<f4*>(a.part_o + at * D + channel + i) = f4{f[i], f[i + 1], f[i + 2], f[i + 3]};
            if (channel == 0) reinterpret_cast<f2*>(a.part_ml)[at] = f2{top, sum};
            continue;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* to = a.out.p + orow * a.out.st + oh * a.out.sh + channel;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f4 y = f4{f[i], f[i + 1], f[i + 2], f[i + 3]} * inv;
            *reinterpret_cast<uint2*>(to + i) = a.out_f16 ? make_uint2(pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]))
                                                          : make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
        }
    }
}

// The parts of the units over joined: a group of D / 8 lanes a column. Grid: UCOLS columns
// of SLOTS units.
template <int D>
__global__ __launch_bounds__(256) void picked_join(CacheAttnArgs a) {
    constexpr int LANES = D / 8, GROUPS = 256 / LANES;
    const int col = blockIdx.x * GROUPS % UCOLS + threadIdx.x / LANES, ch = (threadIdx.x % LANES) * 8;
    const Plot plot(a, blockIdx.x * GROUPS / UCOLS, true);
    if (plot.b < 0) return;
    const int at = plot.tile * UCOLS + col, j = at / a.group;
    const long long row = plot.seq.start + j;
    if (at >= plot.seq.n * a.group || row < 0 || row >= a.c.rows) return;
    float f[8];
    const long long first = (long long)plot.cut * UCOLS + col, step = (long long)plot.rest * UCOLS;
    const float l = join_parts<D, false>(a, (int)plot.parts, ch, [&](int p) { return first + p * step; }, f);
    store_row(a, row, plot.kvh * a.group + at - j * a.group, ch, f, l);
}

constexpr unsigned MOST_LDS = 40u << 10;  // of a unit's lists, beside the kernel's own: two workgroups a CU

}  // namespace

// Units at most: those of the longest rows that each sequence may have, of all rows together.
static long long most_units(int batch, int rows, int group, int kv_heads, int max_new) {
    const long long each = ((long long)max_new * group + UCOLS - 1) / UCOLS;
    const long long all = ((long long)rows * group + UCOLS - 1) / UCOLS + batch;
    return std::min(each * batch, all) * kv_heads;
}

// Whether a call runs in units of 32 columns: up to 8 heads a KV head (of 16 and more a
// unit of 16 columns is one row's, and does nothing twice), and from 64 units on; from 256
// where a wave's step is of several pages or 8 heads of 128 a KV head make a unit four
// rows'. Replayed from a graph, us, units of 16 columns and of 32, 32 pages of 64 of 16384
// tokens, the rows' picks half shared, bf16, rows of one sequence:
//                          64       96       128      160      256      1000
//   32/8 heads of 128      27 29    38 34    39 38    63 43    65 57    233 182
//   16/8 (64 units at 128) 22 26    -        31 32    46 34    47 41    155 115
//   64/8                   31 36    49 48    51 51    76 73    91 77    311 256
//   32/8 heads of 64       22 20    30 23    30 26    49 30    51 39    150 110
//   64/8                   24 23    38 32    39 33    45 47    68 50    -
//   64 pages of 16:
//   32/8 heads of 128      21 25    24 29    25 32    40 35    42 43    -
//   64/8                   19 29    31 34    31 37    50 48    58 51    -
//   32/8 heads of 64       17 18    20 20    20 22    32 25    33 31    -
// fp16 queries of 128 channels do not fit the larger unit's registers in two parts (in part in
// memory, 32/8 heads, 1000 rows: 238 and 245 us, 16 x 32: 127 and 149; 8/8 heads: 106 and 111,
// 62 and 79).
static bool wide_units(int head_dim, bool q_f16, const PickedPlan& p) { return p.chunks && !(head_dim == 128 && q_f16); }

PickedPlan picked_plan(int head_dim, int batch, int rows, int heads, int kv_heads, int max_new, int max_pages,
                       int page_tokens, int top) {
    const int group = heads / kv_heads;
    PickedPlan p{};
    const auto units = [&](int cols) { return ((long long)max_new * group + cols - 1) / cols * kv_heads * batch; };
    const auto steps = [&](int cols) {
        return ((long long)pick_entries(cols, top, group, max_new, max_pages) * page_tokens + USTEP - 1) / USTEP;
    };
    p.lds = pick_lds_bytes(16, top, group, max_new, max_pages);
    p.chunk_lds = pick_lds_bytes(UCOLS, top, group, max_new, max_pages);
    const int least = page_tokens < TOKENS || (head_dim == 128 && group > 4) ? 256 : 64;
    p.chunks = group <= 8 && (long long)max_new * group > 16 && units(UCOLS) >= least && p.chunk_lds <= MOST_LDS &&
               most_units(batch, rows, group, kv_heads, max_new) < 1 << 23;  // (of a launch's 2^32 threads)
    // Of the units over whole rounds, at most; a part is two steps or more.
    p.parts = (int)std::max(1ll, std::min((steps(UCOLS) + 1) / 2, (long long)MAX_SPLITS));
    // Units that leave CUs free have eight waves and are cut into parts, one a CU, of two
    // steps at least, but for the shortest, which a second kernel would not shorten. Replayed
    // from a graph, us, 1, 8, 16 and 32 sequences of a row, 32/8 heads of 128:
    //                                   1 part                  2                       4
    //   32 pages of 64, eight waves     16.1 16.7 18.1 22.2     13.8 14.5 17.1 31.5     11.2 12.2 21.6 31.6
    //   four waves                      21.2 22.0 23.5 25.1     15.7 16.8 18.5 24.6     11.7 12.6 17.4 24.8
    //   128 pages of 64, eight waves    47.2 50.4 51.3 63.0     29.5 32.6 36.9 69.8     19.3 25.6 43.5 69.4
    // and of 16 heads of 64, 64 pages of 16, eight waves: 9.5 9.7 10.6 16.5 and 10.0 10.7 17.2 16.5.
    const long long few = units(16);
    p.wide = few <= 256 && steps(16) > 1;
    p.splits = few > 256 || steps(16) <= 4 ? 1 : (int)std::min(256 / std::max(few, 1ll), steps(16) / 2);
    p.part_rows = std::max<uint64_t>(p.splits > 1 ? (uint64_t)p.splits * rows * heads : 0, p.chunks ? SLOTS * UCOLS : 0);
    return p;
}

hipError_t launch_cache_attend_picked(int head_dim, const CacheAttnArgs& args, const PickedPlan& plan, hipStream_t s) {
    CacheAttnArgs a = args;
    hipError_t e;
    if (wide_units(head_dim, a.q_f16, plan)) {
        a.splits = plan.parts;
        const unsigned wgs = (unsigned)most_units(a.c.batch, a.c.rows, a.group, a.c.kv_heads, a.max_new) + SLOTS;
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(wgs), dim3(256), plan.chunk_lds, s, a);
        };
        const auto of = [&](auto big) {
            constexpr bool BIG = decltype(big)::value;
            if (head_dim == 64)
                go(a.q_f16 ? picked_chunk<64, 2, BIG> : picked_chunk<64, 1, BIG>);
            else
                go(picked_chunk<128, 1, BIG>);  // (wide_units)
        };
        if (a.c.page_shift >= 6)
            of(std::true_type{});
        else
            of(std::false_type{});
        e = hipGetLastError();
        if (e != hipSuccess || a.splits == 1) return e;
        const int groups = 256 / (head_dim / 8);
        hipLaunchKernelGGL((head_dim == 64 ? picked_join<64> : picked_join<128>), dim3(SLOTS * UCOLS / groups), dim3(256), 0,
                           s, a);
        return hipGetLastError();
    }
    a.splits = plan.splits;
    e = launch_cache_attend_few_picked(head_dim, a, plan, s);
    return e == hipSuccess && a.splits > 1 ? launch_cache_join_splits(head_dim, a, s) : e;
}

}  // namespace sage
