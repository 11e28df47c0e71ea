// Attention over the paged 4-bit cache (gfx950).
//
// out[i] = sum_t p_t V_t / sum_t p_t, p_t = 2^(x_t - m), x_t = (q_i . K_t) *
// softmax scale * log2(e), over the slots t that row i sees, with the running
// maximum m of the online softmax: one pass over the cache.
//
// E2M1 codes and an E8M0 scale are exact in bf16, and gfx950 converts two codes
// and their scale in one instruction (v_cvt_scalef32_pk_bf16_fp4), so both
// products run on the bf16 MFMA with fp32 sums: K and V enter exactly, bf16
// queries too, fp16 ones as two bf16 parts. The scaled FP8 x FP4 MFMA would take
// K's codes as they are, but it drops the terms of a dot product that lie some
// 2^-12 below its largest: under a channel of K with a large offset, which the
// softmax cancels, that is more than the differences between the keys.
//
// The probabilities enter the second product as two bf16 parts (half a step of
// half a step: 2^-16 of each); one part, 2^-8 of each, would be an error of the
// size of a bf16 output's own rounding (0.0023 against 64 bits where the output
// alone has 0.0017). Decoding has the room (2% of 63 sequences of up to 16384
// tokens, 7% of 8 rows of 8 sequences behind 20000), chunks do not
// (cache_attn_chunk).
//
// A tile's "columns" are (row, head of the group) pairs of one KV head: S^T =
// K Q^T gives each lane one column and four tokens of each 16-token tile, and
// those four are the order in which O^T = V^T P^T takes its tokens, so P goes
// from one MFMA to the next without leaving the lane's registers.
#include <algorithm>

#include "sage_cache_attn.hpp"

namespace sage {

namespace {

// ---- Few rows ----
//
// The work of a call is a line of units, one for each (sequence, KV head, tile
// of 16 columns), and a unit is a step for each 256 of the sequence's tokens,
// after one more for its beginning and end. The line is cut into equal
// shares, one a workgroup, as many as the chip holds at once: sequences of any
// lengths end together, and only the units that a cut goes through leave
// partial outputs, two a workgroup at most.
// The cache is read once, at one pass's worth of MFMA and conversions beside
// it: the memory bounds it. 63 sequences of up to 16384 tokens (517438 in all),
// 32/8 heads of 128, one row each: 564 MB in 121 us, 4.7 TB/s. (When it took
// 119, cut into equal parts of each sequence instead: 137 us at the best number
// of parts; in twice as many shares as the chip holds: 132.)
constexpr int COLS = 16;  // columns of a workgroup
constexpr int STEP = 4 * TOKENS;

struct Units {
    int steps, tiles;  // of the sequence: steps of a unit's tokens, column tiles (0: no rows)
    __device__ __forceinline__ Units(const CacheAttnArgs& a, const SequenceIndex& s) {
        steps = max(1, (s.len + STEP - 1) / STEP);
        tiles = (s.n * a.group + COLS - 1) / COLS;
    }
    __device__ __forceinline__ long long cost(const CacheDev& c) const {
        return (long long)c.kv_heads * tiles * (steps + 1);
    }
};

// The line as every wave sums it: each lane a run of sequences, `before` the
// runs before the lane's.
struct Line {
    long long before, total;
    int run;
    __device__ __forceinline__ Line(const CacheAttnArgs& a, int lane) {
        const CacheDev& c = a.c;
        run = (c.batch + 63) / 64;
        const int b0 = min(c.batch, lane * run), b1 = min(c.batch, b0 + run);
        long long sum = 0;
#pragma unroll 4
        for (int b = b0; b < b1; b++) sum += Units(a, sequence_index(c, b, a.max_new)).cost(c);
        long long upto = sum;
        for (int d = 1; d < min(64, c.batch); d *= 2) {
            const long long v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        before = upto - sum;
        total = uniform(upto, (c.batch - 1) / run);
    }
};

// Steps of a share; at least two, so that a share is more than a unit's first step.
__device__ __forceinline__ long long share_of(long long total, int wgs) { return max(2ll, (total + wgs - 1) / wgs); }

// QP: bf16 parts of a query. W: waves, four, or eight for whole units that do
// not fill the chip (cache_plan). PICKED: the units' tokens are those of picked
// pages, in a.splits equal parts a unit, a workgroup each: 63 rows of 32 pages of 64,
// 32/8 heads of 128, 134 MB in 36 us, some 5 of them index, lists and page ids one behind the
// other and the rest at a copy's rate.
template <int D, int QP, int W, bool PICKED>
__global__ __launch_bounds__(64 * W, D == 64 && W == 4 ? 3 : 2) void cache_attn(CacheAttnArgs a) {
    constexpr int G = D / 32;        // scale blocks of a row
    constexpr int VT = 64 / G;       // tokens of one V load
    constexpr int UNITS = D / 16;    // 32-byte units of a V row in LDS
    constexpr int KS = D / 32;       // MFMA steps over the channels
    constexpr int PAD = D + 4;       // floats of a column where the waves' parts meet
    constexpr int HALF = TOKENS / 2; // tokens of V in LDS at a time, per wave
    constexpr int LDS = W * (HALF * D * 2 > COLS * PAD * 4 ? HALF * D * 2 : COLS * PAD * 4);
    __shared__ __align__(16) uint8_t lds[LDS];
    extern __shared__ uint32_t pick_lds[];  // PICKED: entries_of's
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const CacheDev& c = a.c;

    // This workgroup's share [pos, stop) of the line, and the sequence b that it
    // begins in, whose part of the line begins at base_b. Or one whole unit.
    int b;
    long long pos, stop, base_b;
    SequenceIndex seq;
    if constexpr (PICKED) {
        b = blockIdx.z, base_b = 0, pos = 0, stop = 1;
        seq = sequence_index(c, b, a.max_new);
    } else if (a.whole) {
        b = blockIdx.z, base_b = 0;
        seq = sequence_index(c, b, a.max_new);
        const Units units(a, seq);
        const int kvh = blockIdx.x % c.kv_heads, tile = blockIdx.x / c.kv_heads;
        if (tile >= units.tiles) return;
        pos = ((long long)kvh * units.tiles + tile) * (units.steps + 1);
        stop = pos + units.steps + 1;
    } else {
        const Line line(a, lane);
        const long long share = share_of(line.total, gridDim.x);
        pos = blockIdx.x * share;
        stop = min(line.total, pos + share);
        if (pos >= stop) return;
        // The last lane whose run begins at pos or before has it in its run.
        const int at = 63 - __builtin_clzll(__ballot(line.before <= pos && lane * line.run < c.batch));
        base_b = uniform(line.before, at);
        b = at * line.run;
        while (true) {
            seq = sequence_index(c, b, a.max_new);
            const long long cost = Units(a, seq).cost(c);
            if (pos < base_b + cost || b >= c.batch - 1) break;
            base_b += cost;
            b++;
        }
    }
    while (pos < stop) {
        const Units units(a, seq);
        if (units.tiles == 0) return;
        const SequenceIndex now = seq;
        const int b_now = b;
        int kvh, tile, s0, s1, split = 0;
        bool whole;
        if constexpr (PICKED) {
            kvh = blockIdx.x % c.kv_heads, split = blockIdx.x / c.kv_heads % a.splits;
            tile = blockIdx.x / c.kv_heads / a.splits;
            if (tile >= units.tiles) return;
            pos = stop;
            whole = a.splits == 1;
        } else {
            const long long idx = (pos - base_b) / (units.steps + 1), begin = base_b + idx * (units.steps + 1);
            const long long next = begin + units.steps + 1;
            kvh = (int)(idx / units.tiles), tile = (int)(idx - (long long)kvh * units.tiles);
            s0 = (int)max(0ll, pos - begin - 1), s1 = (int)(min(stop, next) - begin - 1);
            pos = next;
            if (next >= base_b + units.cost(c)) {  // on to the next sequence that has rows
                base_b = next;
                while (pos < stop && b < c.batch - 1) {
                    seq = sequence_index(c, ++b, a.max_new);
                    if (seq.n) break;
                }
            }
            if (s1 <= s0) continue;  // no more than the unit's beginning
            whole = s0 == 0 && s1 == units.steps;
        }
        const int c0 = tile * COLS, cols = now.n * a.group;
        const int j0 = c0 / a.group, j1 = (min(c0 + COLS, cols) - 1) / a.group;  // its rows
        Entries entries{};
        if constexpr (PICKED) {
            const int pages = (now.limit(j1, a.causal) + (1 << c.page_shift) - 1) >> c.page_shift;
            entries = entries_of<W, COLS>(a, now, b_now, kvh, j0, j1 - j0 + 1, pages, pick_lds);
            const int steps = ((entries.count << c.page_shift) + STEP - 1) / STEP;
            s0 = (int)((long long)steps * split / a.splits), s1 = (int)((long long)steps * (split + 1) / a.splits);
        }
        const long long part = 2ll * blockIdx.x + (s0 == 0);
        const int t0 = s0 * STEP;
        const int j = (c0 + col) / a.group, head = kvh * a.group + (c0 + col) - j * a.group;
        const long long row = now.start + j;
        const bool have = c0 + col < cols && row >= 0 && row < c.rows;
        const int limit = now.limit(j, a.causal);              // this column sees slots below it
        const int least = now.limit(j0, a.causal);             // every column sees these
        // (a picked unit's tokens are its entries')
        const int end = min(s1 * STEP, PICKED ? entries.count << c.page_shift : now.limit(j1, a.causal));

        // Q^T, the second operand: column lane % 16, channels in K's order.
        bf8 q[QP][KS];
        {
            const uint16_t* p = a.q.p + row * a.q.st + head * a.q.sh;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (have) x = load_q(p + g * (D / 4) + 8 * s, a.q_sign);
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
        }

        const int t_first = t0 + wave * TOKENS;
        using Source = std::conditional_t<PICKED, Walk, Pages>;
        auto source = [&] {
            if constexpr (PICKED)
                return Source(entries, c.page_shift, lane, t_first);
            else
                return Source(c, b_now, lane, t_first);
        };
        Source pages = source();
        const uint32_t every = (2u << (j1 - j0)) - 1;  // picked by all rows
        // One step's codes and scales: K's token lane % 16 of each 16-token tile,
        // channels (lane / 16) * D / 4 on; V's token lane / G + i * VT, block lane % G.
        struct Step {
            uint32_t k[4][KS], ks[4];
            uint4 v[G];
            uint32_t vs[G];
            int valid;  // bit i: the page of 16-token tile i is one of the pool's
            int slot[PICKED ? 4 : 1];  // of its first token
            uint32_t rows[PICKED ? 4 : 1];
        };
        // Slot of the first token of 16-token tile i at t, and whether the lane's column
        // sees token k of the tile.
        auto slot_at = [&](int t, int i, const Step& st) {
            return PICKED ? st.slot[PICKED ? i : 0] : t + 16 * i;
        };
        auto sees = [&](int t, int i, int k, const Step& st) {
            return slot_at(t, i, st) + k < limit && (st.valid >> i & 1) &&
                   (!PICKED || (st.rows[PICKED ? i : 0] >> (j - j0) & 1));
        };
        auto row_of = [&](int t, int page) {
            return cache_row(c, max(page, 0), kvh, t & ((1 << c.page_shift) - 1));
        };
        auto load = [&](int t, Step& st) {
            st.valid = 0;
            long long rows[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                int page;
                if constexpr (PICKED)
                    page = pages.of(t + 16 * i, st.slot[i], st.rows[i]);
                else
                    page = pages.of(t + 16 * i);
                st.valid |= (page >= 0) << i;
                rows[i] = row_of(t + 16 * i, page);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint8_t* p = c.k_codes + rows[i] * (D / 2) + (uint32_t)(col * (D / 2) + g * (D / 8));
                if constexpr (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p);
                    st.k[i][0] = x.x, st.k[i][1] = x.y, st.k[i][2] = x.z, st.k[i][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(p);
                    st.k[i][0] = x.x, st.k[i][1] = x.y;
                }
                st.ks[i] = (c.k_scales + rows[i] * G)[(uint32_t)(col * G + g * G / 4)];
            }
#pragma unroll
            for (int i = 0; i < G; i++) {
                long long r = rows[(i * VT) / 16];
                if (VT == 32 && lane >= 32) r = rows[(i * VT) / 16 + 1];
                r += lane / G & 15;
                st.v[i] = *reinterpret_cast<const uint4*>(c.v_codes + r * (D / 2) + (lane % G) * 16);
                st.vs[i] = c.v_scales[r * G + lane % G];
            }
        };

        f4 o[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; u++) o[u] = f4{0, 0, 0, 0};
        float m = NEG_INF, l = 0.0f;
        uint8_t* vl = lds + wave * (HALF * D * 2);

        // Two steps in registers, taken in turns: the loop does both.
        Step one, two;
        auto step = [&](int t, const Step& st) __attribute__((always_inline)) {
            // S^T, tile by tile.
            f4 x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = f4{0, 0, 0, 0};
                const float s = __uint_as_float(st.ks[i] << 23);
#pragma unroll
                for (int n = 0; n < KS; n++) {
                    const bf8 kk = __builtin_bit_cast(bf8, decode8(st.k[i][n], s));
#pragma unroll
                    for (int p = 0; p < QP; p++)
                        x[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[p][n], x[i], 0, 0, 0);
                }
            }
            const int there = st.valid;
            // Blocks of V that are NaN go into LDS as (almost) zeros and are noted:
            // a masked token's must not reach a row through 0 * NaN.
            uint64_t bad[G];
#pragma unroll
            for (int i = 0; i < G; i++) bad[i] = __ballot(st.vs[i] >= V_NAN);
            // The softmax's step.
            bool masked = there != 15;
            if constexpr (PICKED) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    masked = masked || st.slot[i] + 16 > least || st.rows[i] != every;
            } else {
                masked = masked || t + TOKENS > least;
            }
            float mx = NEG_INF;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (masked && !sees(t, i, 4 * g + r, st)) x[i][r] = NEG_INF;
                    mx = fmaxf(mx, x[i][r]);
                }
            mx = fmaxf(m, col_max(mx));
            if (__any((mx - m) * a.qk_mul > SLACK)) {
                const float scale = __builtin_amdgcn_exp2f((m - (mx == NEG_INF ? 0.0f : mx)) * a.qk_mul);
                m = mx;
                l *= scale;
#pragma unroll
                for (int u = 0; u < UNITS; u++) o[u] *= scale;
            }
            const float base = m == NEG_INF ? 0.0f : m * a.qk_mul;
            uint32_t hit = 0;  // blocks of NaN that this lane's tokens bring to its column
            uint64_t any_bad = 0;
#pragma unroll
            for (int i = 0; i < G; i++) any_bad |= bad[i];
            if (any_bad) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int tok = 16 * i + 4 * g + r;
                        const uint32_t blocks = (uint32_t)(bad[16 * i / VT] >> (tok % VT * G)) & ((1u << G) - 1);
                        if (sees(t, i, 4 * g + r, st)) hit |= blocks;
                    }
                hit = col_or(hit);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    x[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][r], a.qk_mul, -base));
                    l += x[i][r];
                }
            // O^T += V^T P^T, 32 tokens a step: V into the wave's part of LDS as
            // bf16, then the lane's tokens of two tiles.
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
#pragma unroll
                for (int n = i * G / 4; n < (i + 2) * G / 4; n++) {
                    const float s = __uint_as_float(st.vs[n] >= V_NAN ? 0 : st.vs[n] << 23);
                    const uint32_t w[4] = {st.v[n].x, st.v[n].y, st.v[n].z, st.v[n].w};
#pragma unroll
                    for (int d = 0; d < 4; d++)
                        *reinterpret_cast<uint4*>(vl + unit_at<D>((lane / G + n * VT) % HALF, (lane % G) * 2 + d / 2,
                                                                  d & 1)) = decode8(w[d], s);
                }
                float e[8];
#pragma unroll
                for (int r = 0; r < 8; r++) e[r] = x[i + r / 4][r % 4];
                bf8 p[2];
                parts_of<2>(e, p);
#pragma unroll
                for (int u = 0; u < UNITS; u++) {
                    const uint8_t* at = vl + unit_at<D>(4 * g + (col >> 2), u, col >> 1 & 1) + (col & 1) * 8;
                    const bf8 vv = read_v(at, 16 * (D * 2));
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        o[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, p[k], o[u], 0, 0, 0);
                }
            }
            if (any_bad) {
                asm volatile("" : "+v"(hit));  // a branch, not a select of every sum in every step
#pragma unroll
                for (int u = 0; u < UNITS; u++)
                    if (hit >> (u / 2) & 1) o[u] = f4{1, 1, 1, 1} * __builtin_nanf("");
            }
        };
        constexpr int STRIDE = W * TOKENS;
        if (t_first < end) load(t_first, one);
        for (int t = t_first; t < end; t += 2 * STRIDE) {
            if (t + STRIDE < end) load(t + STRIDE, two);
            step(t, one);
            if (t + STRIDE >= end) break;
            if (t + 2 * STRIDE < end) load(t + 2 * STRIDE, one);
            step(t + STRIDE, two);
        }
        l = col_sum(l);

        // The waves' parts meet in LDS.
        __shared__ float wm[W][COLS], wl[W][COLS];
        float* ol = reinterpret_cast<float*>(lds);  // [W][COLS][PAD]
        __syncthreads();
#pragma unroll
        for (int u = 0; u < UNITS; u++) *reinterpret_cast<f4*>(ol + (wave * COLS + col) * PAD + 16 * u + 4 * g) = o[u];
        if (g == 0) wm[wave][col] = m * a.qk_mul, wl[wave][col] = l;
        __syncthreads();
        constexpr int TPC = D / 8;  // threads a column, eight channels each
        const int oc = threadIdx.x / TPC, ch = (threadIdx.x % TPC) * 8;
        if (oc < COLS && c0 + oc < cols) {
            const int oj = (c0 + oc) / a.group, oh = kvh * a.group + (c0 + oc) - oj * a.group;
            const long long orow = now.start + oj;
            float top = NEG_INF, sum = 0.0f, f[8] = {};
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, wm[w][oc]);
            const float base = top == NEG_INF ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float s = __builtin_amdgcn_exp2f(wm[w][oc] - base);
                sum += wl[w][oc] * s;
                const float* p = ol + (w * COLS + oc) * PAD + ch;
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] += p[i] * s;
            }
            if (!whole) {
                if (PICKED && (orow < 0 || orow >= c.rows)) return;
                const long long at = PICKED ? ((long long)split * c.rows + orow) * a.heads + oh : part * COLS + oc;
                float* p = a.part_o + at * D + ch;
                *reinterpret_cast<f4*>(p) = f4{f[0], f[1], f[2], f[3]};
                *reinterpret_cast<f4*>(p + 4) = f4{f[4], f[5], f[6], f[7]};
                if (ch == 0) reinterpret_cast<f2*>(a.part_ml)[at] = f2{top, sum};
            } else if (orow >= 0 && orow < c.rows) {
                store_row(a, orow, oh, ch, f, sum);
            }
        }
        if (PICKED) return;
        __syncthreads();  // LDS is the next unit's
    }
}

// ---- Chunks of rows ----
//
// 128 columns a workgroup, 32 a wave, over tiles of 64 tokens. Each thread
// loads 16 (D = 64: 8) bytes of K's and V's codes two tiles ahead; V goes into
// LDS as 16-bit values, K as the codes, which every wave converts for itself
// (one instruction for two codes, beside the MFMAs of the logits): 16-bit keys
// would take a wave's reads of a tile from 20 KB to 32 and the workgroup's
// writes as well, where LDS is active 39% of the time now; which of the two is
// faster was not measured. Chunks of 2048 rows behind 8190 tokens, 32/8 heads of
// 128 (425 GFLOP): 466 us, 0.91 PFLOP/s; the chip's clock falls to 1.9 GHz
// under it, with the MFMA pipe busy 47% of the time.
//
// For a bf16 output the weights are fp16 (2^-11 of each) and V goes through the
// fp16 MFMA, while its scales are within HALF_LEAST .. HALF_MOST, where codes times
// scale are exact normal fp16 values as well; from the first tile with a block
// that fp16 does not hold on, a second loop, entered once, takes two bf16 parts.
// Two parts everywhere took the chunks above from 427 us to 565, fp16 from 448
// to 460 (another box).
constexpr int CCOLS = 128;
// V's scale bytes whose values, 0.5 to 6 times the scale, are normal fp16
// numbers: 2^-13 to 2^13.
constexpr uint32_t HALF_LEAST = 114, HALF_MOST = 140;
// Weights of fp16 are 2^LIFT times those of bf16, from 2^-21 on normal numbers and
// 2^15 at most; the reference that goes with their sums is as much lower.
constexpr float LIFT = 7.0f;
// Whether a scale byte is past HALF_LEAST .. HALF_MOST, and whether its block is
// more than fp16 holds: NaN, or codes (its dwords or'ed) other than zeros.
__device__ __forceinline__ bool past_half(uint32_t scale) { return scale - HALF_LEAST > HALF_MOST - HALF_LEAST; }
__device__ __forceinline__ bool past_half(uint32_t scale, uint32_t codes) {
    return past_half(scale) && (scale >= V_NAN || (codes & 0x77777777u));
}
template <int D>
struct ChunkLds {
    uint8_t v[2][TOKENS * D * 2];
    uint8_t k[2][TOKENS * D / 2];
    uint32_t ks[2][TOKENS];      // the token's scale bytes
    uint64_t bad[2][4];          // V blocks that are NaN, bit (token % 16) * 4 + block, by 16 tokens
    int flags[2][4];             // by 16 tokens: 1 bad blocks, 2 no page, 4 past fp16
};

// QP: bf16 parts of a query. OUT16: the output is fp16.
template <int D, int QP, bool OUT16>
__global__ __launch_bounds__(256, 2) void cache_attn_chunk(CacheAttnArgs a) {
    constexpr int G = D / 32, KS = D / 16, CT = D / 32, WORDS = D / 32;  // WORDS: code dwords a thread loads
    __shared__ __align__(16) ChunkLds<D> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const CacheDev& c = a.c;
    const int b = blockIdx.z, kvh = blockIdx.x % c.kv_heads, at = blockIdx.x / c.kv_heads, split = at % a.splits;
    const int tile = gridDim.x / c.kv_heads / a.splits - 1 - at / a.splits;  // the last rows see most: first
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int first = tile * CCOLS, cols = seq.n * a.group;
    if (first >= cols) return;
    const int chunk = split_tokens(seq.len, a.splits), t0 = split * chunk;
    if (split && t0 >= seq.len) return;
    const int c0 = first + 32 * wave;  // this wave's columns
    const int least = seq.limit(c0 / a.group, a.causal);
    const int end = min(t0 + chunk, seq.limit((min(first + CCOLS, cols) - 1) / a.group, a.causal));
    const int j = (c0 + col) / a.group, head = kvh * a.group + (c0 + col) - j * a.group;
    const long long row = seq.start + j;
    const bool have = c0 + col < cols && row >= 0 && row < c.rows;
    const int limit = seq.limit(j, a.causal);  // this column sees slots below it
    bf8 q[QP][KS];
    {
        const uint16_t* p = a.q.p + row * a.q.st + head * a.q.sh + half * (D / 2);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (have) x = load_q(p + 8 * s, a.q_sign);
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
    }

    // This thread's part of a tile: token tok of the tile, 4 * WORDS bytes of
    // codes. A wave's sixteen tokens are of one page: its place is scalar, and
    // the thread's offset in it never changes.
    const int tok = threadIdx.x >> 2, part = threadIdx.x & 3;
    const uint32_t code_at = (tok & 15) * (D / 2) + part * (D / 8), scale_at = (tok & 15) * G;
    const int in_page = (1 << c.page_shift) - 1, head0 = kvh << c.page_shift, page_rows = c.kv_heads << c.page_shift;
    struct Part {
        uint32_t w[WORDS], sc;
    } kr, vr;
    bool v_there = false;
    Pages pages(c, b, lane, t0 + 16 * wave);
    auto page_of = [&](int t) { return t < end ? pages.of(t + 16 * wave) : -1; };
    auto load_codes = [&](const uint8_t* p, Part& r) {
        if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + code_at);
            r.w[0] = x.x, r.w[1] = x.y, r.w[2] = x.z, r.w[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(p + code_at);
            r.w[0] = x.x, r.w[1] = x.y;
        }
    };
    auto load = [&](int t) {
        const int page = page_of(t);
        const long long row0 = (long long)max(page, 0) * page_rows + (head0 + ((t + 16 * wave) & in_page));
        load_codes(c.k_codes + row0 * (D / 2), kr);
        load_codes(c.v_codes + row0 * (D / 2), vr);
        const uint8_t* p = c.k_scales + row0 * G;
        kr.sc = D == 128 ? *reinterpret_cast<const uint32_t*>(p + scale_at)
                         : *reinterpret_cast<const uint16_t*>(p + scale_at);
        vr.sc = (c.v_scales + row0 * G)[scale_at + part * G / 4];
        v_there = page >= 0;
    };
    const int k_at = D == 128 ? tok * 64 + ((part ^ (tok >> 1 & 3)) << 4)
                              : tok * 32 + (((part >> 1) ^ (tok >> 2 & 1)) << 4) + (part & 1) * 8;
    auto store_k = [&](int buf) {  // the row's 16-byte units permuted by the token
        if constexpr (D == 128)
            *reinterpret_cast<uint4*>(lds.k[buf] + k_at) = make_uint4(kr.w[0], kr.w[1], kr.w[2], kr.w[3]);
        else
            *reinterpret_cast<uint2*>(lds.k[buf] + k_at) = make_uint2(kr.w[0], kr.w[1]);
        lds.ks[buf][tok] = kr.sc;  // (four threads, one value)
    };
    auto store_v = [&](int buf, auto fp16) {
        constexpr bool H16 = decltype(fp16)::value;
        uint32_t sc = vr.sc;
        int flag = v_there ? 0 : 2;
        if (H16) {
            if (__any(past_half(sc))) {
                uint32_t codes = 0;
#pragma unroll
                for (int w = 0; w < WORDS; w++) codes |= vr.w[w];
                if (__any(past_half(sc, codes))) flag |= 4;
            }
        } else {
            const bool nan = sc >= V_NAN;
            const uint64_t bad = __ballot(D == 128 ? nan : nan && !(part & 1));
            if (bad) lds.bad[buf][wave] = bad, flag |= 1;
            if (nan) sc = 0;
        }
        lds.flags[buf][wave] = flag;
        const float s = __uint_as_float(sc << 23);
#pragma unroll
        for (int w = 0; w < WORDS; w++) {
            const int ch = part * (D / 4) + 8 * w;
            *reinterpret_cast<uint4*>(lds.v[buf] + unit_at<D>(tok, ch / 16, ch >> 3 & 1)) = decode8<H16>(vr.w[w], s);
        }
    };

    f16v o[CT];
#pragma unroll
    for (int u = 0; u < CT; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[u][i] = 0.0f;
    float m = NEG_INF, l = 0.0f, lift = OUT16 ? 0.0f : LIFT;
    // Where a lane reads K's codes, and the place of a transposing read of V:
    // lanes 0-15 and 32-47 the first 16 of 32 channels, tokens 4 * half +
    // (lane % 16) / 4.
    const int kx = D == 128 ? (col >> 1 & 3) : (col >> 2 & 1);
    const int kr_at = col * (D / 2), ks_shift = half * (KS / 4) * 8;
    const int vtok = 4 * half + (lane >> 2 & 3), vunit = lane >> 4 & 1;
    auto scores = [&](int buf, int sub, f16v& y) {
#pragma unroll
        for (int i = 0; i < 16; i++) y[i] = 0.0f;
        uint32_t w[KS];
#pragma unroll
        for (int u = 0; u < KS / 4; u++) {
            const uint4 z = *reinterpret_cast<const uint4*>(lds.k[buf] + sub * 32 * (D / 2) + kr_at +
                                                            (((D == 128 ? half * 2 + u : half) ^ kx) << 4));
            w[4 * u] = z.x, w[4 * u + 1] = z.y, w[4 * u + 2] = z.z, w[4 * u + 3] = z.w;
        }
        const uint32_t sc = lds.ks[buf][32 * sub + col] >> ks_shift;
        const float sf[2] = {__uint_as_float((sc & 255) << 23), __uint_as_float((sc >> 8 & 255) << 23)};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const bf8 kk = __builtin_bit_cast(bf8, decode8(w[s], sf[s / 4]));
#pragma unroll
            for (int p = 0; p < QP; p++) y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kk, q[p][s], y, 0, 0, 0);
        }
    };

    // The tiles from t on, with fp16 weights (H16) until a scale of V is past
    // them; returns where they stopped, in every wave alike.
    auto walk = [&](int t, auto fp16) __attribute__((always_inline)) {
        constexpr bool H16 = decltype(fp16)::value;
        if (t < end) {
            load(t);
            store_k(0);
            store_v(0, fp16);
            load(t + TOKENS);
        }
        __syncthreads();
        int buf = 0;
        for (; t < end; t += TOKENS, buf ^= 1) {
            int4 fl = *reinterpret_cast<const int4*>(lds.flags[buf]);
            if (t + TOKENS < end) {
                store_k(buf ^ 1);
                store_v(buf ^ 1, fp16);
                load(t + 2 * TOKENS);
            }
            f16v x[2];
            scores(buf, 0, x[0]);
            scores(buf, 1, x[1]);
            // The flags are waited for here, not where they are read (head dim 64, 2 x 1500
            // rows behind 3000 tokens, 16 heads: 79.1 us against 81.4).
            asm volatile("" : "+v"(fl.x), "+v"(fl.y), "+v"(fl.z), "+v"(fl.w));
            const int flags = __builtin_amdgcn_readfirstlane(fl.x | fl.y | fl.z | fl.w);
            if (H16 && flags & 4) return t;
            uint32_t hit = 0;
            if (flags || t + TOKENS > least) {
                const int fi[4] = {fl.x, fl.y, fl.z, fl.w};
#pragma unroll
                for (int sub = 0; sub < 2; sub++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int k = 32 * sub + 8 * (i / 4) + 4 * half + i % 4, six = 2 * sub + i / 8;
                        const bool seen = t + k < limit && !(fi[six] & 2);
                        if (!seen) x[sub][i] = NEG_INF;
                        if (!H16 && flags & 1) {
                            const uint32_t blocks = (uint32_t)(lds.bad[buf][six] >> ((k & 15) * 4)) & 15;
                            if (seen && (fi[six] & 1)) hit |= blocks;
                        }
                    }
                if (!H16 && flags & 1) {
                    auto r = __builtin_amdgcn_permlane32_swap(hit, hit, false, false);
                    hit = r[0] | r[1];
                }
            }
            float mx = NEG_INF;
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
            const float base = (m == NEG_INF ? 0.0f : m * a.qk_mul) - (H16 ? LIFT : 0.0f);
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[sub][8 * st + i], a.qk_mul, -base));
                        l += e[i];
                    }
                    bf8 p[2];
                    if constexpr (H16)
                        p[0] = __builtin_bit_cast(bf8, make_uint4(pack_f16x2(e[0], e[1]), pack_f16x2(e[2], e[3]),
                                                                  pack_f16x2(e[4], e[5]), pack_f16x2(e[6], e[7])));
                    else
                        parts_of<2>(e, p);
#pragma unroll
                    for (int u = 0; u < CT; u++) {
                        const uint8_t* at = lds.v[buf] + (32 * sub + 16 * st) * (D * 2) +
                                            unit_at<D>(vtok, 2 * u + vunit, lane >> 1 & 1) + (lane & 1) * 8;
                        const bf8 vv = read_v(at, 8 * (D * 2));
                        if constexpr (H16) {
                            o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, vv),
                                                                          __builtin_bit_cast(h8, p[0]), o[u], 0, 0, 0);
                        } else {
#pragma unroll
                            for (int k = 0; k < 2; k++)
                                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv, p[k], o[u], 0, 0, 0);
                        }
                    }
                }
            if (!H16 && flags & 1) {
                asm volatile("" : "+v"(hit));  // a branch, not a select of every sum in every step
#pragma unroll
                for (int u = 0; u < CT; u++)
                    if (hit >> (D == 128 ? u : 2 * u) & 1)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[u][i] = __builtin_nanf("");
            }
            __syncthreads();
        }
        return t;
    };
    if constexpr (OUT16) {
        walk(t0, std::false_type{});
    } else {
        const int t = walk(t0, std::true_type{});
        if (t < end) {
            lift = 0.0f;
            l *= __builtin_amdgcn_exp2f(-LIFT);
#pragma unroll
            for (int u = 0; u < CT; u++) o[u] *= __builtin_amdgcn_exp2f(-LIFT);
            __syncthreads();  // every wave has read the tile's flags
            pages.fill((t + 16 * wave) >> c.page_shift);
            walk(t, std::false_type{});
        }
    }
    {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (!have) return;
    // A lane holds four channels of each eight of its column.
    if (a.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = a.out.p + row * a.out.st + head * a.out.sh;
#pragma unroll
        for (int u = 0; u < CT; u++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f4 f = f4{o[u][i], o[u][i + 1], o[u][i + 2], o[u][i + 3]} * inv;
                const uint2 w = a.out_f16 ? make_uint2(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]))
                                          : make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
                *reinterpret_cast<uint2*>(out + 32 * u + 2 * i + 4 * half) = w;
            }
    } else {
        const long long at = ((long long)split * c.rows + row) * a.heads + head;
#pragma unroll
        for (int u = 0; u < CT; u++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f4*>(a.part_o + at * D + 32 * u + 2 * i + 4 * half) =
                    f4{o[u][i], o[u][i + 1], o[u][i + 2], o[u][i + 3]};
        if (half == 0) {
            a.part_ml[at * 2] = m * a.qk_mul - lift;
            a.part_ml[at * 2 + 1] = l;
        }
    }
}

// The splits of chunks joined, a group of D / 8 lanes a (row, head); SHARE: a workgroup.
template <int D, bool SHARE>
__global__ __launch_bounds__(256) void cache_chunk_join(CacheAttnArgs a) {
    constexpr int LANES = D / 8, GROUPS = 256 / LANES;
    const CacheDev& c = a.c;
    const int b = blockIdx.z, grp = threadIdx.x / LANES, ch = (threadIdx.x % LANES) * 8;
    const int pair = SHARE ? blockIdx.x : blockIdx.x * GROUPS + grp, j = pair / a.heads, h = pair - j * a.heads;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const long long row = seq.start + j;
    if (j >= seq.n || row < 0 || row >= c.rows) return;  // (SHARE: all threads or none)
    const int chunk = split_tokens(seq.len, a.splits);
    const int parts = a.picked ? a.splits : seq.len ? (seq.len + chunk - 1) / chunk : 1;
    const long long first = row * a.heads + h, step = (long long)c.rows * a.heads;
    float f[8];
    const float l = join_parts<D, SHARE>(a, parts, ch, [&](int p) { return first + p * step; }, f);
    if (!SHARE || grp == 0) store_row(a, row, h, ch, f, l);
}

// The units that more than one share has joined: grid x column tiles (SHARE:
// columns) of a sequence, y KV heads, z sequences. wgs: cache_attn's grid.
template <int D, bool SHARE>
__global__ __launch_bounds__(256) void cache_attn_join(CacheAttnArgs a, int wgs) {
    constexpr int LANES = D / 8;
    const CacheDev& c = a.c;
    const int b = blockIdx.z, kvh = blockIdx.y, grp = threadIdx.x / LANES, ch = (threadIdx.x % LANES) * 8;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const Units units(a, seq);
    const int tile = SHARE ? blockIdx.x / COLS : blockIdx.x;
    if (tile >= units.tiles) return;
    const Line line(a, threadIdx.x & 63);
    const long long share = share_of(line.total, wgs);
    long long begin = uniform(line.before, b / line.run);
    for (int i = b / line.run * line.run; i < b; i++) begin += Units(a, sequence_index(c, i, a.max_new)).cost(c);
    begin += (long long)(kvh * units.tiles + tile) * (units.steps + 1) + 1;  // its first token step
    const long long w0 = begin / share, w1 = (begin + units.steps - 1) / share;
    if (w0 == w1) return;  // one share had it all and wrote its rows
    const int col = SHARE ? blockIdx.x % COLS : grp, at = tile * COLS + col, j = at / a.group;
    if (col >= COLS || at >= seq.n * a.group) return;  // (SHARE: all threads or none)
    const long long row = seq.start + j;
    float f[8];
    // The first share's part is its tail, every other's its head.
    const float l = join_parts<D, SHARE>(
        a, (int)(w1 - w0 + 1), ch, [&](int p) { return (2 * (w0 + p) + (p == 0)) * COLS + col; }, f);
    if (row >= 0 && row < c.rows && (!SHARE || grp == 0)) store_row(a, row, kvh * a.group + at - j * a.group, ch, f, l);
}

}  // namespace

// Whether a call runs the chunk kernel: above 64 columns, over which the other
// kernel would read and convert a tile's keys more than four times, and with
// keys to split or tiles that fill the chip. The other kernel and the chunk
// kernel, us, behind 20000 tokens, 32/8 heads of 128 (4 columns a row):
//              1 sequence   2           4            8
//   12 rows    26  30       38   37     57   58      102  104
//   16 rows    27  31       40   40     67   60      130  105
//   17 rows    35  32       51   40     82   60      155  107
//   64 rows    65  51       113  66     205  114     425  206
// 16 heads of 64 (a column a row), 8 sequences: 48 rows 114 and 126 (fp16 120 and
// 178), 64 rows 146 and 127 (fp16 151 and 178), 66 rows 177 and 128 (183 and
// 179). Of 49 to 64 columns the chunk kernel would be the faster one for bf16
// and the slower one for fp16, and a shape does not say which it is. Over 1500
// states, 6 sequences, 16 heads: 448 rows of 64 28 and 32 (fp16 30 and 45), of
// 128 45 and 45 (47 and 64); 100 rows of 64 20 and 21.
static bool in_chunks(int batch, int kv_heads, int group, int max_new, int max_tokens) {
    const long long cols = (long long)max_new * group;
    return cols > 64 && (max_tokens > 2048 || (cols + CCOLS - 1) / CCOLS * kv_heads * batch >= 512);
}

CachePlan cache_plan(int head_dim, int batch, int rows, int heads, int kv_heads, int max_new, int max_tokens) {
    CachePlan p{};
    const int group = heads / kv_heads;
    p.chunks = in_chunks(batch, kv_heads, group, max_new, max_tokens);
    const long long per = p.chunks ? CCOLS : COLS;
    const long long units = ((long long)max_new * group + per - 1) / per * kv_heads * batch;
    if (p.chunks) {
        // Two workgroups a CU fill the chip (four sequences' 64 rows behind 20000
        // tokens, 32/8 heads of 128: 116 us, 131 with half as many, 127 with twice);
        // a split is 512 tokens at least.
        const long long most = (max_tokens + 511) / 512;
        p.wgs = (int)std::max(1ll, std::min({most, 512 / std::max(units, 1ll), (long long)MAX_SPLITS}));
        p.part_rows = p.wgs > 1 ? (uint64_t)p.wgs * rows * heads : 0;
    } else {
        // As many shares as the chip holds workgroups (three a CU, two at head
        // dim 128), no more than the steps that there can be.
        const long long steps = units * ((max_tokens + STEP - 1) / STEP + 1);
        p.wgs = (int)std::max(1ll, std::min<long long>(head_dim == 64 ? 768 : 512, (steps + 1) / 2));
        // Units of a few steps that fill the chip run whole, a workgroup each
        // (a decoder's 448 rows of 16 heads over 1500 states, six sequences: 34 us
        // against 43 in shares); so do units of four steps at most, which a second
        // kernel would not shorten (16 heads over 778 tokens, four waves: 10.6 us against 14),
        // and more sequences than the shares are cheap to find among, which fill
        // the chip whatever their lengths.
        p.whole = max_tokens <= 4 * STEP || batch > 512 || (max_tokens <= 8 * STEP && units >= p.wgs);
        // Whole units that leave CUs free have eight waves, so half as many turns
        // (16 heads over 778 tokens 8.3 us against 9.1, 32/8 heads of 128 over 901
        // tokens 9.7 against 10.8, 32 sequences of them 11.5 against 12.9).
        p.wide = p.whole && units <= 256 && max_tokens > STEP;
        p.part_rows = p.whole ? 0 : 2ull * p.wgs * COLS;
    }
    return p;
}

// Many parts of few columns are joined by a workgroup a column (20000 tokens,
// 32/8 heads of 128: one row each of 2 sequences 21.5 us against 24, of 8 47.7
// against 46.8; chunks of 32 rows 37.4 against 39.3, of 128 76 against 70).
template <int D>
static void join_splits(const CacheAttnArgs& a, hipStream_t s) {
    const long long pairs = (long long)a.max_new * a.heads;
    constexpr int PER = 256 / (D / 8);
    if (a.splits > 8 && pairs * a.c.batch <= 2048)
        hipLaunchKernelGGL((cache_chunk_join<D, true>), dim3((unsigned)pairs, 1, a.c.batch), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((cache_chunk_join<D, false>), dim3((unsigned)((pairs + PER - 1) / PER), 1, a.c.batch),
                           dim3(256), 0, s, a);
}

template <int D>
static hipError_t launch(const CacheAttnArgs& a, const CachePlan& plan, hipStream_t s) {
    const dim3 block(256);
    const unsigned per = plan.chunks ? CCOLS : COLS, heads = a.c.kv_heads, batch = a.c.batch;
    const unsigned tiles = (unsigned)(((long long)a.max_new * a.group + per - 1) / per);
    // KV heads run fastest: the workgroups that read one head's keys are eight or
    // a multiple of it apart where there are as many heads, so on one XCD, whose
    // L2 holds that head's pages and not a part of all (chunks of 2048 rows behind 8190
    // tokens, 32/8 heads of 128: 445 us, 481 with the tiles fastest, fp16 336
    // and 384; 1327 rows over 1500 states, 16 heads of 64: 30.7 and 33.5).
    const auto few = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, a.whole ? dim3(heads * tiles, 1, batch) : dim3(plan.wgs),
                           dim3(plan.wide ? 512 : 256), 0, s, a);
    };
    const auto chunk = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(heads * tiles * a.splits, 1, batch), block, 0, s, a);
    };
    if (plan.chunks) {
        if (a.q_f16)
            chunk(a.out_f16 ? cache_attn_chunk<D, 2, true> : cache_attn_chunk<D, 2, false>);
        else
            chunk(a.out_f16 ? cache_attn_chunk<D, 1, true> : cache_attn_chunk<D, 1, false>);
    } else if (a.q_f16) {
        few(plan.wide ? cache_attn<D, 2, 8, false> : cache_attn<D, 2, 4, false>);
    } else {
        few(plan.wide ? cache_attn<D, 1, 8, false> : cache_attn<D, 1, 4, false>);
    }
    if (plan.chunks) {
        if (a.splits > 1) join_splits<D>(a, s);
    } else if (!a.whole) {
        if ((long long)tiles * heads * batch <= 32)
            hipLaunchKernelGGL((cache_attn_join<D, true>), dim3(tiles * COLS, heads, batch), block, 0, s, a, plan.wgs);
        else
            hipLaunchKernelGGL((cache_attn_join<D, false>), dim3(tiles, heads, batch), block, 0, s, a, plan.wgs);
    }
    return hipGetLastError();
}

hipError_t launch_cache_attend(int head_dim, const CacheAttnArgs& a, const CachePlan& plan, hipStream_t s) {
    return head_dim == 64 ? launch<64>(a, plan, s) : launch<128>(a, plan, s);
}

hipError_t launch_cache_attend_few_picked(int head_dim, const CacheAttnArgs& a, const PickedPlan& plan, hipStream_t s) {
    const unsigned tiles = (unsigned)(((long long)a.max_new * a.group + COLS - 1) / COLS);
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(tiles * a.splits * a.c.kv_heads, 1, a.c.batch), dim3(plan.wide ? 512 : 256),
                           plan.lds, s, a);
    };
    const auto of = [&](auto waves) {
        constexpr int W = decltype(waves)::value;
        if (head_dim == 64)
            go(a.q_f16 ? cache_attn<64, 2, W, true> : cache_attn<64, 1, W, true>);
        else
            go(a.q_f16 ? cache_attn<128, 2, W, true> : cache_attn<128, 1, W, true>);
    };
    if (plan.wide)
        of(std::integral_constant<int, 8>{});
    else
        of(std::integral_constant<int, 4>{});
    return hipGetLastError();
}

hipError_t launch_cache_join_splits(int head_dim, const CacheAttnArgs& a, hipStream_t s) {
    head_dim == 64 ? join_splits<64>(a, s) : join_splits<128>(a, s);
    return hipGetLastError();
}

}  // namespace sage
