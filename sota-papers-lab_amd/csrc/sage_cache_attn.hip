// Attention over the paged 4-bit cache (gfx950).
//
// out[i] = sum_t p_t V_t / sum_t p_t, p_t = 2^(x_t - m), x_t = (q_i . K_t) *
// softmax scale * log2(e), over the slots t that row i sees, with the running
// maximum m of the online softmax: one pass over the cache.
//
// E2M1 codes and an E8M0 scale are exact in bf16, and gfx950 converts two codes
// and their scale in one instruction (v_cvt_scalef32_pk_bf16_fp4), so both
// products run on the bf16 MFMA with fp32 sums: K and V enter exactly, bf16
// queries too, fp16 ones as two bf16 parts; the probabilities are rounded to
// bf16 (half a step: 2^-8 of each). The scaled FP8 x FP4 MFMA would take K's
// codes as they are, but it drops the terms of a dot product that lie some
// 2^-12 below its largest: under a channel of K with a large offset, which the
// softmax cancels, that is more than the differences between the keys.
//
// A tile's "columns" are (row, head of the group) pairs of one KV head: S^T =
// K Q^T gives each lane one column and four tokens of each 16-token tile, and
// those four are the order in which O^T = V^T P^T takes its tokens, so P goes
// from one MFMA to the next without leaving the lane's registers.
#include "sage_cache.hpp"

namespace sage {

namespace {

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int COLS = 16;    // columns of a workgroup
constexpr int TOKENS = 64;  // tokens of a wave's step
constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ uint32_t cvt2(uint32_t codes, float s, int which) {
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
__device__ __forceinline__ uint4 decode8(uint32_t codes, float s) {
    return make_uint4(cvt2(codes, s, 0), cvt2(codes, s, 1), cvt2(codes, s, 2), cvt2(codes, s, 3));
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
__device__ __forceinline__ uint32_t col_or(uint32_t v) {
    auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = r[0] | r[1];
    r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return r[0] | r[1];
}

// Tokens of one split of a sequence of len tokens: whole steps of the
// workgroup's four waves.
__device__ __forceinline__ int split_tokens(int len, int splits) {
    const int step = 4 * TOKENS;
    return ((len + splits - 1) / splits + step - 1) / step * step;
}

// One step's codes and scales of a wave, as loaded.
template <int D>
struct Step {
    uint32_t k[4][D / 32];     // [16-token tile][dwords]: token lane % 16, channels (lane / 16) * D / 4 ..
    uint4 v[D / 32];           // token lane / (D / 32) + i * 2048 / D, channels (lane % (D / 32)) * 32 ..
    uint32_t ks[4], vs[D / 32];
    int valid;  // bit i: the page of 16-token tile i is one of the pool's
};

template <int D>
__global__ __launch_bounds__(256, 2) void cache_attn(CacheAttnArgs a) {
    constexpr int G = D / 32;        // scale blocks of a row
    constexpr int VT = 64 / G;       // tokens of one V load
    constexpr int UNITS = D / 16;    // 32-byte units of a V row in LDS
    constexpr int KS = D / 32;       // MFMA steps over the channels
    __shared__ __align__(16) uint8_t lds[4][TOKENS * D * 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits, kvh = blockIdx.y, b = blockIdx.z;
    const CacheDev& c = a.c;

    // The sequence's rows and tokens.
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int c0 = tile * COLS, cols = seq.n * a.group;
    if (c0 >= cols) return;
    const int chunk = split_tokens(seq.len, a.splits), t0 = split * chunk;
    if (split && t0 >= seq.len) return;
    const int j = (c0 + col) / a.group, head = kvh * a.group + (c0 + col) - j * a.group;
    const long long row = seq.start + j;
    const bool have = c0 + col < cols && row >= 0 && row < c.rows;
    const int limit = seq.limit(j, a.causal);              // this column sees slots below it
    const int least = seq.limit(c0 / a.group, a.causal);   // every column sees these
    const int end = min(t0 + chunk, seq.limit((min(c0 + COLS, cols) - 1) / a.group, a.causal));

    // Q^T, the second operand: column lane % 16, channels in K's order.
    bf8 q[2][KS];
    {
        const uint16_t* p = a.q.p + row * a.q.st + head * a.q.sh;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (have) x = *reinterpret_cast<const uint4*>(p + g * (D / 4) + 8 * s);
            if (a.q_f16) {
                float f[8], hi[8];
                unpack8(x, f, true);
#pragma unroll
                for (int i = 0; i < 8; i++) q[0][s][i] = (__bf16)f[i], hi[i] = (float)q[0][s][i];
#pragma unroll
                for (int i = 0; i < 8; i++) q[1][s][i] = (__bf16)(f[i] - hi[i]);
            } else {
                q[0][s] = __builtin_bit_cast(bf8, x);
            }
        }
    }

    auto load = [&](int t, Step<D>& st) {
        st.valid = 0;
        long long rows[4];  // code row of each 16-token tile
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int page = cache_page(c, b, t + 16 * i);
            st.valid |= (page >= 0) << i;
            rows[i] = cache_row(c, max(page, 0), kvh, (t + 16 * i) & ((1 << c.page_shift) - 1));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint8_t* p = c.k_codes + (rows[i] + col) * (D / 2) + g * (D / 8);
            if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                st.k[i][0] = x.x, st.k[i][1] = x.y, st.k[i][2] = x.z, st.k[i][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                st.k[i][0] = x.x, st.k[i][1] = x.y;
            }
            st.ks[i] = c.k_scales[(rows[i] + col) * G + g * G / 4];
        }
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int tok = lane / G + i * VT;
            long long r = rows[(i * VT) / 16];
            if (VT == 32 && lane >= 32) r = rows[(i * VT) / 16 + 1];
            r += tok & 15;
            st.v[i] = *reinterpret_cast<const uint4*>(c.v_codes + r * (D / 2) + (lane % G) * 16);
            st.vs[i] = c.v_scales[r * G + lane % G];
        }
    };

    f4 o[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; u++) o[u] = f4{0, 0, 0, 0};
    float m = NEG_INF, l = 0.0f;
    uint8_t* vl = lds[wave];
    // Where a lane's rows of V lie: 32-byte units permuted by the token, so
    // that the eight tokens a transposing read takes at once meet all banks.
    auto unit_at = [&](int tok, int u) {
        const int f = D == 128 ? tok & 7 : (tok >> 1) & 3;
        return tok * (D * 2) + ((u ^ f) << 5);
    };

    Step<D> cur;
    const int t_first = t0 + wave * TOKENS;
    if (t_first < end) load(t_first, cur);
    for (int t = t_first; t < end; t += 4 * TOKENS) {
        Step<D> nxt;
        const bool more = t + 4 * TOKENS < end;
        if (more) load(t + 4 * TOKENS, nxt);
        // S^T, tile by tile.
        f4 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = f4{0, 0, 0, 0};
            const float s = __uint_as_float(cur.ks[i] << 23);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const bf8 kk = __builtin_bit_cast(bf8, decode8(cur.k[i][k], s));
                x[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[0][k], x[i], 0, 0, 0);
                if (a.q_f16) x[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[1][k], x[i], 0, 0, 0);
            }
        }
        // V into LDS as bf16. Blocks that are NaN go in as (almost) zeros and
        // are noted: a masked token's must not reach a row through 0 * NaN.
        uint64_t bad[G];
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int tok = lane / G + i * VT;
            const bool nan = cur.vs[i] == 255;
            bad[i] = __ballot(nan);
            const float s = __uint_as_float(nan ? 0 : cur.vs[i] << 23);
            const uint32_t w[4] = {cur.v[i].x, cur.v[i].y, cur.v[i].z, cur.v[i].w};
#pragma unroll
            for (int d = 0; d < 4; d++)
                *reinterpret_cast<uint4*>(vl + unit_at(tok, (lane % G) * 2 + d / 2) + (d & 1) * 16) = decode8(w[d], s);
        }
        // The softmax's step.
        const bool masked = t + TOKENS > least || cur.valid != 15;
        float mx = NEG_INF;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[i][r] *= a.qk_mul;
                if (masked && (t + 16 * i + 4 * g + r >= limit || !(cur.valid >> i & 1))) x[i][r] = NEG_INF;
                mx = fmaxf(mx, x[i][r]);
            }
        mx = fmaxf(m, col_max(mx));
        const float base = mx == NEG_INF ? 0.0f : mx;
        if (__any(mx > m)) {
            const float scale = __builtin_amdgcn_exp2f(m - base);
            l *= scale;
#pragma unroll
            for (int u = 0; u < UNITS; u++) o[u] *= scale;
        }
        m = mx;
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
                    if (t + tok < limit && (cur.valid >> i & 1)) hit |= blocks;
                }
            hit = col_or(hit);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[i][r] = __builtin_amdgcn_exp2f(x[i][r] - base);
                l += x[i][r];
            }
        // O^T += V^T P^T, 32 tokens a step: the lane's tokens of two tiles.
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            bf8 p;
#pragma unroll
            for (int r = 0; r < 4; r++) p[r] = (__bf16)x[i][r], p[4 + r] = (__bf16)x[i + 1][r];
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                typedef __attribute__((address_space(3))) s4* lp;
                const int tok = 16 * i + 4 * g + (col >> 2);
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(vl + unit_at(tok, u) + (col & 3) * 8));
                const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(vl + unit_at(tok + 16, u) + (col & 3) * 8));
                typedef short s8 __attribute__((ext_vector_type(8)));
                const s8 vv = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                o[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, vv), p, o[u], 0, 0, 0);
            }
        }
        if (any_bad)
#pragma unroll
            for (int u = 0; u < UNITS; u++)
                if (hit >> (u / 2) & 1) o[u] = f4{1, 1, 1, 1} * __builtin_nanf("");
        if (more) cur = nxt;
    }
    l = col_sum(l);

    // The four waves' parts meet in LDS.
    constexpr int PAD = D + 4;
    __shared__ float wm[4][COLS], wl[4][COLS];
    float* ol = reinterpret_cast<float*>(lds[0]);  // [4][COLS][PAD]
    static_assert(4 * COLS * PAD * 4 <= sizeof lds, "");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < UNITS; u++) *reinterpret_cast<f4*>(ol + (wave * COLS + col) * PAD + 16 * u + 4 * g) = o[u];
    if (g == 0) wm[wave][col] = m, wl[wave][col] = l;
    __syncthreads();
    constexpr int TPC = D / 8;  // threads a column, eight channels each
    const int oc = threadIdx.x / TPC, ch = (threadIdx.x % TPC) * 8;
    if (oc >= COLS || c0 + oc >= cols) return;
    const int oj = (c0 + oc) / a.group, oh = kvh * a.group + (c0 + oc) - oj * a.group;
    const long long orow = seq.start + oj;
    if (orow < 0 || orow >= c.rows) return;
    float top = NEG_INF, sum = 0.0f, f[8] = {};
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, wm[w][oc]);
    const float base = top == NEG_INF ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float s = __builtin_amdgcn_exp2f(wm[w][oc] - base);
        sum += wl[w][oc] * s;
        const float* p = ol + (w * COLS + oc) * PAD + ch;
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] += p[i] * s;
    }
    if (a.splits == 1) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] *= inv;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = a.out_f16 ? pack_f16x2(f[2 * i], f[2 * i + 1]) : pack_bf16x2(f[2 * i], f[2 * i + 1]);
        *reinterpret_cast<uint4*>(a.out.p + orow * a.out.st + oh * a.out.sh + ch) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        const long long at = ((long long)split * c.rows + orow) * a.heads + oh;
        float* p = a.part_o + at * D + ch;
        *reinterpret_cast<f4*>(p) = f4{f[0], f[1], f[2], f[3]};
        *reinterpret_cast<f4*>(p + 4) = f4{f[4], f[5], f[6], f[7]};
        if (ch == 0) {
            a.part_ml[at * 2] = top;
            a.part_ml[at * 2 + 1] = sum;
        }
    }
}

// The splits' parts of one (row, head) joined, in the order of the splits: a
// wave a pair, D / 64 channels a lane.
template <int D>
__global__ __launch_bounds__(256) void cache_attn_join(CacheAttnArgs a) {
    const CacheDev& c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.z;
    const SequenceIndex seq = sequence_index(c, b, a.max_new);
    const int i = blockIdx.x * 4 + wave, j = i / a.heads, h = i - j * a.heads;
    const long long row = seq.start + j;
    if (j >= seq.n || row < 0 || row >= c.rows) return;
    const int chunk = split_tokens(seq.len, a.splits), parts = seq.len ? (seq.len + chunk - 1) / chunk : 1;
    const long long at = row * a.heads + h, step = (long long)c.rows * a.heads;
    float m = NEG_INF, l = 0.0f;
    float f[D / 64] = {};
    for (int p = 0; p < parts; p++) {
        const float pm = a.part_ml[(at + p * step) * 2], pl = a.part_ml[(at + p * step) * 2 + 1];
        const float mx = fmaxf(m, pm), base = mx == NEG_INF ? 0.0f : mx;
        const float s0 = __builtin_amdgcn_exp2f(m - base), s1 = __builtin_amdgcn_exp2f(pm - base);
        l = l * s0 + pl * s1;
#pragma unroll
        for (int k = 0; k < D / 64; k++) f[k] = f[k] * s0 + a.part_o[(at + p * step) * D + lane * (D / 64) + k] * s1;
        m = mx;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* out = a.out.p + row * a.out.st + h * a.out.sh + lane * (D / 64);
#pragma unroll
    for (int k = 0; k < D / 64; k++)
        out[k] = (uint16_t)(a.out_f16 ? pack_f16x2(f[k] * inv, 0.0f) : pack_bf16x2(f[k] * inv, 0.0f));
}

}  // namespace

int cache_splits(int head_dim, int batch, int kv_heads, int group, int max_new, int max_tokens) {
    (void)head_dim;
    const long long tiles = ((long long)max_new * group + COLS - 1) / COLS;
    const long long units = tiles * kv_heads * batch;
    const long long most = (max_tokens + 511) / 512;
    return (int)std::max(1ll, std::min({most, 4096 / std::max(units, 1ll), 256ll}));
}

template <int D>
static hipError_t launch(const CacheAttnArgs& a, hipStream_t s) {
    const unsigned tiles = (unsigned)(((long long)a.max_new * a.group + COLS - 1) / COLS);
    hipLaunchKernelGGL((cache_attn<D>), dim3(tiles * a.splits, a.c.kv_heads, a.c.batch), dim3(256), 0, s, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((cache_attn_join<D>), dim3((unsigned)(((long long)a.max_new * a.heads + 3) / 4), 1, a.c.batch), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_cache_attend(int head_dim, const CacheAttnArgs& a, hipStream_t s) {
    return head_dim == 64 ? launch<64>(a, s) : launch<128>(a, s);
}

}  // namespace sage
