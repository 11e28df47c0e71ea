// Rotary positions and the paged 4-bit cache's writes and reads (gfx950).
//
// Compiled with -ffp-contract=off: every product and sum of the rotation is
// rounded in fp32 as written, and its result once to the 16-bit type, so that
// sage_cache_append's keys are those of sage_rotary_apply bit for bit.
#include <algorithm>

#include "sage_cache.hpp"

namespace sage {

namespace {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint4 pack8(const float* f, bool f16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = f16 ? pack_f16x2(f[2 * i], f[2 * i + 1]) : pack_bf16x2(f[2 * i], f[2 * i + 1]);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight channels that nothing reads again before the call's end: the hint keeps
// them from driving out the table and the lines being written (a rotation of
// 5003 rows of 96 heads of 64, 124 MB: 26 us, 30.5 without it; 14879 rows of 16
// KV heads of 64 appended and read back: 40 us, 47 without it).
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u4*>(p)));
}

__device__ __forceinline__ float load1(const uint16_t* p, bool f16) {
    return f16 ? f16_to_f32(*p) : __uint_as_float((uint32_t)*p << 16);
}

// The turns of a lane's eight channels c0 .. c0 + 7.
// VEC: rot is a multiple of 16, so that the lane's pairs are whole vectors of
// the table and its partners (HALF) those that one lane of the head holds. Other
// rots go channel by channel and load the partners one by one (5003 rows of
// 96 heads of 64, HALF: rot 64 26 us, 62 57 us; pairs of neighbours: 26 us both).
template <bool VEC>
struct Turns {
    f2 cs[8];   // channel c0 + k's pair
    int from;   // HALF: the lane of the wave that holds the lane's partners
    bool on;    // whether any of its channels turns

    // At position pos; NaN where the table has no such position.
    __device__ __forceinline__ void load(const RotaryDev& r, int pos, int c0) {
        const bool in = (unsigned)pos < (unsigned)r.table_rows;
        const f2* row = reinterpret_cast<const f2*>(r.table) + (long long)(in ? pos : 0) * (r.rot >> 1);
        const int half = r.rot >> 1;
        on = c0 < r.rot;
        from = (threadIdx.x & 63) + (c0 < half ? half : -half) / 8;
        if (!on) return;
        if (VEC) {
            const int i = r.layout ? c0 >> 1 : c0 < half ? c0 : c0 - half;
            const float4* v = reinterpret_cast<const float4*>(row + i);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (r.layout && k > 1) break;
                const float4 x = v[k];
                if (r.layout) {
                    cs[4 * k & 7] = cs[(4 * k + 1) & 7] = f2{x.x, x.y};
                    cs[(4 * k + 2) & 7] = cs[(4 * k + 3) & 7] = f2{x.z, x.w};
                } else {
                    cs[2 * k] = f2{x.x, x.y};
                    cs[2 * k + 1] = f2{x.z, x.w};
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int c = c0 + k;
                if (c < r.rot) cs[k] = row[r.layout ? c >> 1 : (c < half ? c : c - half)];
            }
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (!in) cs[k] = f2{__builtin_nanf(""), __builtin_nanf("")};
            if (r.transpose) cs[k].y = -cs[k].y;
        }
    }

    // The lane's channels raw of the row at p, turned, in x. All lanes of the
    // head call together: they exchange their channels.
    __device__ __forceinline__ void apply(const RotaryDev& r, const uint16_t* p, int c0, bool f16, uint4 raw,
                                          float (&x)[8]) const {
        unpack8(raw, x, f16);
        if (!on) return;
        if (r.layout) {
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                if (VEC || c0 + k < r.rot) {
                    const float a = x[k], b = x[k + 1];
                    x[k] = a * cs[k].x - b * cs[k].y;
                    x[k + 1] = b * cs[k].x + a * cs[k].y;
                }
            return;
        }
        const int half = r.rot >> 1;
        float z[8];
        if (VEC) {
            unpack8(make_uint4(__shfl(raw.x, from), __shfl(raw.y, from), __shfl(raw.z, from), __shfl(raw.w, from)), z,
                    f16);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (c0 + k < r.rot) z[k] = load1(p + (c0 + k < half ? c0 + k + half : c0 + k - half), f16);
        }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (VEC || c0 + k < r.rot) {
                const float t = z[k] * cs[k].y;
                x[k] = (VEC ? c0 : c0 + k) < half ? x[k] * cs[k].x - t : x[k] * cs[k].x + t;
            }
    }
};

// A workgroup's run of `parts` parts, gridDim.y of which there are (share_heads).
__device__ __forceinline__ int run_of(int parts) { return (parts + gridDim.y - 1) / gridDim.y; }

// ---- rotary ----
//
// y_a = x_a cos - x_b sin, y_b = x_b cos + x_a sin for each pair (a, b) of
// channels: 16 bits in and out and six operations a pair, so the memory bounds
// it (16126 rows of 40 heads of 128, 334 MB: 68 us, 4.9 TB/s, a large copy's rate).
// A wave holds one row's heads, D / 8 lanes a head and eight channels a lane,
// so the turns of a lane's channels are loaded once and serve every head.
// A head's loads come before its stores, all in one wave: out may be x.
// Two heads' loads are in flight together.
template <int D, bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    constexpr int CH = D / 8, SLOTS = 64 / CH, AHEAD = VEC ? 2 : 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * 4 + wave;
    if (row >= (long long)a.batch * a.tokens) return;
    const int b = (int)(row / a.tokens), t = (int)(row - (long long)b * a.tokens);
    const int c0 = (lane % CH) * 8;
    Turns<VEC> turns;
    turns.load(a.r, a.r.positions ? a.r.positions[row] : t, c0);
    const uint16_t* px = a.x.p + b * a.x.sb + t * a.x.st;
    uint16_t* po = a.out.p + b * a.out.sb + t * a.out.st;
    const int run = run_of((a.heads + SLOTS - 1) / SLOTS) * SLOTS, end = min(a.heads, (int)(blockIdx.y + 1) * run);
    for (int h = blockIdx.y * run + lane / CH; h < end; h += AHEAD * SLOTS) {
        uint4 x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (h + i * SLOTS < end) x[i] = load_once(px + (h + i * SLOTS) * a.x.sh + c0);
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (h + i * SLOTS < end) {
                float f[8];
                turns.apply(a.r, px + (h + i * SLOTS) * a.x.sh, c0, a.f16, x[i], f);
                *reinterpret_cast<uint4*>(po + (h + i * SLOTS) * a.out.sh + c0) = pack8(f, a.f16);
            }
    }
}

// Workgroups in y that share the heads of a row among them, a run of heads
// each: all the parts (a workgroup's heads at a time) where there are few
// rows, and fewer as the rows fill the chip by themselves, so that what a
// thread looks up for its row serves several heads. blocks: workgroups of the
// rows; fill: workgroups that are enough. 1024 for the rotation (the 5003 rows
// above, before the hint: 30.8 us, 32 with 2048, 45 with 8192), 1536 for the
// append (6000 rows of 40 KV heads of 128, with the read: 70 us, 76 with 1024,
// 73 with 2048), 4096 for the read, whose loads are a quarter as wide (46875 rows
// of 8 KV heads of 128: 51.6 us, 53.5 with 2048 and with 8192).
unsigned share_heads(long long blocks, long long parts, long long fill) {
    return (unsigned)std::min(parts, std::max(1ll, (fill + blocks - 1) / blocks));
}

// ---- append and read ----

// Four lanes' 32 channels -> their scale byte and each lane's four code bytes.
// The least e with top <= 6 * 2^e: 6 * 2^e = 1.5 * 2^(e + 2), so top's
// exponent less two, and one more where its mantissa is over 1.5. Bytes 1 ..
// 253 (a block of zeros or of values under 2^-124: 1).
__device__ __forceinline__ uint32_t encode(const float (&x)[8], uint32_t& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
    if (top >= 0x7f800000u) {
        scale = 255;
        return 0;
    }
    const int e = (int)((top + 0x3fffffu) >> 23) - 2;
    scale = (uint32_t)max(e, 1);
    const float s = __uint_as_float(scale << 23);
    uint32_t codes = 0;  // v_cvt_scalef32_pk_fp4_f32: x / s, nearest, ties to the even code
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], s, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], s, 3);
    return codes;
}

// The place of a row in the pool. Every thread of a workgroup asks; up to
// STARTS - 1 sequences are looked through in LDS, one load instead of a chain.
constexpr int STARTS = 1024;
struct Place {
    int b, slot, page;
    long long at;  // the slot's code row for KV head 0
};
__device__ __forceinline__ Place place_of(CacheDev c, int row, int* starts) {
    if (c.batch < STARTS) {
        for (int i = threadIdx.x; i <= c.batch; i += blockDim.x) starts[i] = c.starts[i];
        __syncthreads();
        c.starts = starts;
    }
    Place p{-1, -1, -1, 0};
    if (row >= c.rows) return p;
    p.b = sequence_of(c, row);
    if (p.b < 0) return p;
    p.slot = slot_of(c, p.b, row);
    p.page = cache_page(c, p.b, p.slot);
    p.at = cache_row(c, max(p.page, 0), 0, p.slot & ((1 << c.page_shift) - 1));
    return p;
}

// The append reads 16-bit rows and writes 17/64 of their bytes; the memory
// bounds it (14879 rows of 16 KV heads of 64, 77 MB in 23 us: 3.3 TB/s; a part's
// code rows come from pieces of one head, 128 bytes of each row), and a
// step's 64 rows the launch and four loads in a row (the sequence, its length,
// its page and the table): 5.5 us.
// Grid: x = rows in steps of a workgroup's; y = shares of the parts, which are
// the KV heads of K, then of V, then the query heads. A workgroup's rows are
// consecutive and of one head at a time: their code rows are consecutive
// too, so the stores fill whole lines. Two parts' loads are ahead of the two at
// work, the first two ahead of the lookups.
template <int D, bool VEC>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr int CH = D / 8, ROWS = 256 / CH, AHEAD = VEC ? 2 : 1;
    __shared__ int starts[STARTS];
    const int c0 = ((int)threadIdx.x % CH) * 8, row = blockIdx.x * ROWS + threadIdx.x / CH;
    const int kv = a.c.kv_heads, parts = 2 * kv + (a.q.p ? a.heads : 0);
    const int run = run_of(parts), end = min(parts, (int)(blockIdx.y + 1) * run);
    auto is_v = [&](int part) { return part >= kv && part < 2 * kv; };
    auto row_of = [&](int part) {
        const RowView& in = part >= 2 * kv ? a.q : is_v(part) ? a.v : a.k;
        return in.p + row * in.st + (part >= 2 * kv ? part - 2 * kv : is_v(part) ? part - kv : part) * in.sh;
    };
    uint4 next[AHEAD];
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (row < a.c.rows && first + i < end) next[i] = load_once(row_of(first + i) + c0);
    };
    load(blockIdx.y * run);
    const Place place = place_of(a.c, row, starts);
    if (place.b < 0) return;
    Turns<VEC> turns;
    turns.on = false;
    if (a.r.table) turns.load(a.r, a.r.positions ? a.r.positions[row] : place.slot, c0);
    for (int first = blockIdx.y * run; first < end; first += AHEAD) {
        uint4 raw[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) raw[i] = next[i];
        load(first + AHEAD);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int part = first + i;
            if (part >= end) break;
            float x[8];
            if (!is_v(part) && turns.on) {
                turns.apply(a.r, row_of(part), c0, a.f16, raw[i], x);
                raw[i] = pack8(x, a.f16);
            }
            if (part >= 2 * kv) {
                *reinterpret_cast<uint4*>(a.q_out.p + row * a.q_out.st + (part - 2 * kv) * a.q_out.sh + c0) = raw[i];
                continue;
            }
            unpack8(raw[i], x, a.f16);
            uint32_t scale;
            const uint32_t codes = encode(x, scale);
            if (place.page < 0) continue;
            const long long at = place.at + ((long long)(is_v(part) ? part - kv : part) << a.c.page_shift);
            uint8_t* code = is_v(part) ? a.c.v_codes : a.c.k_codes;
            uint8_t* sc = is_v(part) ? a.c.v_scales : a.c.k_scales;
            *reinterpret_cast<uint32_t*>(code + at * (D / 2) + c0 / 2) = codes;
            if (c0 % CACHE_BLOCK == 0) sc[at * (D / CACHE_BLOCK) + c0 / CACHE_BLOCK] = (uint8_t)scale;
        }
    }
}

// The other way in the same grid: 17/64 of the bytes in, the rest out. Four
// parts' loads, of four bytes and one a lane, are in flight together (46875 rows of
// 8 KV heads of 128, 243 MB: 51.6 us, 4.7 TB/s; one part at a time 57).
template <int D>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
    constexpr int CH = D / 8, ROWS = 256 / CH, AHEAD = 4;
    __shared__ int starts[STARTS];
    const int c0 = ((int)threadIdx.x % CH) * 8, row = blockIdx.x * ROWS + threadIdx.x / CH, kv = a.c.kv_heads;
    const Place place = place_of(a.c, row, starts);
    if (place.b < 0) return;
    const int run = run_of(2 * kv), end = min(2 * kv, (int)(blockIdx.y + 1) * run);
    for (int first = blockIdx.y * run; first < end; first += AHEAD) {
        uint32_t codes[AHEAD], scales[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int part = first + i;
            if (part >= end) break;
            const bool is_v = part >= kv;
            codes[i] = scales[i] = 0;  // a slot that holds nothing: zeros
            if (place.page < 0) continue;
            const long long at = place.at + ((long long)(is_v ? part - kv : part) << a.c.page_shift);
            codes[i] = *reinterpret_cast<const uint32_t*>((is_v ? a.c.v_codes : a.c.k_codes) + at * (D / 2) + c0 / 2);
            scales[i] = (is_v ? a.c.v_scales : a.c.k_scales)[at * (D / CACHE_BLOCK) + c0 / CACHE_BLOCK];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int part = first + i;
            if (part >= end) break;
            const bool is_v = part >= kv;
            const float s = __uint_as_float(scales[i] << 23);  // 255: infinity, which the conversion turns into NaN
            const f2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], s, 0),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], s, 1),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], s, 2),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], s, 3)};
            float x[8];
#pragma unroll
            for (int k = 0; k < 4; k++) x[2 * k] = v[k].x, x[2 * k + 1] = v[k].y;
            const RowView& o = is_v ? a.v : a.k;
            *reinterpret_cast<uint4*>(o.p + row * o.st + (is_v ? part - kv : part) * o.sh + c0) = pack8(x, a.f16);
        }
    }
}

}  // namespace

hipError_t launch_rotary(int head_dim, const RotaryArgs& a, hipStream_t s) {
    const long long blocks = ((long long)a.batch * a.tokens + 3) / 4;
    const int slots = 64 / (head_dim / 8);
    const dim3 grid((unsigned)blocks, share_heads(blocks, std::min(65535, (a.heads + slots - 1) / slots), 1024));
    const bool vec = a.r.rot % 16 == 0;
    if (head_dim == 64)
        hipLaunchKernelGGL((vec ? rotary_kernel<64, true> : rotary_kernel<64, false>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((vec ? rotary_kernel<128, true> : rotary_kernel<128, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_cache_append(int head_dim, const AppendArgs& a, hipStream_t s) {
    const int rows = 256 / (head_dim / 8);
    const long long blocks = ((long long)a.c.rows + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, share_heads(blocks, 2 * a.c.kv_heads + (a.q.p ? a.heads : 0), 1536));
    const bool vec = a.r.rot % 16 == 0;  // (no rotation: 0)
    if (head_dim == 64)
        hipLaunchKernelGGL((vec ? append_kernel<64, true> : append_kernel<64, false>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((vec ? append_kernel<128, true> : append_kernel<128, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_cache_read(int head_dim, const ReadArgs& a, hipStream_t s) {
    const int rows = 256 / (head_dim / 8);
    const long long blocks = ((long long)a.c.rows + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, share_heads(blocks, 2 * a.c.kv_heads, 4096));
    if (head_dim == 64)
        hipLaunchKernelGGL(read_kernel<64>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(read_kernel<128>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace sage
