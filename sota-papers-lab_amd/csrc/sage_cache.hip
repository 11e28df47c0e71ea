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

__device__ __forceinline__ uint4 pack8(const float* f, bool f16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = f16 ? pack_f16x2(f[2 * i], f[2 * i + 1]) : pack_bf16x2(f[2 * i], f[2 * i + 1]);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float load1(const uint16_t* p, bool f16) {
    return f16 ? f16_to_f32(*p) : __uint_as_float((uint32_t)*p << 16);
}

// cos and sin of the rotation pairs of a lane's eight channels c0 .. c0 + 7 at
// `pos` (pair k of channel c0 + k under HALF; pairs c0 / 2 + k / 2 under
// PAIRS), NaN where the table has no such position.
__device__ __forceinline__ void load_turns(const RotaryDev& r, int pos, int c0, f2 (&cs)[8]) {
    const bool in = (unsigned)pos < (unsigned)r.table_rows;
    const f2* row = reinterpret_cast<const f2*>(r.table) + (long long)(in ? pos : 0) * (r.rot >> 1);
    const int half = r.rot >> 1;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int c = c0 + k;
        const int i = r.layout ? c >> 1 : (c < half ? c : c - half);
        if (c < r.rot) cs[k] = row[i];
        if (!in) cs[k] = f2{__builtin_nanf(""), __builtin_nanf("")};
        if (r.transpose) cs[k].y = -cs[k].y;
    }
}

// Channels c0 .. c0 + 7 of the row at `p`, rotated (x: the channels as they
// are, on return as they go out).
__device__ __forceinline__ void turn(const RotaryDev& r, const uint16_t* p, int c0, const f2 (&cs)[8], bool f16,
                                     float (&x)[8]) {
    if (c0 >= r.rot) return;
    if (r.layout) {
#pragma unroll
        for (int k = 0; k < 8; k += 2)
            if (c0 + k < r.rot) {
                const float a = x[k], b = x[k + 1];
                x[k] = a * cs[k].x - b * cs[k].y;
                x[k + 1] = b * cs[k].x + a * cs[k].y;
            }
        return;
    }
    const int half = r.rot >> 1;
    float y[8];
    if ((half & 7) == 0) {  // the partners are eight channels of one vector
        unpack8(*reinterpret_cast<const uint4*>(p + (c0 < half ? c0 + half : c0 - half)), y, f16);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (c0 + k < r.rot) y[k] = load1(p + (c0 + k < half ? c0 + k + half : c0 + k - half), f16);
    }
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (c0 + k < r.rot) {
            const float t = y[k] * cs[k].y;
            x[k] = c0 + k < half ? x[k] * cs[k].x - t : x[k] * cs[k].x + t;
        }
}

// ---- rotary ----
//
// A wave holds one row's heads, D / 8 lanes a head and eight channels a lane,
// so the turns of a lane's channels are loaded once and serve every head.
// A head's loads come before its stores, all in one wave: out may be x.
template <int D>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    constexpr int CH = D / 8, SLOTS = 64 / CH;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * 4 + wave;
    if (row >= (long long)a.batch * a.tokens) return;
    const int b = (int)(row / a.tokens), t = (int)(row - (long long)b * a.tokens);
    const int c0 = (lane % CH) * 8;
    f2 cs[8];
    load_turns(a.r, a.r.positions ? a.r.positions[row] : t, c0, cs);
    for (int h = blockIdx.y * SLOTS + lane / CH; h < a.heads; h += gridDim.y * SLOTS) {
        const uint16_t* p = a.x.p + b * a.x.sb + t * a.x.st + h * a.x.sh;
        uint16_t* o = a.out.p + b * a.out.sb + t * a.out.st + h * a.out.sh;
        float x[8];
        unpack8(*reinterpret_cast<const uint4*>(p + c0), x, a.f16);
        turn(a.r, p, c0, cs, a.f16, x);
        *reinterpret_cast<uint4*>(o + c0) = pack8(x, a.f16);
    }
}

// Workgroups in y that share the heads of a row among them: all the parts
// (steps of a workgroup's heads) where there are few rows, and fewer as the
// rows fill the chip by themselves, so that what a thread looks up for its row
// serves several heads. blocks: workgroups of the rows.
unsigned share_heads(long long blocks, long long parts) {
    return (unsigned)std::min(parts, std::max(1ll, (4096 + blocks - 1) / blocks));
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

// Grid: x = rows in steps of a workgroup's; y = shares of the parts, which are
// the KV heads of K, then of V, then the query heads. A workgroup's rows are
// consecutive and of one head at a time: their code rows are consecutive
// too, so the stores fill whole lines.
template <int D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr int CH = D / 8, ROWS = 256 / CH;
    __shared__ int starts[STARTS];
    const int c0 = ((int)threadIdx.x % CH) * 8, row = blockIdx.x * ROWS + threadIdx.x / CH;
    const int kv = a.c.kv_heads, parts = 2 * kv + (a.q.p ? a.heads : 0);
    const Place place = place_of(a.c, row, starts);
    if (place.b < 0) return;
    f2 cs[8];
    if (a.r.table) load_turns(a.r, a.r.positions ? a.r.positions[row] : place.slot, c0, cs);
    for (int part = blockIdx.y; part < parts; part += gridDim.y) {
        const bool is_v = part >= kv && part < 2 * kv, is_q = part >= 2 * kv;
        const int h = is_q ? part - 2 * kv : is_v ? part - kv : part;
        const RowView& in = is_q ? a.q : is_v ? a.v : a.k;
        const uint16_t* p = in.p + row * in.st + h * in.sh;
        float x[8];
        unpack8(*reinterpret_cast<const uint4*>(p + c0), x, a.f16);
        if (!is_v && a.r.table) {
            turn(a.r, p, c0, cs, a.f16, x);
            const uint4 y = pack8(x, a.f16);
            if (is_q) {
                *reinterpret_cast<uint4*>(a.q_out.p + row * a.q_out.st + h * a.q_out.sh + c0) = y;
                continue;
            }
            unpack8(y, x, a.f16);
        }
        uint32_t scale;
        const uint32_t codes = encode(x, scale);
        if (place.page < 0) continue;
        const long long at = place.at + ((long long)h << a.c.page_shift);
        uint8_t* code = is_v ? a.c.v_codes : a.c.k_codes;
        uint8_t* sc = is_v ? a.c.v_scales : a.c.k_scales;
        *reinterpret_cast<uint32_t*>(code + at * (D / 2) + c0 / 2) = codes;
        if (c0 % CACHE_BLOCK == 0) sc[at * (D / CACHE_BLOCK) + c0 / CACHE_BLOCK] = (uint8_t)scale;
    }
}

template <int D>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
    constexpr int CH = D / 8, ROWS = 256 / CH;
    __shared__ int starts[STARTS];
    const int c0 = ((int)threadIdx.x % CH) * 8, row = blockIdx.x * ROWS + threadIdx.x / CH, kv = a.c.kv_heads;
    const Place place = place_of(a.c, row, starts);
    if (place.b < 0) return;
    for (int part = blockIdx.y; part < 2 * kv; part += gridDim.y) {
        const bool is_v = part >= kv;
        const int h = is_v ? part - kv : part;
        float x[8] = {};
        if (place.page >= 0) {
            const long long at = place.at + ((long long)h << a.c.page_shift);
            const uint32_t codes =
                *reinterpret_cast<const uint32_t*>((is_v ? a.c.v_codes : a.c.k_codes) + at * (D / 2) + c0 / 2);
            const uint32_t sc = (is_v ? a.c.v_scales : a.c.k_scales)[at * (D / CACHE_BLOCK) + c0 / CACHE_BLOCK];
            const float s = __uint_as_float(sc << 23);  // 255: infinity, which the conversion turns into NaN
            const f2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3)};
#pragma unroll
            for (int k = 0; k < 4; k++) x[2 * k] = v[k].x, x[2 * k + 1] = v[k].y;
        }
        const RowView& o = is_v ? a.v : a.k;
        *reinterpret_cast<uint4*>(o.p + row * o.st + h * o.sh + c0) = pack8(x, a.f16);
    }
}

}  // namespace

hipError_t launch_rotary(int head_dim, const RotaryArgs& a, hipStream_t s) {
    const long long blocks = ((long long)a.batch * a.tokens + 3) / 4;
    const int slots = 64 / (head_dim / 8);
    const dim3 grid((unsigned)blocks, share_heads(blocks, std::min(65535, (a.heads + slots - 1) / slots)));
    if (head_dim == 64)
        hipLaunchKernelGGL(rotary_kernel<64>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(rotary_kernel<128>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_cache_append(int head_dim, const AppendArgs& a, hipStream_t s) {
    const int rows = 256 / (head_dim / 8);
    const long long blocks = ((long long)a.c.rows + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, share_heads(blocks, 2 * a.c.kv_heads + (a.q.p ? a.heads : 0)));
    if (head_dim == 64)
        hipLaunchKernelGGL(append_kernel<64>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(append_kernel<128>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_cache_read(int head_dim, const ReadArgs& a, hipStream_t s) {
    const int rows = 256 / (head_dim / 8);
    const long long blocks = ((long long)a.c.rows + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, share_heads(blocks, 2 * a.c.kv_heads));
    if (head_dim == 64)
        hipLaunchKernelGGL(read_kernel<64>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(read_kernel<128>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace sage
