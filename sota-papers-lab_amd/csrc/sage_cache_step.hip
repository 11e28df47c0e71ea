// A step's index from the requests' lengths (gfx950): starts, lengths, new pages,
// and each row's position, slot and sequence.
//
// Sums over the requests in front of each: of rows (its start), of new pages (its
// place in the ring) and of pages given back. One workgroup makes them, since each needs all
// before it, and every request's own numbers fit its threads' registers; the rows
// follow, in the same launch where they are few, else in one that fills the chip.
// Whether the step can be served is known before anything is written, so
// that an input may be the output of the same kind. The memory moved is 16 bytes
// a row and request, so a step is bound by latency: the loads of news and past, the sums,
// the ring (or the table) and the stores.
#include <algorithm>

#include "sage_cache.hpp"

namespace sage {

namespace {

typedef long long ll;
typedef ll ll2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 1024;  // at most, of the workgroup that makes the sums

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, int shift) {
    return (tokens >> shift) + ((tokens & ((1u << shift) - 1)) != 0);
}

// What a request asks for: rows, new pages (held: those it has), columns past
// the table, pages that it gives back. Below 2^32 all of them, and sums of them stop
// there: what a step can be served with is below 2^31.
struct Sums {
    uint32_t rows, fresh, back, over;
    __device__ __forceinline__ void operator+=(const Sums& o) {
        rows = __builtin_elementwise_add_sat(rows, o.rows), fresh = __builtin_elementwise_add_sat(fresh, o.fresh);
        back = __builtin_elementwise_add_sat(back, o.back), over = __builtin_elementwise_add_sat(over, o.over);
    }
};
struct Request {
    Sums s;
    uint32_t past, held;
    bool ended;
    __device__ __forceinline__ Request(const StepArgs& a, int news, int past_) {
        past = max(past_, 0);
        ended = news < 0;
        held = pages_of(past, a.page_shift);
        const uint32_t rows = max(news, 0), want = pages_of(past + rows, a.page_shift), most = a.max_pages;
        s = Sums{rows, ended ? 0 : want - held, ended ? min(held, most) : 0, !ended && want > most ? want - most : 0};
    }
};

// v of the lanes of CTRL's place, 0 where there is none: a step of a sum over the lanes before.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ Sums moved(const Sums& s) {
    return {moved<CTRL, ROWS>(s.rows), moved<CTRL, ROWS>(s.fresh), moved<CTRL, ROWS>(s.back), moved<CTRL, ROWS>(s.over)};
}
// Of the lanes up to each.
__device__ __forceinline__ Sums upto_lane(Sums s) {
    s += moved<0x111, 0xf>(s);  // row_shr:1, 2, 4, 8
    s += moved<0x112, 0xf>(s);
    s += moved<0x114, 0xf>(s);
    s += moved<0x118, 0xf>(s);
    s += moved<0x142, 0xa>(s);  // row_bcast:15 into rows 1 and 3
    s += moved<0x143, 0xc>(s);  // row_bcast:31 into rows 2 and 3
    return s;
}
__device__ __forceinline__ Sums of_lane(const Sums& s, int lane) {
    auto get = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); };
    return {get(s.rows), get(s.fresh), get(s.back), get(s.over)};
}

// The ring as the step finds it; numbers that make no sense are brought into range.
struct Ring {
    int head, count, cap;
    __device__ __forceinline__ Ring(const StepArgs& a) : cap(a.cap) {
        head = (int)((uint32_t)a.state_in[0] % (uint32_t)cap);
        count = min(max(a.state_in[1], 0), cap);
    }
    // The place i behind the first; i < 2^31.
    __device__ __forceinline__ int at(uint32_t i) const { return (int)(((uint32_t)head + i) % (uint32_t)cap); }
};

// One row: its page from the ring where its column is new, else from the table.
// `first`: of the request's new pages, in the ring; `held`: its columns before the step.
struct RowPlace {
    int position, sequence;
    ll slot;
};
__device__ __forceinline__ RowPlace place_row(const StepArgs& a, int b, int position, int held, int first) {
    const int col = position >> a.page_shift, in_page = (1 << a.page_shift) - 1;
    const ll cell = (ll)b * a.max_pages + col;
    int page;
    if (col >= held) {
        const ll at = (ll)first + (col - held);
        page = a.ring[at < a.cap ? at : at - a.cap];
        if ((position & in_page) == 0) a.page_table[cell] = page;  // the column's first row
    } else {
        page = a.page_table[cell];
    }
    RowPlace p{position, b, -1};
    if ((unsigned)page < (unsigned)a.pages) p.slot = ((ll)page << a.page_shift) + (position & in_page);
    return p;
}

__device__ __forceinline__ void write_row(const StepArgs& a, int row, const RowPlace& p) {
    if (a.positions) a.positions[row] = p.position;
    if (a.sequences) a.sequences[row] = p.sequence;
    if (a.slots) a.slots[row] = p.slot;
}

// The pages of an ended request, by a wave: columns 0 .. n - 1 to the ring from `to` on.
__device__ __forceinline__ void give_back(const StepArgs& a, int b, int n, int to) {
    const int lane = threadIdx.x & 63;
    for (int i = lane; i < n; i += 64) {
        const ll at = (ll)to + i;
        a.ring[at < a.cap ? at : at - a.cap] = a.page_table[(ll)b * a.max_pages + i];
    }
}

// The last request whose start is at or before the row; starts[0] = 0 and row < starts[batch].
template <class Starts>
__device__ __forceinline__ int request_of(const Starts& starts, int batch, int row) {
    int lo = 0, hi = batch;  // starts[lo] <= row < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= row)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// The sums, and with ROWS (a request a thread at most) everything else too.
// scratch [batch] gets the ring's place of each request's first page, taken or given back,
// and behind them [batch] the pages it gives back.
template <int N, bool ROWS>
__global__ __launch_bounds__(N) void step_kernel(StepArgs a) {
    __shared__ Sums waves[16];
    __shared__ int starts[ROWS ? N + 1 : 1], past_of[ROWS ? N : 1], first_of[ROWS ? N : 1], back_of[ROWS ? N : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Ring ring(a);
    const int run = ROWS ? 1 : (a.batch + N - 1) / N;
    const int b0 = min(a.batch, (int)threadIdx.x * run), b1 = min(a.batch, b0 + run);
    Sums mine{0, 0, 0, 0};
    for (int b = b0; b < b1; b++) mine += Request(a, a.news[b], a.past[b]).s;
    mine.back = min(mine.back, 1u << 31);  // past any ring: so that the sum before is too, where the sum with it stops
    Sums at = upto_lane(mine);
    if (lane == 63) waves[wave] = at;
    __syncthreads();  // (the inputs that may be outputs too are read)
    Sums all = upto_lane(lane < N / 64 ? waves[lane] : Sums{0, 0, 0, 0});
    // The sums before the thread's; exact where the step is good, and `back` up to the ring's room.
    at.rows -= mine.rows, at.fresh -= mine.fresh, at.back -= mine.back;
    if (wave) at += of_lane(all, wave - 1);
    all = of_lane(all, 15);
    const uint32_t count = ring.count, room = ring.cap - ring.count;
    uint32_t missing = all.fresh > count ? all.fresh - count : 0;
    missing = __builtin_elementwise_add_sat(missing, all.over);
    const uint32_t more = all.rows > (uint32_t)a.rows ? all.rows - a.rows : 0;
    const bool good = missing == 0 && more == 0;
    for (int b = b0; b < b1; b++) {
        const Request q(a, a.news[b], a.past[b]);
        const int start = good ? (int)at.rows : 0;
        const int first = q.ended ? ring.at(count + min(at.back, room)) : ring.at(good ? at.fresh : 0);
        const int back = at.back < room ? (int)min(q.s.back, room - at.back) : 0;
        a.starts[b] = start;
        a.lengths[b] = q.ended ? 0 : (int)(q.past + (good ? q.s.rows : 0));
        if (ROWS) {
            starts[b] = start, past_of[b] = (int)q.past, first_of[b] = first, back_of[b] = back;
        } else {
            a.scratch[b] = first;
            a.scratch[a.batch + b] = back;
        }
        at += q.s;
    }
    const int rows = good ? (int)all.rows : 0;
    if (threadIdx.x == 0) {
        a.starts[a.batch] = rows;
        if (ROWS) starts[a.batch] = rows;
        const uint32_t taken = good ? all.fresh : 0;
        a.state[0] = ring.at(taken);
        a.state[1] = (int)(count - taken + min(all.back, room));
        a.state[2] = (int)min(missing, 2147483647u);
        a.state[3] = (int)min(more, 2147483647u);
    }
    if (!ROWS) return;
    __syncthreads();
    for (int row = threadIdx.x; row < a.rows; row += N) {
        RowPlace p{0, -1, -1};
        if (row < rows) {
            const int b = request_of(starts, a.batch, row);
            p = place_row(a, b, past_of[b] + row - starts[b], (int)pages_of(past_of[b], a.page_shift), first_of[b]);
        }
        write_row(a, row, p);
    }
    if (all.back == 0) return;
    for (int b = wave; b < a.batch; b += N / 64)
        if (back_of[b]) give_back(a, b, back_of[b], first_of[b]);
}

// The request of a row below starts[batch] (another one's number for any other row), by
// a wave: 512 starts at a time, so one round of loads up to 512 requests, two up to 32768.
constexpr int AT_ONCE = 8;
__device__ __forceinline__ int request_of_wave(const int* starts, int batch, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = batch;  // starts[lo] <= row < starts[lo + n]
    while (n > 64 * AT_ONCE) {
        const int run = (n + 63) / 64, at = lo + lane * run;
        const int from = max(__builtin_popcountll(__ballot(at < lo + n && starts[at] <= row)) - 1, 0);
        n = min(run, n - from * run);
        lo += from * run;
    }
    int start[AT_ONCE], upto = 0;
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) start[i] = starts[min(lo + i * 64 + lane, batch)];
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) upto += __builtin_popcountll(__ballot(i * 64 + lane < n && start[i] <= row));
    return lo + max(upto - 1, 0);
}

// The rows of a large step, four a thread, and behind their workgroups a
// wave for each request that may have ended. A wave whose rows are all one
// request's looks it up once; others look through the starts of the next 64, row by row.
constexpr int ROWS_WG = 1024, ROWS_WAVE = ROWS_WG / 4;
__global__ __launch_bounds__(256) void step_rows_kernel(StepArgs a, int row_wgs) {
    if ((int)blockIdx.x >= row_wgs) {
        const int b = ((int)blockIdx.x - row_wgs) * 4 + (threadIdx.x >> 6);
        if (b < a.batch && a.scratch[a.batch + b]) give_back(a, b, a.scratch[a.batch + b], a.scratch[b]);
        return;
    }
    const int total = a.starts[a.batch], row0 = blockIdx.x * ROWS_WG + threadIdx.x * 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wave0 = __builtin_amdgcn_readfirstlane(row0);
    RowPlace p[4];
    const int one = __builtin_amdgcn_readfirstlane(request_of_wave(a.starts, a.batch, wave0));
    if (a.batch && wave0 + ROWS_WAVE <= a.starts[one + 1]) {
        const int start = a.starts[one], past = a.lengths[one] - (a.starts[one + 1] - start);
        const int held = (int)pages_of(past, a.page_shift), first = a.scratch[one];
        // Four tokens are of two pages at most: the first one's and the last one's.
        const int t = past + row0 - start, in_page = (1 << a.page_shift) - 1, turn = (t | in_page) + 1;
        const int* table = a.page_table + (ll)one * a.max_pages;
        auto page_of = [&](int col) {
            const uint32_t at = (uint32_t)first + (uint32_t)(col - held);
            return col < held ? table[col] : a.ring[at < (uint32_t)a.cap ? at : at - a.cap];
        };
        const int c0 = t >> a.page_shift, c1 = (t + 3) >> a.page_shift;
        const int p0 = page_of(c0), p1 = c1 == c0 ? p0 : page_of(c1);
        // The row that begins a new column writes it.
        if (c0 >= held && (t & in_page) == 0) a.page_table[(ll)one * a.max_pages + c0] = p0;
        if (c1 > c0 && c1 >= held) a.page_table[(ll)one * a.max_pages + c1] = p1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int page = t + i < turn ? p0 : p1;
            p[i] = RowPlace{t + i, one, -1};
            if ((unsigned)page < (unsigned)a.pages) p[i].slot = ((ll)page << a.page_shift) + ((t + i) & in_page);
        }
    } else {
        __shared__ int lds[4][65];
        int* next = lds[wave];
        const int most = min(64, a.batch - one);  // starts[one] .. starts[one + most]
        next[lane] = a.starts[min(one + lane, a.batch)];
        if (lane == 0) next[64] = a.starts[min(one + 64, a.batch)];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        int b = -1, start = 0, end = 0, past = 0, held = 0, first = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = row0 + i;
            p[i] = RowPlace{0, -1, -1};
            if (row >= total) continue;
            if (row >= end) {
                b = row < next[most] ? one + request_of(next, most, row) : request_of(a.starts, a.batch, row);
                start = a.starts[b], end = a.starts[b + 1];
                past = a.lengths[b] - (end - start), held = (int)pages_of(past, a.page_shift), first = a.scratch[b];
            }
            p[i] = place_row(a, b, past + row - start, held, first);
        }
    }
    if (row0 + 3 < a.rows) {
        if (a.positions)
            *reinterpret_cast<int4*>(a.positions + row0) =
                make_int4(p[0].position, p[1].position, p[2].position, p[3].position);
        if (a.sequences)
            *reinterpret_cast<int4*>(a.sequences + row0) =
                make_int4(p[0].sequence, p[1].sequence, p[2].sequence, p[3].sequence);
        if (a.slots) {
            *reinterpret_cast<ll2*>(a.slots + row0) = ll2{p[0].slot, p[1].slot};
            *reinterpret_cast<ll2*>(a.slots + row0 + 2) = ll2{p[2].slot, p[3].slot};
        }
        return;
    }
    for (int i = 0; i < 4 && row0 + i < a.rows; i++) write_row(a, row0 + i, p[i]);
}

}  // namespace

// One launch where a workgroup has the requests in its threads and few rows and
// pages to see to. Replayed from a graph, us, 64 requests:
//   rows                            64    512   1024  2048  4096  8192
//   one launch of 256 threads       2.9   3.9   5.5   8.7   15.3  28.0
//   one launch of 1024              3.4   3.7   3.9   4.8   6.7   10.3
//   two launches                    7.2   5.9   6.0   6.6   6.6   6.7
// (the eager call pays the host another 2 us for the second). A call that fills the
// chip, 512 requests of 1380301 rows together: 12.2 us for 23 MB, of which the second
// launch's chain start -> request -> page -> rows takes most; without the slots' 11 MB 10.0
// (13.0 with 64 starts at a time and a look through LDS by every workgroup of two requests; 11.6 with
// stores past the caches, which leave them to the next call's loads).
hipError_t launch_cache_step(const StepArgs& a, hipStream_t s) {
    const bool one = a.batch <= THREADS && a.rows <= 4 * THREADS && (ll)a.batch * a.max_pages <= 1 << 18;
    if (one && a.batch <= 256 && a.rows <= 256) {
        hipLaunchKernelGGL((step_kernel<256, true>), dim3(1), dim3(256), 0, s, a);
    } else if (one) {
        hipLaunchKernelGGL((step_kernel<THREADS, true>), dim3(1), dim3(THREADS), 0, s, a);
    } else {
        hipLaunchKernelGGL((step_kernel<THREADS, false>), dim3(1), dim3(THREADS), 0, s, a);
        const int row_wgs = (int)(((ll)a.rows + ROWS_WG - 1) / ROWS_WG);
        hipLaunchKernelGGL(step_rows_kernel, dim3(row_wgs + (a.batch + 3) / 4), dim3(256), 0, s, a, row_wgs);
    }
    return hipGetLastError();
}

}  // namespace sage
