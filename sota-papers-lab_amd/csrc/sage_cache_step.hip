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

constexpr int THREADS = 1024;

__device__ __forceinline__ ll pages_of(ll tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

// What a request asks for: rows, new pages (held: those it has), columns past
// the table, pages that it gives back.
struct Request {
    ll rows, fresh, over, back, past, held;
    bool ended;
    __device__ __forceinline__ Request(const StepArgs& a, int news, int past_) {
        past = max(past_, 0);
        ended = news < 0;
        rows = max(news, 0);
        held = pages_of(past, a.page_shift);
        const ll want = pages_of(past + rows, a.page_shift);
        fresh = ended ? 0 : want - held;
        over = ended ? 0 : max(0ll, want - a.max_pages);
        back = ended ? min(held, (ll)a.max_pages) : 0;
    }
};

struct Sums {
    ll rows, fresh, back, over;
    __device__ __forceinline__ void operator+=(const Sums& o) {
        rows += o.rows, fresh += o.fresh, back += o.back, over += o.over;
    }
};

__device__ __forceinline__ Sums shfl_up(const Sums& s, int d) {
    return {__shfl_up(s.rows, d), __shfl_up(s.fresh, d), __shfl_up(s.back, d), __shfl_up(s.over, d)};
}

// The ring as the step finds it; numbers that make no sense are brought into range.
struct Ring {
    int head, count, cap;
    __device__ __forceinline__ Ring(const StepArgs& a) : cap(a.cap) {
        head = (int)((uint32_t)a.state_in[0] % (uint32_t)cap);
        count = min(max(a.state_in[1], 0), cap);
    }
    __device__ __forceinline__ int at(ll i) const { return (int)((head + i) % cap); }
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
template <bool ROWS>
__global__ __launch_bounds__(THREADS) void step_kernel(StepArgs a) {
    __shared__ Sums waves[THREADS / 64];
    __shared__ int starts[ROWS ? THREADS + 1 : 1], past_of[ROWS ? THREADS : 1], first_of[ROWS ? THREADS : 1],
        back_of[ROWS ? THREADS : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Ring ring(a);
    const int run = (a.batch + THREADS - 1) / THREADS;
    const int b0 = min(a.batch, (int)threadIdx.x * run), b1 = min(a.batch, b0 + run);
    Sums mine{0, 0, 0, 0};
    for (int b = b0; b < b1; b++) {
        const Request q(a, a.news[b], a.past[b]);
        mine += Sums{q.rows, q.fresh, q.back, q.over};
    }
    Sums upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const Sums o = shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 63) waves[wave] = upto;
    __syncthreads();  // (the inputs that may be outputs too are read)
    Sums all{0, 0, 0, 0}, at{0, 0, 0, 0};
    for (int w = 0; w < THREADS / 64; w++) {
        if (w == wave) at = all;
        all += waves[w];
    }
    at += upto;
    at.rows -= mine.rows, at.fresh -= mine.fresh, at.back -= mine.back;
    const ll missing = max(0ll, all.fresh - ring.count) + all.over, more = max(0ll, all.rows - a.rows);
    const bool good = missing == 0 && more == 0;
    const ll room = ring.cap - ring.count;
    for (int b = b0; b < b1; b++) {
        const Request q(a, a.news[b], a.past[b]);
        const int start = good ? (int)at.rows : 0;
        const int first = q.ended ? ring.at((ring.count + min(at.back, room))) : ring.at(good ? at.fresh : 0);
        const int back = (int)max(0ll, min(q.back, room - at.back));
        a.starts[b] = start;
        a.lengths[b] = q.ended ? 0 : (int)(q.past + (good ? q.rows : 0));
        if (ROWS) {
            starts[b] = start, past_of[b] = (int)q.past, first_of[b] = first, back_of[b] = back;
        } else {
            a.scratch[b] = first;
            a.scratch[a.batch + b] = back;
        }
        at.rows += q.rows, at.fresh += q.fresh, at.back += q.back;
    }
    const int rows = good ? (int)all.rows : 0;
    if (threadIdx.x == 0) {
        a.starts[a.batch] = rows;
        if (ROWS) starts[a.batch] = rows;
        a.state[0] = ring.at(good ? all.fresh : 0);
        a.state[1] = (int)(ring.count - (good ? all.fresh : 0) + min(all.back, room));
        a.state[2] = (int)min(missing, 2147483647ll);
        a.state[3] = (int)min(more, 2147483647ll);
    }
    if (!ROWS) return;
    __syncthreads();
    for (int row = threadIdx.x; row < a.rows; row += THREADS) {
        RowPlace p{0, -1, -1};
        if (row < rows) {
            const int b = request_of(starts, a.batch, row);
            p = place_row(a, b, past_of[b] + row - starts[b], (int)pages_of(past_of[b], a.page_shift), first_of[b]);
        }
        write_row(a, row, p);
    }
    if (all.back == 0) return;
    for (int b = wave; b < a.batch; b += THREADS / 64)
        if (back_of[b]) give_back(a, b, back_of[b], first_of[b]);
}

// The rows of a large step, four a thread, and behind their workgroups a
// wave for each request that may have ended.
constexpr int ROWS_WG = 1024, STARTS = 2048;
__global__ __launch_bounds__(256) void step_rows_kernel(StepArgs a, int row_wgs) {
    if ((int)blockIdx.x >= row_wgs) {
        const int b = ((int)blockIdx.x - row_wgs) * 4 + (threadIdx.x >> 6);
        if (b < a.batch && a.scratch[a.batch + b]) give_back(a, b, a.scratch[a.batch + b], a.scratch[b]);
        return;
    }
    __shared__ int lds[STARTS];
    const int* starts = a.starts;
    if (a.batch < STARTS) {
        for (int i = threadIdx.x; i <= a.batch; i += 256) lds[i] = a.starts[i];
        __syncthreads();
        starts = lds;
    }
    const int total = starts[a.batch], row0 = blockIdx.x * ROWS_WG + threadIdx.x * 4;
    if (row0 >= a.rows) return;
    int b = -1, start = 0, end = 0, past = 0, held = 0, first = 0;
    RowPlace p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = row0 + i;
        p[i] = RowPlace{0, -1, -1};
        if (row >= total) continue;
        if (row >= end) {
            b = request_of(starts, a.batch, row);
            start = starts[b], end = starts[b + 1];
            past = a.lengths[b] - (end - start), held = (int)pages_of(past, a.page_shift), first = a.scratch[b];
        }
        p[i] = place_row(a, b, past + row - start, held, first);
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
// pages to see to; its rounds of 1024 rows are cheaper than a second launch up to 8.
hipError_t launch_cache_step(const StepArgs& a, hipStream_t s) {
    if (a.batch <= THREADS && a.rows <= 8 * THREADS && (ll)a.batch * a.max_pages <= 1 << 18) {
        hipLaunchKernelGGL(step_kernel<true>, dim3(1), dim3(THREADS), 0, s, a);
    } else {
        hipLaunchKernelGGL(step_kernel<false>, dim3(1), dim3(THREADS), 0, s, a);
        const int row_wgs = (int)(((ll)a.rows + ROWS_WG - 1) / ROWS_WG);
        hipLaunchKernelGGL(step_rows_kernel, dim3(row_wgs + (a.batch + 3) / 4), dim3(256), 0, s, a, row_wgs);
    }
    return hipGetLastError();
}

}  // namespace sage
