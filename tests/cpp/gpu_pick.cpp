// A step's index, rotary axes, page bounds, picks and the attention over them
// through the C++ host API (include/spl_sage.hpp) on the GPU. Values are chosen so
// that the results are exact: positions of angle 0 turn nothing, equal keys give the mean of
// the values of the picked pages.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstring>
#include <vector>

#include "spl_sage.hpp"

using namespace spl_sage;

static int failures = 0;
#define CHECK(x)                                                \
    do {                                                        \
        if (!(x)) {                                             \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x); \
            failures++;                                         \
        }                                                       \
    } while (0)

static void hip_ok(hipError_t e) {
    if (e != hipSuccess) {
        std::printf("HIP error: %s\n", hipGetErrorString(e));
        std::exit(2);
    }
}

template <class T>
struct Dev {
    T* p = nullptr;
    std::size_t n;
    explicit Dev(const std::vector<T>& h) : n(h.size()) {
        hip_ok(hipMalloc((void**)&p, n * sizeof(T)));
        hip_ok(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    ~Dev() { (void)hipFree(p); }
    Dev(const Dev&) = delete;
    std::vector<T> host() const {
        std::vector<T> h(n);
        hip_ok(hipDeviceSynchronize());
        hip_ok(hipMemcpy(h.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return h;
    }
};

static uint16_t bf16(float f) {
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return (uint16_t)(u >> 16);
}
static float f32(uint16_t h) {
    const uint32_t u = (uint32_t)h << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

int main() {
    check_device(0);
    const std::size_t D = 64, H = 2, rows = 66, top = 2;
    const SageAttention sa = SageAttention::create(nullptr, D);
    // Two requests of 1 and 64 rows, one row of padding; six pages of 16, all free.
    const cache::CacheShape shape{2, rows, 64, H, 1, 6, 16, 4};
    Dev<int32_t> news({1, 64}), past({0, 0}), ring({5, 0, 2, 3, 1, 4}), state({0, 6, 0, 0});
    Dev<int32_t> starts(std::vector<int32_t>(3)), lengths(std::vector<int32_t>(2)), table(std::vector<int32_t>(8, -1));
    const std::vector<int32_t> zeros(rows);
    Dev<int32_t> positions(zeros), sequences(zeros), scratch(std::vector<int32_t>(4));
    Dev<int64_t> slots(std::vector<int64_t>(zeros.begin(), zeros.end()));
    const cache::Step step{starts.p, 3, lengths.p, 2, table.p, 8, positions.p, rows, slots.p, rows, sequences.p, rows, state.p, 4,
                           scratch.p, 4};
    cache::tables(sa, shape, cache::Requests{news.p, 2, past.p, 2}, cache::FreePages{ring.p, 6, state.p, 4}, step);
    CHECK(starts.host() == (std::vector<int32_t>{0, 1, 65}) && lengths.host() == (std::vector<int32_t>{1, 64}));
    CHECK(table.host() == (std::vector<int32_t>{5, -1, -1, -1, 0, 2, 3, 1}));
    CHECK(state.host() == (std::vector<int32_t>{5, 1, 0, 0}));
    const std::vector<int64_t> got = slots.host();
    CHECK(got[0] == 80 && got[1] == 0 && got[16] == 15 && got[17] == 32 && got[64] == 31 && got[65] == -1);
    CHECK(positions.host()[64] == 63 && sequences.host()[64] == 1 && sequences.host()[65] == -1);

    // Keys of ones; values 2 on the first page of a request and 4 on the others.
    const cache::Sizes sz = cache::sizes(shape, D);
    const std::vector<uint8_t> no_codes(sz.codes), no_scales(sz.scales);
    Dev<uint8_t> kc(no_codes), vc(no_codes), ks(no_scales), vs(no_scales);
    const cache::Pool pool{kc.p, ks.p, vc.p, vs.p, sz.codes, sz.scales};
    const cache::Index index = cache::index_of(step);
    std::vector<uint16_t> k(rows * D, bf16(1.0f)), v(rows * D), q(rows * H * D);
    for (std::size_t row = 0; row < rows; row++)
        for (std::size_t c = 0; c < D; c++) v[row * D + c] = bf16(row < 17 ? 2.0f : 4.0f);
    for (std::size_t i = 0; i < q.size(); i++) q[i] = bf16(0.125f * (float)(i % 7));
    Dev<uint16_t> dk(k), dv(v), dq(q), dqr(std::vector<uint16_t>(q.size())), dout(std::vector<uint16_t>(q.size(), 0x4242));
    const Strides kvst{0, D, D}, qst{0, H * D, D};
    const rotary::Table t = rotary::axes_table({4, 6, 6}, 3, 10000.0, {}, false, true);
    CHECK(t.rot == 32 && t.cos_sin.size() == 96 && t.cos_sin[0] == 1.0f && t.cos_sin[1] == 0.0f);
    Dev<float> dt(t.cos_sin);
    Dev<int32_t> zero(std::vector<int32_t>(3 * rows, 0));
    rotary::Axes axes{dt.p, dt.n, {4, 6, 6}, rotary::AxisLayout::AxisHalf, false, zero.p, 3 * rows, rows};
    const Tensor tq{dq.p, dq.n, qst};
    const TensorMut tqr{dqr.p, dqr.n, qst};
    cache::append(sa, shape, pool, index, Tensor{dk.p, dk.n, kvst}, Tensor{dv.p, dv.n, kvst}, axes, &tq, &tqr);
    std::vector<uint16_t> turned = dqr.host();
    for (std::size_t i = 65 * H * D; i < q.size(); i++) CHECK(turned[i] == 0);  // (padding)
    turned.resize(65 * H * D);
    CHECK(turned == std::vector<uint16_t>(q.begin(), q.begin() + 65 * H * D));
    axes.layout = rotary::AxisLayout::Pairs;
    rotary::apply(sa, Shape{1, H, rows}, axes, tq, tqr);
    CHECK(dqr.host() == q);

    // A key of 1 is four quarters: 64 sixteenths of its scale, 2^-2.
    Dev<int8_t> bc(std::vector<int8_t>(6 * 2 * D, 9));
    Dev<uint8_t> bs(std::vector<uint8_t>(6, 9));
    const cache::Bounds bounds{bc.p, bs.p, bc.n, bs.n};
    cache::update_bounds(sa, shape, pool, index, bounds);
    const std::vector<int8_t> hb = bc.host();
    const std::vector<uint8_t> hs = bs.host();
    for (std::size_t page = 0; page < 6; page++) {
        CHECK(hs[page] == (page == 4 ? 9 : 125));
        for (std::size_t c = 0; c < 2 * D; c++) CHECK(hb[page * 2 * D + c] == (page == 4 ? 9 : 64));
    }

    const cache::PickWorkspace ws(sa, shape, top);
    Dev<int32_t> picked(std::vector<int32_t>(rows * top, -9));
    cache::pick(sa, ws, bounds, index, tq, picked.p, picked.n);
    const std::vector<int32_t> p = picked.host();
    CHECK(p[0] == 0 && p[1] == -1 && p[2] == 0 && p[3] == -1);                    // rows that see one page
    CHECK(p[2 * 20] == 0 && p[2 * 20 + 1] == 1 && p[128] == 0 && p[129] == 3);    // the first and the own
    CHECK(p[130] == -9 && p[131] == -9);                                          // padding
    cache::attend_picked(sa, ws, pool, index, picked.p, picked.n, tq, TensorMut{dout.p, dout.n, qst});
    const std::vector<uint16_t> out = dout.host();
    for (std::size_t i = 0; i < H * D; i++) {
        CHECK(f32(out[i]) == 2.0f && f32(out[H * D + i]) == 2.0f);
        CHECK(f32(out[64 * H * D + i]) == 3.0f);  // 16 tokens of 2 and 16 of 4
        CHECK(out[65 * H * D + i] == 0x4242);
    }
    try {
        cache::pick(sa, ws, bounds, index, tq, picked.p, picked.n - 1);
        CHECK(!"a short list was accepted");
    } catch (const Error& e) {
        CHECK(e.status() == SAGE_ERR_INVALID && std::strstr(e.what(), "picked pages: buffer holds"));
    }
    std::printf("%d failure(s)\n", failures);
    return failures ? 1 : 0;
}
