// The rotary and cache calls of the C++ host API (include/spl_sage.hpp) on the
// GPU. Values are chosen so that the results are exact: keys and values on the
// cache's own levels come back as they went in, a position of angle 0 turns
// nothing, a sequence of one token attends to it alone, and equal keys give
// the mean of the values (a power of two of them).
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
    const std::size_t D = 64, H = 2, rows = 5;
    const SageAttention sa = SageAttention::create(nullptr, D);
    // Sequences of one token and of four, on shuffled pages of 16.
    const cache::CacheShape shape{2, rows, 4, H, 1, 6, 16, 2};
    const cache::Sizes sz = cache::sizes(shape, D);
    CHECK(sz.codes == 6 * 16 * 32 && sz.scales == 6 * 16 * 2);
    const std::vector<uint8_t> no_codes(sz.codes), no_scales(sz.scales);
    Dev<uint8_t> kc(no_codes), vc(no_codes), ks(no_scales), vs(no_scales);
    Dev<int32_t> starts({0, 1, 5}), lengths({1, 4}), table({5, 0, 2, 3});
    const cache::Pool pool{kc.p, ks.p, vc.p, vs.p, sz.codes, sz.scales};
    const cache::Index index{starts.p, 3, lengths.p, 2, table.p, 4};
    const float levels[8] = {0, 0.5f, 1, 1.5f, 2, 3, 4, 6};
    std::vector<uint16_t> k(rows * D), v(rows * D), q(rows * H * D);
    for (std::size_t i = 0; i < rows * D; i++) {
        // 4 v on the levels and each 32 channels with a 6 among them; one key for all.
        k[i] = bf16(levels[(i % D) % 8]);
        v[i] = bf16((i % 3 ? -0.25f : 0.25f) * levels[i % 32 == 7 ? 7 : (i * 5 + i / D) % 8]);
    }
    for (std::size_t i = 0; i < q.size(); i++) q[i] = bf16(0.125f * (float)(i % 7));
    Dev<uint16_t> dk(k), dv(v), dq(q), dqr(std::vector<uint16_t>(q.size())), dkb(std::vector<uint16_t>(k.size())),
        dvb(std::vector<uint16_t>(v.size())), dout(std::vector<uint16_t>(q.size()));
    const Strides kvst{0, D, D}, qst{0, H * D, D};

    // Every row at position 0: cos 1, sin 0.
    const rotary::Table t = rotary::Table::create(32, 8);
    Dev<float> dt(t.cos_sin);
    Dev<int32_t> zero(std::vector<int32_t>(rows, 0));
    const rotary::Rotary r{dt.p, dt.n, 32, rotary::Layout::Pairs, zero.p, rows};
    const Tensor tq{dq.p, dq.n, qst};
    const TensorMut tqr{dqr.p, dqr.n, qst};
    cache::append(sa, shape, pool, index, Tensor{dk.p, dk.n, kvst}, Tensor{dv.p, dv.n, kvst}, &r, &tq, &tqr);
    CHECK(dqr.host() == q);
    cache::read(sa, shape, pool, index, TensorMut{dkb.p, dkb.n, kvst}, TensorMut{dvb.p, dvb.n, kvst});
    CHECK(dkb.host() == k && dvb.host() == v);
    // A quarter turn and back.
    std::vector<float> quarter(32 * 8);
    for (std::size_t i = 0; i < quarter.size(); i += 2) quarter[i] = 0.0f, quarter[i + 1] = 1.0f;
    Dev<float> dqt(quarter);
    const rotary::Rotary r4{dqt.p, dqt.n, 32, rotary::Layout::Half, zero.p, rows};
    rotary::apply(sa, Shape{1, H, rows}, r4, tq, tqr);
    std::vector<uint16_t> turned = dqr.host();
    bool ok = true;
    for (std::size_t i = 0; i < q.size(); i += D)
        for (std::size_t c = i; c < i + 16; c++) ok &= f32(turned[c]) == -f32(q[c + 16]) && turned[c + 16] == q[c];
    CHECK(ok);
    rotary::apply(sa, Shape{1, H, rows}, r4, Tensor{dqr.p, dqr.n, qst}, tqr, true);
    CHECK(dqr.host() == q);

    const cache::CacheWorkspace ws(sa, shape);
    for (const bool causal : {true, false}) {
        cache::AttendOptions o;
        o.causal = causal;
        cache::attend(sa, ws, pool, index, tq, TensorMut{dout.p, dout.n, qst}, o);
        const std::vector<uint16_t> out = dout.host();
        ok = true;
        for (std::size_t row = 0; row < rows; row++)
            for (std::size_t h = 0; h < H; h++)
                for (std::size_t c = 0; c < D; c++) {
                    // Row 0: its own value. Rows 1, 2 and 4 see 1, 2 and 4 equal keys (causal), or all four.
                    const std::size_t seen = row == 0 ? 1 : causal ? row : 4, from = row == 0 ? 0 : 1;
                    if (seen == 3) continue;
                    float sum = 0;
                    for (std::size_t i = 0; i < seen; i++) sum += f32(v[(from + i) * D + c]);
                    ok &= f32(out[(row * H + h) * D + c]) == sum / (float)seen;
                }
        CHECK(ok);
    }
    try {
        cache::attend(sa, ws, pool, index, Tensor{dq.p, dq.n - 1, qst}, TensorMut{dout.p, dout.n, qst});
        CHECK(!"a short query buffer was accepted");
    } catch (const Error& e) {
        CHECK(e.status() == SAGE_ERR_INVALID && std::strstr(e.what(), "Q: buffer holds"));
    }
    std::printf("%d failure(s)\n", failures);
    return failures ? 1 : 0;
}
