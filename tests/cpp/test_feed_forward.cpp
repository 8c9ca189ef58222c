// The feed-forward operators through the C++ mirror: norm with int8 output, int8 linear layer, routing, and the refusal of a bad call.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "lib/matmul_intf.h"

static int g_fail = 0;
#define CHECK(cond, ...)                                         \
    do {                                                         \
        if (!(cond)) {                                           \
            std::printf("FAIL %s:%d: ", __FILE__, __LINE__);     \
            std::printf(__VA_ARGS__);                            \
            std::printf("\n");                                   \
            ++g_fail;                                            \
        }                                                        \
    } while (0)

template <class T>
struct DevBuf {
    T* p = nullptr;
    size_t n = 0;
    explicit DevBuf(size_t count) : n(count) { ascb200_malloc(reinterpret_cast<void**>(&p), count * sizeof(T)); }
    explicit DevBuf(const std::vector<T>& h) : DevBuf(h.size())
    {
        ascb200_memcpy_h2d(p, h.data(), h.size() * sizeof(T), nullptr);
        ascb200_stream_sync(nullptr);
    }
    ~DevBuf() { ascb200_free(p); }
    AscendC::LocalTensor<T> Tensor() const { return AscendC::LocalTensor<T>(p, n); }
    std::vector<T> Download() const
    {
        std::vector<T> h(n);
        ascb200_memcpy_d2h(h.data(), p, n * sizeof(T), nullptr);
        ascb200_stream_sync(nullptr);
        return h;
    }
};

int main()
{
    if (ascb200_init(0) != 0) {
        std::printf("no B200 available\n");
        return 2;
    }
    const int M = 50, K = 256, N = 96;
    std::mt19937 rng(7);
    std::normal_distribution<float> normal;
    std::vector<float> x(M * K), r(M * K), gamma(K), ch(N), bias(N);
    std::vector<int8_t> w(N * K);
    for (auto& v : x) v = normal(rng);
    for (auto& v : r) v = normal(rng);
    for (auto& v : gamma) v = 1.0f + 0.1f * normal(rng);
    for (auto& v : ch) v = 0.001f * (1.0f + std::fabs(normal(rng)));
    for (auto& v : bias) v = normal(rng);
    for (auto& v : w) v = static_cast<int8_t>(static_cast<int>(rng() % 255) - 127);
    DevBuf<float> dx(x), dr(r), dg(gamma), dch(ch), db(bias), dsum(M * K), dscale(M), dy(M * N), dn(M * K);
    DevBuf<int8_t> dw(w), dq(M * K);
    AscendC::RmsNorm(dn.Tensor(), dx.Tensor(), dg.Tensor(), 1e-6f);
    AscendC::RmsNormQuant(dq.Tensor(), dscale.Tensor(), dsum.Tensor(), dx.Tensor(), dr.Tensor(), dg.Tensor(), 1e-6f);
    AscendC::LinearA8W8(dy.Tensor(), dq.Tensor(), dw.Tensor(), dscale.Tensor(), dch.Tensor(), db.Tensor(), AscendC::LocalTensor<float>(), ASCB200_ACT_SILU);
    CHECK(AscendC::GetLastError() == 0, "operator error %d", AscendC::GetLastError());
    const auto sum = dsum.Download(), scale = dscale.Download(), y = dy.Download(), norm = dn.Download();
    const auto q = dq.Download();
    int bad = 0;
    for (int m = 0; m < M; ++m) {
        double ss = 0, ss0 = 0, top = 0;
        for (int k = 0; k < K; ++k) {
            const double h = static_cast<double>(x[m * K + k]) + r[m * K + k];
            bad += std::fabs(sum[m * K + k] - h) > 1e-6 * (1 + std::fabs(h));
            ss += h * h, ss0 += static_cast<double>(x[m * K + k]) * x[m * K + k];
        }
        for (int k = 0; k < K; ++k) top = std::max(top, std::fabs((static_cast<double>(x[m * K + k]) + r[m * K + k]) / std::sqrt(ss / K + 1e-6) * gamma[k]));
        bad += std::fabs(scale[m] - top / 127) > 1e-5 * top / 127;
        for (int k = 0; k < K; ++k) {
            const double v = (static_cast<double>(x[m * K + k]) + r[m * K + k]) / std::sqrt(ss / K + 1e-6) * gamma[k];
            bad += std::fabs(q[m * K + k] * static_cast<double>(scale[m]) - v) > scale[m] * 0.501;
            bad += std::fabs(norm[m * K + k] - x[m * K + k] / std::sqrt(ss0 / K + 1e-6) * gamma[k]) > 1e-5 * (1 + std::fabs(norm[m * K + k]));
        }
        for (int n = 0; n < N; ++n) {
            long long acc = 0;
            for (int k = 0; k < K; ++k) acc += static_cast<long long>(q[m * K + k]) * w[n * K + k];
            const double z = static_cast<double>(acc) * ch[n] * scale[m] + bias[n], want = z / (1 + std::exp(-z));
            bad += std::fabs(y[m * N + n] - want) > 1e-5 * (1 + std::fabs(want));
        }
    }
    CHECK(bad == 0, "norm and linear: %d values wrong", bad);

    const int E = 20, TOP = 3;
    std::vector<float> logits(M * E);
    for (auto& v : logits) v = normal(rng);
    DevBuf<float> dl(logits), dwt(M * TOP), dloss(1);
    DevBuf<int32_t> didx(M * TOP);
    DevBuf<int64_t> dcount(E), dnum(1);
    const size_t bytes = ascb200_route_workspace_bytes(M, E);
    DevBuf<uint8_t> room(bytes);
    ascb200_route_desc d = {};
    d.tokens = M, d.experts = E, d.top_k = TOP, d.dtype = ASCB200_F32, d.renorm = 1;
    d.logits_dev = dl.p, d.idx_dev = didx.p, d.weights_dev = dwt.p, d.counts_dev = dcount.p, d.num_tokens_dev = dnum.p, d.loss_dev = dloss.p;
    d.workspace_dev = room.p, d.workspace_bytes = bytes;
    AscendC::Route(d);
    CHECK(AscendC::GetLastError() == 0, "operator error %d", AscendC::GetLastError());
    const auto idx = didx.Download();
    const auto counts = dcount.Download();
    std::vector<int64_t> seen(E, 0);
    bad = 0;
    for (int m = 0; m < M; ++m)
        for (int j = 0; j < TOP; ++j) {
            const int e = idx[m * TOP + j];
            if (e < 0 || e >= E) {
                ++bad;
                continue;
            }
            ++seen[e];
            int before = 0;
            for (int f = 0; f < E; ++f) before += logits[m * E + f] > logits[m * E + e];
            bad += before != j;
        }
    for (int e = 0; e < E; ++e) bad += seen[e] != counts[e];
    CHECK(bad == 0 && dnum.Download()[0] == M, "routing: %d wrong", bad);

    AscendC::RmsNorm(AscendC::LocalTensor<float>(), AscendC::LocalTensor<float>(dx.p, K), dg.Tensor(), 1e-6f);  // no destination: latched, no launch
    CHECK(AscendC::GetLastError() == ASCB200_EINVAL, "expected EINVAL, got %d", AscendC::GetLastError());
    std::printf(g_fail ? "%d checks failed\n" : "feed forward ok\n", g_fail);
    return g_fail ? 1 : 0;
}
