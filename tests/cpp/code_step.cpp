// The operators that answer with codes through include/aq_mi355x.hpp (test
// infrastructure): norm, 4-bit product and sampling in a chain, each against
// its definition in doubles on what the one before it wrote.
//
// Exit status: 0 all checks passed, 1 a check failed, 77 no GPU.
#include "aq_mi355x.hpp"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <memory>
#include <stdexcept>
#include <vector>

namespace {

int failures = 0;

void expect(bool ok, const char *what) {
    std::printf("%s %s\n", ok ? "PASS" : "FAIL", what);
    std::fflush(stdout);
    if (!ok) ++failures;
}

template <typename T>
struct Device {
    T *p = nullptr;
    size_t n;
    explicit Device(size_t count) : n(count) {
        if (hipMalloc(reinterpret_cast<void **>(&p), n * sizeof(T)) != hipSuccess) throw std::runtime_error("hipMalloc");
    }
    explicit Device(const std::vector<T> &v) : Device(v.size()) {
        if (hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) throw std::runtime_error("hipMemcpy");
    }
    Device(const Device &) = delete;
    ~Device() { (void)hipFree(p); }
    std::vector<T> host() const {
        std::vector<T> v(n);
        if (hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) != hipSuccess) throw std::runtime_error("hipMemcpy");
        return v;
    }
};

// Numbers in [-1, 1) from a linear congruence.
struct Numbers {
    uint32_t s = 12345;
    float next() {
        s = s * 1664525u + 1013904223u;
        return static_cast<float>(static_cast<int32_t>(s)) * 0x1p-31f;
    }
};

void run(aq::Context &ctx) {
    constexpr int M = 3, D = 200, N = 150, G = 64, groups = (D + G - 1) / G;
    Numbers r;
    std::vector<float> x(M * D), residual(M * D), weight(D);
    for (float &v : x) v = r.next();
    for (float &v : residual) v = r.next();
    for (float &v : weight) v = 1.0f + 0.25f * r.next();
    Device<float> dx(x), dr(residual), dw(weight), dh(M * D), dy(M * D), dscale(M * groups);
    Device<int8_t> dq(static_cast<size_t>(M * D));
    aq::NormOutputs out;
    out.sum = dh.p;
    out.sum_ld = D;
    out.y = dy.p;
    out.y_ld = D;
    out.q_type = AQ_T_I8;
    out.group = G;
    out.q = dq.p;
    out.scale = dscale.p;
    aq::add_rmsnorm(ctx, AQ_T_F32, dx.p, D, dr.p, D, dw.p, M, D, 1e-6f, out);
    ctx.synchronize();
    const std::vector<float> h = dh.host(), y = dy.host(), scale = dscale.host();
    const std::vector<int8_t> q = dq.host();
    bool sums = true, rows = true, eight = true;
    for (int m = 0; m < M; ++m) {
        double ss = 0;
        for (int d = 0; d < D; ++d) {
            sums &= h[m * D + d] == x[m * D + d] + residual[m * D + d];
            ss += static_cast<double>(h[m * D + d]) * h[m * D + d];
        }
        for (int d = 0; d < D; ++d) {
            const double want = static_cast<double>(h[m * D + d]) * weight[d] / std::sqrt(ss / D + 1e-6);
            const double s = scale[m * groups + d / G];
            rows &= std::fabs(y[m * D + d] - want) <= 2e-6 * std::fabs(want);
            eight &= std::fabs(q[m * D + d] * s - want) <= 0.501 * s;
        }
    }
    expect(sums, "x + residual");
    expect(rows, "normalised rows");
    expect(eight, "8-bit rows");

    std::vector<uint8_t> codes(N * (D / 2)), zero(N * groups);
    std::vector<uint16_t> ws(N * groups);
    std::vector<float> bias(N);
    for (uint8_t &v : codes) v = static_cast<uint8_t>(128 + 127 * r.next());
    for (uint8_t &v : zero) v = static_cast<uint8_t>(7.5f + 7.0f * r.next());
    for (uint16_t &v : ws) v = static_cast<uint16_t>(0x2C00 + 256 * (1 + r.next()));   // F16 from 1/16 on
    for (float &v : bias) v = r.next();
    const auto f16 = [](uint16_t b) { return std::ldexp(1.0 + (b & 1023) / 1024.0, (b >> 10) - 15); };
    aq::Q4Linear linear(ctx, N, D, G, codes.data(), ws.data(), zero.data(), bias.data());
    Device<float> dlogits(M * N);
    linear.forward(AQ_T_I8, dq.p, D, M, AQ_T_F32, dlogits.p, N, dscale.p, G);
    ctx.synchronize();
    const std::vector<float> logits = dlogits.host();
    bool product = true;
    for (int m = 0; m < M; ++m)
        for (int n = 0; n < N; ++n) {
            double want = bias[n], size = std::fabs(bias[n]);
            for (int d = 0; d < D; ++d) {
                const int code = codes[n * (D / 2) + d / 2] >> (d % 2 * 4) & 15;
                const double term = q[m * D + d] * static_cast<double>(scale[m * groups + d / G]) *
                                    (code - zero[n * groups + d / G]) * f16(ws[n * groups + d / G]);
                want += term;
                size += std::fabs(term);
            }
            product &= std::fabs(logits[m * N + n] - want) <= 1e-6 * size;
        }
    expect(product, "4-bit product of the 8-bit rows");

    const std::vector<float> u{0.0f, 0.5f, 0.999f}, temperature{0.0f, 0.7f, 1.3f};
    const std::vector<int32_t> top_k{0, 5, 1};
    Device<float> du(u), dt(temperature), dlogp(M);
    Device<int32_t> dk(top_k), dtoken(M);
    aq::SampleFilters filters;
    filters.temperature = dt.p;
    filters.top_k = dk.p;
    aq::sample(ctx, AQ_T_F32, dlogits.p, N, M, N, du.p, filters, dtoken.p, dlogp.p);
    ctx.synchronize();
    const std::vector<int32_t> token = dtoken.host();
    const std::vector<float> logp = dlogp.host();
    bool drawn = true;
    for (int m = 0; m < M; ++m) {
        int above = 0;   // logits before the drawn one in the falling order
        if (token[m] < 0 || token[m] >= N) {
            drawn = false;
            continue;
        }
        for (int n = 0; n < N; ++n) {
            const float a = logits[m * N + n], b = logits[m * N + token[m]];
            above += a > b || (a == b && n < token[m]);
        }
        drawn &= above < (m == 1 ? 5 : 1) && logp[m] <= 0.0f && (m == 1 || logp[m] == 0.0f);
    }
    expect(drawn, "sampled codes");

    bool refused = false;
    try {
        linear.forward(AQ_T_I8, dq.p, D, M, AQ_T_F32, dlogits.p, N);
    } catch (const std::runtime_error &) {
        refused = true;
    }
    expect(refused, "8-bit rows without scales are refused");
}

}  // namespace

int main() {
    std::unique_ptr<aq::Context> ctx;
    try {
        ctx = std::make_unique<aq::Context>(0);
    } catch (const std::runtime_error &e) {
        std::printf("no GPU: %s\n", e.what());
        return 77;
    }
    try {
        run(*ctx);
    } catch (const std::exception &e) {
        expect(false, e.what());
    }
    return failures ? 1 : 0;
}
