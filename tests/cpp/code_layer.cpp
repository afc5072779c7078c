// The operators of a layer that answers with codes through
// include/aq_mi355x.hpp (test infrastructure): an 8-bit product, attention over
// a prefix and attention to an encoder's states in a chain, each against its
// definition in doubles on what the one before it wrote.
//
// Exit status: 0 all checks passed, 1 a check failed, 77 no GPU.
#include "aq_mi355x.hpp"

#include <cmath>
#include <cstdio>
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
    explicit Device(const std::vector<T> &v) : n(v.size()) {
        if (hipMalloc(reinterpret_cast<void **>(&p), n * sizeof(T)) != hipSuccess ||
            hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice) != hipSuccess)
            throw std::runtime_error("device memory");
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
    uint32_t s = 999;
    float next() {
        s = s * 1664525u + 1013904223u;
        return static_cast<float>(static_cast<int32_t>(s)) * 0x1p-31f;
    }
    std::vector<float> rows(size_t n) {
        std::vector<float> v(n);
        for (float &x : v) x = next();
        return v;
    }
};

constexpr int B = 2, T = 3, H = 4, KV = 2, D = 40, P = 70, S = 9, E = 50, K = 200, N = H * D;

// One row's attention: keys given by a function of (index, column) each.
template <typename KeyAt, typename ValueAt>
bool row_is(const float *got, const float *q, int keys, KeyAt k, ValueAt v, double scale) {
    std::vector<double> p(static_cast<size_t>(keys));
    double top = -1e300, total = 0;
    for (int j = 0; j < keys; ++j) {
        double z = 0;
        for (int d = 0; d < D; ++d) z += static_cast<double>(q[d]) * k(j, d);
        p[j] = z * scale;
        top = std::fmax(top, p[j]);
    }
    for (double &x : p) total += x = std::exp(x - top);
    bool ok = true;
    for (int d = 0; d < D; ++d) {
        double o = 0;
        for (int j = 0; j < keys; ++j) o += p[j] * v(j, d);
        // values are below 1 and scores below 2: some 2^-24 for each step of 200 or so
        ok &= std::fabs(got[d] - (keys ? o / total : 0)) <= 2e-5;
    }
    return ok;
}

void run(aq::Context &ctx) {
    Numbers r;
    // x [B T, K] -> q [B, T, H, D], in F32
    const std::vector<float> x = r.rows(B * T * K);
    std::vector<int8_t> w(N * K);
    for (int8_t &v : w) v = static_cast<int8_t>(std::lrint(127 * r.next()));
    std::vector<float> ws(N), bias = r.rows(N);
    for (float &v : ws) v = (1.5f + r.next()) / 2000;
    const aq::I8Linear linear(ctx, N, K, w.data(), ws.data(), bias.data());
    const Device<float> dx(x), dq(std::vector<float>(B * T * N, 0)), dout(std::vector<float>(B * T * N, 0));
    linear.forward(AQ_T_F32, dx.p, K, B * T, AQ_T_F32, dq.p, N);
    ctx.synchronize();
    const std::vector<float> q = dq.host();
    bool products = true;
    for (int m = 0; m < B * T; ++m) {
        double most = 0;
        for (int k = 0; k < K; ++k) most = std::fmax(most, std::fabs(x[m * K + k]));
        for (int n = 0; n < N; ++n) {
            double sum = 0;
            for (int k = 0; k < K; ++k) sum += std::rint(x[m * K + k] * 127.0 / most) * w[n * K + k];
            sum *= most / 127 * ws[n];
            products &= std::fabs(q[m * N + n] - (sum + bias[n])) <= 4e-7 * (std::fabs(sum) + std::fabs(bias[n]));
        }
    }
    expect(products, "8-bit product of floating rows");

    const std::vector<float> pk = r.rows(P * KV * D), pv = r.rows(P * KV * D), k = r.rows(B * S * KV * D), v = r.rows(B * S * KV * D);
    const Device<float> dpk(pk), dpv(pv), dk(k), dv(v);
    const std::vector<int32_t> len{S, 5};
    const Device<int32_t> dlen(len);
    const aq_heads hq{dq.p, T * N, N, D}, hout{dout.p, T * N, N, D};
    const float scale = 1 / std::sqrt(static_cast<float>(D));
    aq::AttentionShape shape;
    shape.B = B, shape.T = T, shape.S = S, shape.heads = H, shape.kv_heads = KV, shape.D = D;
    aq::AttentionLengths lengths;
    lengths.kv_len = dlen.p;
    aq::prefix_attention(ctx, AQ_T_F32, shape, P, hq, {dpk.p, 0, KV * D, D}, {dpv.p, 0, KV * D, D}, {dk.p, S * KV * D, KV * D, D},
                         {dv.p, S * KV * D, KV * D, D}, hout, scale, lengths);
    ctx.synchronize();
    const std::vector<float> first = dout.host();
    bool prefix = true;
    for (int b = 0; b < B; ++b)
        for (int t = 0; t < T; ++t)
            for (int h = 0; h < H; ++h) {
                const int g = h / (H / KV), own = len[b] - T + t + 1, at = ((b * T + t) * H + h) * D;
                const auto of = [&](const std::vector<float> &shared, const std::vector<float> &mine) {
                    return [&shared, &mine, b, g](int j, int d) {
                        return static_cast<double>(j < P ? shared[(j * KV + g) * D + d] : mine[((b * S + j - P) * KV + g) * D + d]);
                    };
                };
                prefix &= row_is(&first[at], &q[at], P + own, of(pk, k), of(pv, v), scale);
            }
    expect(prefix, "attention over a shared prefix");

    // What it wrote asks one encoder's states, with a mask, in place.
    const std::vector<float> ek = r.rows(E * KV * D), ev = r.rows(E * KV * D);
    std::vector<uint8_t> mask(E);
    std::vector<int> kept;
    for (int j = 0; j < E; ++j)
        if ((mask[j] = j % 3 != 1)) kept.push_back(j);
    const Device<float> dek(ek), dev(ev);
    const Device<uint8_t> dmask(mask);
    shape.S = E;
    aq::AttentionLengths seen;
    seen.mask = dmask.p;
    aq::cross_attention(ctx, AQ_T_F32, shape, hout, {dek.p, 0, KV * D, D}, {dev.p, 0, KV * D, D}, hout, scale, seen);
    ctx.synchronize();
    const std::vector<float> second = dout.host();
    bool cross = true;
    for (int m = 0; m < B * T * H; ++m) {
        const int g = m % H / (H / KV);
        const auto of = [&](const std::vector<float> &e) {
            return [&e, &kept, g](int j, int d) { return static_cast<double>(e[(kept[j] * KV + g) * D + d]); };
        };
        cross &= row_is(&second[m * D], &first[m * D], static_cast<int>(kept.size()), of(ek), of(ev), scale);
    }
    expect(cross, "attention to an encoder's states, in place");
    bool refused = false;
    try {
        aq::cross_attention(ctx, AQ_T_F32, shape, hq, {}, {}, hout, scale);
    } catch (const std::runtime_error &e) {
        refused = std::string(e.what()).find("aq_cross_attention") != std::string::npos;
    }
    expect(refused, "a refusal is an exception with the call's name");
}

}  // namespace

int main() {
    int count = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || count == 0) {
        std::printf("no GPU\n");
        return 77;
    }
    try {
        aq::Context ctx(0);
        run(ctx);
    } catch (const std::exception &e) {
        std::printf("FAIL %s\n", e.what());
        return 1;
    }
    return failures != 0;
}
