// Root-mean-square norm with the residual's addition and an output in 8 bits
// with scales (aq_add_rmsnorm).
//
// One pass: a row is held in registers between its reduction and its output,
// so every input is read once.  With p = h * weight and r = 1 / sqrt(mean(h^2)
// + eps), y = p * r, and the 8-bit value y / scale = p * (L / max |p|) does
// not depend on r: the group maxima of p are taken in the same sweep as the
// sum of squares.
//
// A row of D columns is nv = ceil(D / 8) vectors of 8; vector v of a row
// belongs to thread v % threads, so 4, 8 or 16 adjacent lanes hold a group of
// 32, 64 or 128 columns and its maximum is a butterfly within them.
//
// Bound by memory: 16384 bf16 rows of 8192 with every output (1.2 GB) take
// 218 us, 5.5 TB/s, 6000 f16 rows of 4096 without y (172 MB) 35.5 us, 4.8
// TB/s; a copy of 2 GB runs at 4.8 TB/s on the same card.  Few rows are bound
// by latency: a thread waits for its vector of x, then of residual, then of
// weight (a test of the row's end in each lane and the store of the sum lie
// between the loads), and for the next vector only after those (fp32: x and
// residual together).  One row of 1024 takes 3.0 us, the launch, three such
// waits and the reduction; 1499 fp32 rows of 1001, 1.5 waves a SIMD that wait
// four times each, 10 us, where the bytes need 5.3.
#include "aq_device_math.hpp"
#include "aq_internal.hpp"
#include "aq_types.hpp"

namespace {

using namespace aq_types;

struct norm_args {
    const void *x, *residual, *weight;
    void *sum, *y, *q;
    float *scale;
    int64_t x_ld, residual_ld, sum_ld, y_ld, M, D;
    float eps;
    int q_type, group;   // group 0: one scale a row
};

// The smallest maximum of |p| with a scale: L / max stays finite above it.
constexpr float kLeastMax = 0x1p-118f;

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The larger of two magnitudes by their bits, where NaN is above infinity:
// a maximum that a NaN does not leave.
__device__ inline float mag_max(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

template <int LANES>
__device__ inline float lanes_max(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = mag_max(v, __shfl_xor(v, o));
    return v;
}

// 8 values of p as 8-bit values times `inv`.
__device__ inline uint2 quantize8(const float (&p)[8], float inv, bool e4m3) {
    if (e4m3) {
        uint32_t lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(p[0] * inv, p[1] * inv, lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(p[2] * inv, p[3] * inv, lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(p[4] * inv, p[5] * inv, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(p[6] * inv, p[7] * inv, hi, true);
        return make_uint2(lo, hi);
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w[h] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[h] |= (static_cast<uint32_t>(static_cast<int>(rintf(p[4 * h + i] * inv))) & 255u) << (8 * i);
    }
    return make_uint2(w[0], w[1]);
}

__device__ inline void store_q8(void *q, int64_t row, int64_t D, int64_t at, uint2 v) {
    uint8_t *to = static_cast<uint8_t *>(q) + row * D;
    if (at + 8 <= D) {
        std::memcpy(to + at, &v, 8);
    } else {
        uint8_t b[8];
        std::memcpy(b, &v, 8);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < D) to[at + i] = b[i];
    }
}

// 1 / sqrt(m), root = sqrt(m) rounded: the reciprocal's error comes from what
// is left of 1 - m r^2, so the result is within little more than half a unit,
// where the two roundings alone give up to one and a half.
__device__ inline float inverse_root(float m, float root) {
    const float r = 1.0f / root, t = m * r;
    const float left = __fmaf_rn(-__fmaf_rn(m, r, -t), r, __fmaf_rn(-t, r, 1.0f));
    return left == left ? __fmaf_rn(0.5f * r, left, r) : r;   // not for m = 0 or infinity
}

// max |y| / L from max |p| and the root: by the product of root and L, two
// roundings, where 1 / root, max |y| and its quotient would be three.
__device__ inline float scale_of(float pmax, float root, float r, bool e4m3) {
    if (!(pmax * r < INFINITY)) return NAN;   // y is not finite
    return pmax < kLeastMax ? 0.0f : pmax / (root * (e4m3 ? 448.0f : 127.0f));
}

__device__ inline float inverse_of(float pmax, bool e4m3) {
    return pmax < kLeastMax ? 0.0f : (e4m3 ? 448.0f : 127.0f) / pmax;
}

// WAVES waves hold one row, VPT vectors a thread; WAVES = 1 puts four rows in
// a block.
template <typename T, int WAVES, int VPT>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void add_rmsnorm_kernel(norm_args a) {
    constexpr int kThreads = 64 * WAVES;
    using raw = typename T::raw;
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int tid = WAVES == 1 ? lane : static_cast<int>(threadIdx.x);
    const int64_t row = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
    if (WAVES == 1 && row >= a.M) return;   // a whole wave; no barrier follows where WAVES is 1
    const raw *x = static_cast<const raw *>(a.x) + row * a.x_ld;
    const raw *res = a.residual ? static_cast<const raw *>(a.residual) + row * a.residual_ld : nullptr;

    float p[VPT][8], pmax[VPT];
    float ss = 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int64_t at = static_cast<int64_t>(v * kThreads + tid) * 8;
        pmax[v] = 0.0f;
        if (at >= a.D) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[v][i] = 0.0f;
            continue;
        }
        load8<T>(x, at, a.D, p[v]);
        if (res) {
            float r[8];
            load8<T>(res, at, a.D, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[v][i] = T::load(T::store(p[v][i] + r[i]));
        }
        if (a.sum) store8<T>(static_cast<raw *>(a.sum) + row * a.sum_ld, at, a.D, p[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __fmaf_rn(p[v][i], p[v][i], ss);
        if (a.weight) {
            float w[8];
            load8<T>(static_cast<const raw *>(a.weight), at, a.D, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[v][i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) pmax[v] = mag_max(pmax[v], fabsf(p[v][i]));
    }

    ss = wave_sum(ss);
    float rowmax = pmax[0];
    if (a.q && !a.group) {
#pragma unroll
        for (int v = 1; v < VPT; ++v) rowmax = mag_max(rowmax, pmax[v]);
        rowmax = lanes_max<64>(rowmax);
    }
    if constexpr (WAVES > 1) {
        __shared__ float part[2][WAVES];
        if (lane == 0) {
            part[0][wave] = ss;
            part[1][wave] = rowmax;
        }
        __syncthreads();
        ss = part[0][0];
        rowmax = part[1][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            ss += part[0][w];
            rowmax = mag_max(rowmax, part[1][w]);
        }
    }
    const float mean = ss / static_cast<float>(a.D) + a.eps, root = aq_math::sqrt_rn(mean), r = inverse_root(mean, root);

    const bool e4m3 = a.q_type == AQ_T_E4M3;
    const int64_t groups = a.group ? (a.D + a.group - 1) / a.group : 1;
    if (a.q && !a.group && tid == 0) a.scale[row] = scale_of(rowmax, root, r, e4m3);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int64_t at = static_cast<int64_t>(v * kThreads + tid) * 8;
        float m = rowmax;
        if (a.q && a.group) {
            m = lanes_max<4>(pmax[v]);
            if (a.group > 32) m = mag_max(m, __shfl_xor(m, 4));
            if (a.group > 64) m = mag_max(m, __shfl_xor(m, 8));
        }
        if (at >= a.D) continue;
        if (a.y) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = p[v][i] * r;
            store8<T>(static_cast<raw *>(a.y) + row * a.y_ld, at, a.D, y);
        }
        if (a.q) {
            store_q8(a.q, row, a.D, at, quantize8(p[v], inverse_of(m, e4m3), e4m3));
            if (a.group && at % a.group == 0) a.scale[row * groups + at / a.group] = scale_of(m, root, r, e4m3);
        }
    }
}

// Rows longer than the registers of a block: the same in two sweeps, the
// second over h again (from `sum` where it is written, since x or residual
// may be its buffer).
template <typename T>
__global__ __launch_bounds__(1024) void add_rmsnorm_long_kernel(norm_args a) {
    using raw = typename T::raw;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const raw *x = static_cast<const raw *>(a.x) + row * a.x_ld;
    const raw *res = a.residual ? static_cast<const raw *>(a.residual) + row * a.residual_ld : nullptr;
    raw *sum = a.sum ? static_cast<raw *>(a.sum) + row * a.sum_ld : nullptr;
    const raw *weight = static_cast<const raw *>(a.weight);

    auto row8 = [&](const raw *from, const raw *add, int64_t at, float (&h)[8]) {
        load8<T>(from, at, a.D, h);
        if (add) {
            float r[8];
            load8<T>(add, at, a.D, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = T::load(T::store(h[i] + r[i]));
        }
    };
    auto weigh = [&](int64_t at, float (&h)[8]) {
        if (!weight) return;
        float w[8];
        load8<T>(weight, at, a.D, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] *= w[i];
    };

    float ss = 0.0f, rowmax = 0.0f;
    for (int64_t base = 0; base < a.D; base += 8192) {
        const int64_t at = base + threadIdx.x * 8;
        if (at < a.D) {
            float h[8];
            row8(x, res, at, h);
            if (sum) store8<T>(sum, at, a.D, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __fmaf_rn(h[i], h[i], ss);
            weigh(at, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) rowmax = mag_max(rowmax, fabsf(h[i]));
        }
    }
    __shared__ float part[2][16];
    ss = wave_sum(ss);
    rowmax = lanes_max<64>(rowmax);
    if (lane == 0) {
        part[0][wave] = ss;
        part[1][wave] = rowmax;
    }
    __syncthreads();
    ss = part[0][0];
    rowmax = part[1][0];
#pragma unroll
    for (int w = 1; w < 16; ++w) {
        ss += part[0][w];
        rowmax = mag_max(rowmax, part[1][w]);
    }
    const float mean = ss / static_cast<float>(a.D) + a.eps, root = aq_math::sqrt_rn(mean), r = inverse_root(mean, root);

    const bool e4m3 = a.q_type == AQ_T_E4M3;
    const int64_t groups = a.group ? (a.D + a.group - 1) / a.group : 1;
    if (a.q && !a.group && threadIdx.x == 0) a.scale[row] = scale_of(rowmax, root, r, e4m3);
    for (int64_t base = 0; base < a.D; base += 8192) {
        const int64_t at = base + threadIdx.x * 8;
        float p[8] = {};
        float m = 0.0f;
        if (at < a.D) {
            row8(sum ? sum : x, sum ? nullptr : res, at, p);
            weigh(at, p);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = mag_max(m, fabsf(p[i]));
        }
        if (a.q && a.group) {
            m = lanes_max<4>(m);
            if (a.group > 32) m = mag_max(m, __shfl_xor(m, 4));
            if (a.group > 64) m = mag_max(m, __shfl_xor(m, 8));
        } else {
            m = rowmax;
        }
        if (at < a.D) {
            if (a.y) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = p[i] * r;
                store8<T>(static_cast<raw *>(a.y) + row * a.y_ld, at, a.D, y);
            }
            if (a.q) {
                store_q8(a.q, row, a.D, at, quantize8(p, inverse_of(m, e4m3), e4m3));
                if (a.group && at % a.group == 0) a.scale[row * groups + at / a.group] = scale_of(m, root, r, e4m3);
            }
        }
    }
}

// Rows of one launch: a grid has fewer than 2^32 threads.
constexpr int64_t kRowsAtOnce = int64_t{1} << 21;

template <typename T>
void launch(aq_ctx *ctx, const norm_args &a) {
    using raw = typename T::raw;
    const int64_t nv = (a.D + 7) / 8, scales = a.group ? (a.D + a.group - 1) / a.group : 1;
    const auto go = [&](auto kernel, int waves) {
        for (int64_t m = 0; m < a.M; m += kRowsAtOnce) {
            norm_args b = a;
            b.M = a.M - m < kRowsAtOnce ? a.M - m : kRowsAtOnce;
            b.x = static_cast<const raw *>(a.x) + m * a.x_ld;
            if (a.residual) b.residual = static_cast<const raw *>(a.residual) + m * a.residual_ld;
            if (a.sum) b.sum = static_cast<raw *>(a.sum) + m * a.sum_ld;
            if (a.y) b.y = static_cast<raw *>(a.y) + m * a.y_ld;
            if (a.q) {
                b.q = static_cast<uint8_t *>(a.q) + m * a.D;
                b.scale = a.scale + m * scales;
            }
            const uint32_t grid = static_cast<uint32_t>(waves == 1 ? (b.M + 3) / 4 : b.M);
            aq_launch_timed(ctx, true, kernel, dim3(grid), dim3(waves == 1 ? 256 : 64 * waves), 0u, b);
        }
    };
    // A wave a row needs no barrier, and two vectors a thread cost less than
    // twice the waves, once there are rows for all of the card: 4096 bf16 rows
    // of 1024 take 10.4 us with <1, 2>, 11.4 with <4, 1>, of 4096 26.6 with
    // <4, 2>, 27.8 with <8, 1>, of 8192 55.6 with <8, 2>, 61.4 with <16, 1>.
    // Before that a row's own time counts: one takes 4.2 and 3.2, 4.7 and
    // 3.7, 5.0 and 4.4 us; the two meet at about 512 to 1024 rows.
    const bool few = a.M <= 512;
    if (nv <= 64) go(add_rmsnorm_kernel<T, 1, 1>, 1);
    else if (nv <= 128 && !few) go(add_rmsnorm_kernel<T, 1, 2>, 1);
    else if (nv <= 256) go(add_rmsnorm_kernel<T, 4, 1>, 4);
    else if (nv <= 512 && !few) go(add_rmsnorm_kernel<T, 4, 2>, 4);
    else if (nv <= 512) go(add_rmsnorm_kernel<T, 8, 1>, 8);
    else if (nv <= 1024 && !few) go(add_rmsnorm_kernel<T, 8, 2>, 8);
    else if (nv <= 1024) go(add_rmsnorm_kernel<T, 16, 1>, 16);
    else if (nv <= 2048) go(add_rmsnorm_kernel<T, 16, 2>, 16);
    else if (nv <= 4096) go(add_rmsnorm_kernel<T, 16, 4>, 16);
    else go(add_rmsnorm_long_kernel<T>, 16);
}

}  // namespace

extern "C" aq_status aq_add_rmsnorm(aq_ctx *ctx, int type, const void *x, int64_t x_ld, const void *residual,
                                    int64_t residual_ld, const void *weight, int64_t M, int64_t D, float eps,
                                    void *sum, int64_t sum_ld, void *y, int64_t y_ld, int q_type, int64_t group,
                                    void *q, float *scale) {
    if (!ctx) return AQ_E_INVALID_ARG;
    if (type != AQ_T_F32 && type != AQ_T_F16 && type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_add_rmsnorm: type %d is not F32, F16 or BF16", type);
    if (M < 0 || M > INT32_MAX || D < 1 || D > (int64_t(1) << 30))
        return aq_fail(ctx, AQ_E_SHAPE, "aq_add_rmsnorm: M=%lld D=%lld (D from 1 to 2^30)", static_cast<long long>(M),
                       static_cast<long long>(D));
    if (!(eps >= 0.0f)) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_add_rmsnorm: eps %g is negative or NaN", eps);
    if (q && q_type != AQ_T_I8 && q_type != AQ_T_E4M3)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_add_rmsnorm: q_type %d is not I8 or E4M3", q_type);
    if (q && group != 0 && group != 32 && group != 64 && group != 128)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_add_rmsnorm: group %lld is not 0, 32, 64 or 128",
                       static_cast<long long>(group));
    if (M == 0) return AQ_OK;
    if (!x || (q != nullptr) != (scale != nullptr) || (!sum && !y && !q))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_add_rmsnorm: null x, q without scale, or no output");
    if (x_ld < D || (residual && residual_ld < D) || (sum && sum_ld < D) || (y && y_ld < D))
        return aq_fail(ctx, AQ_E_SHAPE, "aq_add_rmsnorm: a row stride is below D=%lld", static_cast<long long>(D));
    if (sum && sum == y) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_add_rmsnorm: sum and y are one buffer");
    if ((sum == x && sum_ld != x_ld) || (y == x && y_ld != x_ld) ||
        (residual && ((sum == residual && sum_ld != residual_ld) || (y == residual && y_ld != residual_ld))))
        return aq_fail(ctx, AQ_E_SHAPE, "aq_add_rmsnorm: an output in an input's buffer needs its row stride");
    aq_device_guard g(ctx->device);
    norm_args a{x, residual, weight, sum, y, q, scale, x_ld, residual_ld, sum_ld, y_ld, M, D, eps, q_type,
                static_cast<int>(q ? group : 0)};
    if (type == AQ_T_F32) launch<f32>(ctx, a);
    else if (type == AQ_T_F16) launch<f16>(ctx, a);
    else launch<bf16>(ctx, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}
