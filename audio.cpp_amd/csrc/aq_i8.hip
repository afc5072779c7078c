// Products with 8-bit whole-number weights, a scale for each row of W and
// each row of x (aq_i8_*).
//
// Layout.  A tile is 16 rows of W, a k-block 64 columns: 1 KB, 16 bytes a
// lane, in the order of the 16x16x64 matrix instruction's operand: lane l
// holds row l % 16, columns 16 (l / 16) ..+15 of the k-block.  Rows and
// columns past the end are zeros, so x may hold anything there.  A packed x
// has the same layout, by 16 rows of x.
//
// The sums are whole numbers of 32 bits (in_features below 2^17, so that
// 128 * 128 of them fit) and do not depend on an order; what is rounded is the
// sum's conversion to fp32 (2^-24), the two scalings and the bias.
#include "aq_internal.hpp"
#include "aq_types.hpp"

#include <new>

struct aq_i8 {
    int device = -1;   // of the creating context; the handle may outlive it
    int64_t N = 0, K = 0;
    int tiles = 0, kblocks = 0;
    uint8_t *w = nullptr;   // [tiles][kblocks][64 lanes][16]
    float *scale = nullptr;
    float *bias = nullptr;
};

namespace {

using namespace aq_types;

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct args {
    const uint8_t *w;
    const float *scale, *bias;
    const uint8_t *x;       // rows, or packed
    const float *x_scale;   // [M]
    void *y;
    int64_t x_ld, y_ld;
    int M, N, K, tiles, kblocks, y_type;
};

__device__ inline i32x4 load16(const uint8_t *p) {
    typedef i32x4 any __attribute__((aligned(1)));
    return *reinterpret_cast<const any *>(p);
}

// The tiles from rows of W: one thread a lane's 16 bytes.
__global__ __launch_bounds__(256) void i8_tiles_kernel(const uint8_t *from, int64_t N, int64_t K, int64_t kblocks,
                                                       int64_t count, i32x4 *to) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= count) return;
    const int64_t lane = i & 63, block = i >> 6;
    const int64_t n = block / kblocks * 16 + (lane & 15), k0 = block % kblocks * 64 + 16 * (lane >> 4);
    uint32_t w[4] = {};
#pragma unroll
    for (int c = 0; c < 16; ++c)
        if (n < N && k0 + c < K) w[c / 4] |= static_cast<uint32_t>(from[n * K + k0 + c]) << (8 * (c % 4));
    to[i] = i32x4{static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3])};
}

// x[m][k..k+15] as bytes, zeros past the end.
__device__ inline i32x4 load_tail(const uint8_t *row, int k, int K) {
    uint32_t w[4] = {};
#pragma unroll
    for (int c = 0; c < 16; ++c)
        if (k + c < K) w[c / 4] |= static_cast<uint32_t>(row[k + c]) << (8 * (c % 4));
    return i32x4{static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3])};
}

// ---- rows of x in operand order ---------------------------------------------

// 16 rows a block, one wave a row; rows past M are zeros.  I8 rows are moved.
// A floating row is brought to 8 bits: its largest magnitude, then q = the
// whole number nearest to x * 127 / max, ties to even.  Twice the quotient is
// formed in 64 bits with an error below 2^-44; where it is not a whole number
// it is at least 2^-32 off one (x and max have 24 bits, and x is near or above
// max / 254 where it matters), so within 2^-40 it is one, and every q is exact.
__global__ __launch_bounds__(1024) void i8_pack_kernel(const uint8_t *x, int64_t x_ld, int M, int K, int kblocks,
                                                       i32x4 *to) {
    const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int64_t m = static_cast<int64_t>(blockIdx.x) * 16 + r;
    i32x4 *const out = to + static_cast<int64_t>(blockIdx.x) * kblocks * 64 + r;
    const uint8_t *row = x + m * x_ld;
    for (int c = lane; c < kblocks * 4; c += 64) {
        i32x4 v = {0, 0, 0, 0};
        if (m < M) v = 16 * c + 16 <= K ? load16(row + 16 * c) : load_tail(row, 16 * c, K);
        out[(c >> 2) * 64 + (c & 3) * 16] = v;
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void i8_quantize_kernel(const typename T::raw *x, int64_t x_ld, int M, int K,
                                                           int kblocks, i32x4 *to, float *scale) {
    const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int64_t m = static_cast<int64_t>(blockIdx.x) * 16 + r;
    i32x4 *const out = to + static_cast<int64_t>(blockIdx.x) * kblocks * 64 + r;
    const typename T::raw *row = x + m * x_ld;
    uint32_t most = 0;   // magnitudes compare like their bits, with infinity and NaN above all others
    if (m < M)
        for (int c = lane; 8 * c < K; c += 64) {
            float v[8];
            load8<T>(row, 8 * c, K, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        }
#pragma unroll
    for (int d = 32; d; d >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
    const bool finite = most < 0x7F800000u;
    const double top = static_cast<double>(__uint_as_float(most)), per = finite && most ? 254.0 / top : 0.0;
    for (int c = lane; c < kblocks * 4; c += 64) {
        uint32_t w[4] = {};
        if (m < M) {
            float v[16];
            load8<T>(row, 16 * c, K, *reinterpret_cast<float(*)[8]>(v));
            load8<T>(row, 16 * c + 8, K, *reinterpret_cast<float(*)[8]>(v + 8));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                double twice = static_cast<double>(v[i]) * per;
                const double near = __builtin_rint(twice);
                if (__builtin_fabs(twice - near) < 0x1p-40) twice = near;
                const int q = finite ? static_cast<int>(__builtin_rint(0.5 * twice)) : 0;
                w[i / 4] |= (static_cast<uint32_t>(q) & 255u) << (8 * (i % 4));
            }
        }
        out[(c >> 2) * 64 + (c & 3) * 16] =
            i32x4{static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3])};
    }
    if (m < M && lane == 0) scale[m] = finite ? static_cast<float>(top / 127.0) : __uint_as_float(0x7FC00000u);
}

// ---- the product ---------------------------------------------------------------

// Four columns n.. of row m from their sums.
__device__ inline void store4(const args &a, int m, int n, i32x4 sum) {
    if (m >= a.M || n >= a.N) return;
    const float xs = a.x_scale[m];
    const int most = min(4, a.N - n);
    float o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int at = n + min(c, most - 1);
        o[c] = static_cast<float>(sum[c]) * a.scale[at] * xs;   // (the scales' product alone may be subnormal)
        if (a.bias) o[c] += a.bias[at];
    }
    const int64_t at = m * a.y_ld + n;
    if (a.y_type == AQ_T_F32) {
        float *y = static_cast<float *>(a.y) + at;
        if (most == 4) std::memcpy(y, o, 16);
        else for (int c = 0; c < most; ++c) y[c] = o[c];
    } else {
        uint16_t h[4];
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
            if (a.y_type == AQ_T_F16) f16::store2(h + c, o[c], o[c + 1]);
            else bf16::store2(h + c, o[c], o[c + 1]);
        }
        uint16_t *y = static_cast<uint16_t *>(a.y) + at;
        if (most == 4) std::memcpy(y, h, 8);
        else for (int c = 0; c < most; ++c) y[c] = h[c];
    }
}

// A block: RT tiles times 16 MT rows of x; its waves take U k-blocks in turn
// and their sums are joined in LDS.
template <bool PACKED, int RT, int MT, int U>
__global__ __launch_bounds__(512) void i8_product_kernel(args a) {
    extern __shared__ i32x4 red[];   // [waves][RT * MT][64]
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int tile0 = static_cast<int>(blockIdx.x) * RT, m0 = static_cast<int>(blockIdx.y) * 16 * MT;
    const uint8_t *w[RT], *x[MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
        w[r] = a.w + (static_cast<int64_t>(min(tile0 + r, a.tiles - 1)) * a.kblocks * 64 + lane) * 16;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (PACKED) x[t] = a.x + (static_cast<int64_t>(min(m0 / 16 + t, (a.M - 1) / 16)) * a.kblocks * 64 + lane) * 16;
        else x[t] = a.x + min(m0 + 16 * t + col, a.M - 1) * a.x_ld + 16 * quad;   // rows past the end repeat the last one
    }
    i32x4 sum[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[r][t] = i32x4{0, 0, 0, 0};

    const auto add = [&](const i32x4 (&wv)[RT], const i32x4 (&xv)[MT]) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) sum[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[r], xv[t], sum[r][t], 0, 0, 0);
    };
    const int whole = PACKED ? a.kblocks : a.K / 64;   // k-blocks without columns past the end
    const auto load = [&](int kb, i32x4 (&wv)[RT], i32x4 (&xv)[MT]) {
#pragma unroll
        for (int r = 0; r < RT; ++r) wv[r] = load16(w[r] + static_cast<int64_t>(kb) * 1024);
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[t] = load16(x[t] + (PACKED ? kb * int64_t{1024} : kb * int64_t{64}));
    };
    i32x4 wv[U][RT], xv[U][MT];
    int kb = wave * U;
#pragma unroll 1
    for (; kb + U <= whole; kb += waves * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(kb + u, wv[u], xv[u]);
        __builtin_amdgcn_sched_barrier(0);   // the loads go out before the arithmetic
#pragma unroll
        for (int u = 0; u < U; ++u) add(wv[u], xv[u]);
    }
#pragma unroll 1
    for (; kb < whole; ++kb) {   // fewer than U are left, for one wave
        load(kb, wv[0], xv[0]);
        add(wv[0], xv[0]);
    }
    if (!PACKED && whole < a.kblocks && wave == waves - 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r) wv[0][r] = load16(w[r] + static_cast<int64_t>(whole) * 1024);
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[0][t] = load_tail(x[t] - 16 * quad, 64 * whole + 16 * quad, a.K);
        add(wv[0], xv[0]);
    }
    if (waves == 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t) store4(a, m0 + 16 * t + col, (tile0 + r) * 16 + 4 * quad, sum[r][t]);
        return;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[(wave * RT * MT + r * MT + t) * 64 + lane] = sum[r][t];
    __syncthreads();
    for (int i = wave; i < RT * MT; i += waves) {
        i32x4 v = red[i * 64 + lane];
        for (int k = 1; k < waves; ++k) v += red[(k * RT * MT + i) * 64 + lane];
        store4(a, m0 + 16 * (i % MT) + col, (tile0 + i / MT) * 16 + 4 * quad, v);
    }
}

template <bool PACKED, int RT, int MT, int U>
aq_status launch(aq_ctx *ctx, const args &a, int waves) {
    const int most = (a.kblocks + U - 1) / U;
    if (waves > most) waves = most;
    const uint32_t lds = static_cast<uint32_t>(waves * RT * MT * 1024);
    auto kernel = i8_product_kernel<PACKED, RT, MT, U>;
    aq_status st = aq_launch_lds(ctx, reinterpret_cast<const void *>(kernel), lds, "aq_i8_forward");
    if (st != AQ_OK) return st;
    const dim3 grid(static_cast<uint32_t>((a.tiles + RT - 1) / RT), static_cast<uint32_t>((a.M + 16 * MT - 1) / (16 * MT)));
    aq_launch_timed(ctx, true, kernel, grid, dim3(static_cast<uint32_t>(64 * waves)), lds, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}

template <bool PACKED>
aq_status launch_product(aq_ctx *ctx, const args &a) {
    if (a.M <= 16) return launch<PACKED, 1, 1, 4>(ctx, a, 8);
    if (a.M <= 32) return launch<PACKED, 2, 2, 2>(ctx, a, 8);
    return launch<PACKED, 4, 4, 1>(ctx, a, 4);
}

// Rows of x at a time in operand order: 64 MB of them, but at least 64.
constexpr int64_t kPackedBytes = int64_t{64} << 20;

void free_all(aq_i8 *w) {
    for (void *p : {static_cast<void *>(w->w), static_cast<void *>(w->scale), static_cast<void *>(w->bias)})
        if (p) (void)hipFree(p);
    delete w;
}

}  // namespace

extern "C" {

aq_status aq_i8_upload(aq_ctx *ctx, int64_t out_features, int64_t in_features, const int8_t *w, const float *scale,
                       const float *bias, aq_i8 **out) {
    if (out) *out = nullptr;
    if (!ctx || !w || !scale || !out) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_i8_upload: null argument");
    const int64_t N = out_features, K = in_features;
    if (N < 1 || K < 1 || N > (int64_t{1} << 24) || K >= (int64_t{1} << 17) || N > (int64_t{1} << 34) / K)
        return aq_fail(ctx, AQ_E_SHAPE,
                       "aq_i8_upload: out_features=%lld (1 to 2^24) in_features=%lld (1 to 2^17 - 1), at most 2^34 weights",
                       (long long)N, (long long)K);
    aq_device_guard g(ctx->device);
    aq_i8 *h = new (std::nothrow) aq_i8();
    if (!h) return aq_fail(ctx, AQ_E_NOMEM, "aq_i8_upload: host allocation failed");
    h->device = ctx->device;
    h->N = N;
    h->K = K;
    h->tiles = static_cast<int>((N + 15) / 16);
    h->kblocks = static_cast<int>((K + 63) / 64);
    const int64_t pieces = int64_t{h->tiles} * h->kblocks * 64;
    uint8_t *rows = nullptr;
    hipError_t e = hipMalloc(&h->w, static_cast<size_t>(pieces) * 16);
    if (e == hipSuccess) e = hipMalloc(&h->scale, static_cast<size_t>(N) * 4);
    if (e == hipSuccess) e = hipMemcpy(h->scale, scale, static_cast<size_t>(N) * 4, hipMemcpyHostToDevice);
    if (e == hipSuccess && bias) {
        e = hipMalloc(&h->bias, static_cast<size_t>(N) * 4);
        if (e == hipSuccess) e = hipMemcpy(h->bias, bias, static_cast<size_t>(N) * 4, hipMemcpyHostToDevice);
    }
    if (e == hipSuccess) e = hipMalloc(&rows, static_cast<size_t>(N * K));
    if (e == hipSuccess) e = hipMemcpy(rows, w, static_cast<size_t>(N * K), hipMemcpyHostToDevice);
    if (e == hipSuccess) {
        hipLaunchKernelGGL(i8_tiles_kernel, dim3(static_cast<uint32_t>((pieces + 255) / 256)), dim3(256), 0, ctx->stream, rows,
                           N, K, int64_t{h->kblocks}, pieces, reinterpret_cast<i32x4 *>(h->w));
        e = hipGetLastError();
        const hipError_t e2 = hipStreamSynchronize(ctx->stream);
        if (e == hipSuccess) e = e2;
    }
    if (rows) (void)hipFree(rows);
    if (e != hipSuccess) {
        free_all(h);
        (void)hipGetLastError();   // reported below, and no error of the caller's next launch
        return aq_fail(ctx, e == hipErrorOutOfMemory ? AQ_E_NOMEM : AQ_E_DEVICE, "aq_i8_upload: %s", hipGetErrorString(e));
    }
    *out = h;
    return AQ_OK;
}

aq_status aq_i8_forward(aq_ctx *ctx, const aq_i8 *w, int x_type, const void *x, int64_t x_ld, const float *x_scale,
                        int64_t M, int y_type, void *y, int64_t y_ld) {
    if (!ctx || !w) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_i8_forward: null argument");
    if (w->device != ctx->device)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_i8_forward: weights belong to another device");
    if (x_type != AQ_T_I8 && x_type != AQ_T_F32 && x_type != AQ_T_F16 && x_type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_i8_forward: x_type %d is not I8, F32, F16 or BF16", x_type);
    if (y_type != AQ_T_F32 && y_type != AQ_T_F16 && y_type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_i8_forward: y_type %d is not F32, F16 or BF16", y_type);
    if (M < 0 || M > int64_t{1} << 20)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_i8_forward: M=%lld (0 to 2^20)", (long long)M);
    if (M == 0) return AQ_OK;
    if (!x || !y || (x_type == AQ_T_I8) != (x_scale != nullptr))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_i8_forward: null x or y, or x_scale without an 8-bit x");
    if (x_ld < w->K || y_ld < w->N)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_i8_forward: x_ld=%lld below in_features=%lld, or y_ld=%lld below out_features=%lld",
                       (long long)x_ld, (long long)w->K, (long long)y_ld, (long long)w->N);
    aq_device_guard g(ctx->device);
    args a{w->w, w->scale, w->bias, static_cast<const uint8_t *>(x), x_scale, y, x_ld, y_ld, static_cast<int>(M),
           static_cast<int>(w->N), static_cast<int>(w->K), w->tiles, w->kblocks, y_type};
    if (x_type == AQ_T_I8 && M <= 16) return launch_product<false>(ctx, a);
    int64_t rows = kPackedBytes / (int64_t{w->kblocks} * 64) / 64 * 64;
    if (rows < 64) rows = 64;
    if (rows > (M + 15) / 16 * 16) rows = (M + 15) / 16 * 16;
    const size_t bytes = static_cast<size_t>(rows) * static_cast<size_t>(w->kblocks) * 64;
    uint8_t *packed = nullptr;
    aq_status st = aq_ctx_scratch(ctx, 8, bytes + static_cast<size_t>(rows) * 4, reinterpret_cast<void **>(&packed));
    if (st != AQ_OK) return st;
    float *const scales = reinterpret_cast<float *>(packed + bytes);
    const int64_t x_size = x_type == AQ_T_I8 ? 1 : x_type == AQ_T_F32 ? 4 : 2, y_size = y_type == AQ_T_F32 ? 4 : 2;
    for (int64_t m = 0; m < M; m += rows) {
        args b = a;
        b.M = static_cast<int>(M - m < rows ? M - m : rows);
        const uint8_t *from = static_cast<const uint8_t *>(x) + m * x_ld * x_size;
        i32x4 *const to = reinterpret_cast<i32x4 *>(packed);
        const dim3 grid(static_cast<uint32_t>((b.M + 15) / 16)), block(1024);
        if (x_type == AQ_T_I8)
            aq_launch_timed(ctx, false, i8_pack_kernel, grid, block, 0u, from, x_ld, b.M, b.K, b.kblocks, to);
        else if (x_type == AQ_T_F32)
            aq_launch_timed(ctx, false, i8_quantize_kernel<f32>, grid, block, 0u, reinterpret_cast<const float *>(from), x_ld,
                            b.M, b.K, b.kblocks, to, scales);
        else if (x_type == AQ_T_F16)
            aq_launch_timed(ctx, false, i8_quantize_kernel<f16>, grid, block, 0u, reinterpret_cast<const uint16_t *>(from),
                            x_ld, b.M, b.K, b.kblocks, to, scales);
        else
            aq_launch_timed(ctx, false, i8_quantize_kernel<bf16>, grid, block, 0u, reinterpret_cast<const uint16_t *>(from),
                            x_ld, b.M, b.K, b.kblocks, to, scales);
        AQ_HIP(ctx, hipGetLastError());
        b.x = packed;
        b.x_scale = x_scale ? x_scale + m : scales;
        b.y = static_cast<char *>(y) + m * y_ld * y_size;
        st = launch_product<true>(ctx, b);
        if (st != AQ_OK) return st;
    }
    return AQ_OK;
}

aq_status aq_i8_release(aq_i8 *w) {
    if (!w) return AQ_E_INVALID_ARG;
    aq_device_guard g(w->device);
    free_all(w);
    return AQ_OK;
}

}  // extern "C"
