// Products with 4-bit weights and group scales (aq_q4_*): the upload and the
// C ABI.  The kernels are in aq_q4_kernels.hpp.
#include "aq_q4.hpp"

#include <new>

struct aq_q4 {
    int device = -1;   // of the creating context; the handle may outlive it
    int64_t N = 0, K = 0, group = 0;
    int tiles = 0, kblocks = 0;
    uint8_t *codes = nullptr;
    uint16_t *scale = nullptr;
    uint8_t *zero = nullptr;
    float *bias = nullptr;
};

namespace {

// The tiles' codes from rows of packed ones: one thread a dword.  Rows and
// columns past the end hold code 0 (their scales are 0, and x is 0 there).
__global__ __launch_bounds__(256) void q4_codes_kernel(const uint8_t *from, int64_t row_bytes, int64_t N, int64_t K,
                                                       int64_t kblocks, int64_t dwords, uint32_t *to) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= dwords) return;
    const int64_t j = i & 3, lane = (i >> 2) & 63, block = i >> 8;
    const int64_t n = block / kblocks * 16 + (lane & 15);
    const int64_t k0 = block % kblocks * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    for (int c = 0; c < 8; ++c) {
        if (n >= N || k0 + c >= K) break;
        const uint32_t b = from[n * row_bytes + (k0 + c) / 2];
        w |= (c & 1 ? b >> 4 : b & 15u) << (4 * ((c & 1) * 4 + c / 2));
    }
    to[i] = w;
}

// Scales (or zeros) by tile: [tile][k-block][subs][16]; 0 past the end.
template <typename E>
__global__ __launch_bounds__(256) void q4_groups_kernel(const E *from, int64_t N, int64_t groups, int64_t padded,
                                                        int64_t count, E *to) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= count) return;
    const int64_t n = i / (padded * 16) * 16 + i % 16, g = i / 16 % padded;
    to[i] = n < N && g < groups ? from[n * groups + g] : E(0);
}

uint32_t blocks_of(int64_t n) { return static_cast<uint32_t>((n + 255) / 256); }

// Host array -> temporary device copy.
template <typename E>
hipError_t staged(const E *host, size_t n, E **dev) {
    hipError_t e = hipMalloc(dev, n * sizeof(E));
    return e == hipSuccess ? hipMemcpy(*dev, host, n * sizeof(E), hipMemcpyHostToDevice) : e;
}

void free_all(aq_q4 *w) {
    for (void *p : {static_cast<void *>(w->codes), static_cast<void *>(w->scale), static_cast<void *>(w->zero),
                    static_cast<void *>(w->bias)})
        if (p) (void)hipFree(p);
    delete w;
}

}  // namespace

extern "C" {

aq_status aq_q4_upload(aq_ctx *ctx, int64_t out_features, int64_t in_features, int64_t group, const uint8_t *codes,
                       const void *scale, const uint8_t *zero, const float *bias, aq_q4 **out) {
    if (out) *out = nullptr;
    if (!ctx || !codes || !scale || !out) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_upload: null argument");
    const int64_t N = out_features, K = in_features;
    if (group != 32 && group != 64 && group != 128)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_upload: group %lld is not 32, 64 or 128", (long long)group);
    if (N < 1 || K < 1 || N > (int64_t{1} << 24) || K > (int64_t{1} << 24) || N > (int64_t{1} << 34) / K)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_q4_upload: out_features=%lld in_features=%lld (each 1 to 2^24, 2^34 weights)",
                       (long long)N, (long long)K);
    const int64_t groups = (K + group - 1) / group, row_bytes = (K + 1) / 2;
    if (zero)
        for (int64_t i = 0; i < N * groups; ++i)
            if (zero[i] > 15)
                return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_upload: zero[%lld] = %d is above 15", (long long)i, zero[i]);
    aq_device_guard g(ctx->device);
    aq_q4 *w = new (std::nothrow) aq_q4();
    if (!w) return aq_fail(ctx, AQ_E_NOMEM, "aq_q4_upload: host allocation failed");
    w->device = ctx->device;
    w->N = N;
    w->K = K;
    w->group = group;
    w->tiles = static_cast<int>((N + 15) / 16);
    w->kblocks = static_cast<int>((K + 127) / 128);
    const int64_t dwords = int64_t{w->tiles} * w->kblocks * 256;
    const int64_t padded = w->kblocks * (128 / group), per = int64_t{w->tiles} * padded * 16;

    uint8_t *d_codes = nullptr, *d_zero = nullptr;
    uint16_t *d_scale = nullptr;
    hipError_t e = hipMalloc(&w->codes, static_cast<size_t>(dwords) * 4);
    if (e == hipSuccess) e = hipMalloc(&w->scale, static_cast<size_t>(per) * 2);
    if (e == hipSuccess) e = staged(codes, static_cast<size_t>(N * row_bytes), &d_codes);
    if (e == hipSuccess) e = staged(static_cast<const uint16_t *>(scale), static_cast<size_t>(N * groups), &d_scale);
    if (e == hipSuccess && zero) {
        e = hipMalloc(&w->zero, static_cast<size_t>(per));
        if (e == hipSuccess) e = staged(zero, static_cast<size_t>(N * groups), &d_zero);
    }
    if (e == hipSuccess && bias) e = staged(bias, static_cast<size_t>(N), &w->bias);
    if (e == hipSuccess) {
        hipLaunchKernelGGL(q4_codes_kernel, dim3(blocks_of(dwords)), dim3(256), 0, ctx->stream, d_codes, row_bytes, N, K,
                           int64_t{w->kblocks}, dwords, reinterpret_cast<uint32_t *>(w->codes));
        hipLaunchKernelGGL(q4_groups_kernel<uint16_t>, dim3(blocks_of(per)), dim3(256), 0, ctx->stream, d_scale, N, groups,
                           padded, per, w->scale);
        if (zero)
            hipLaunchKernelGGL(q4_groups_kernel<uint8_t>, dim3(blocks_of(per)), dim3(256), 0, ctx->stream, d_zero, N,
                               groups, padded, per, w->zero);
        e = hipGetLastError();
        const hipError_t e2 = hipStreamSynchronize(ctx->stream);
        if (e == hipSuccess) e = e2;
    }
    for (void *p : {static_cast<void *>(d_codes), static_cast<void *>(d_zero), static_cast<void *>(d_scale)})
        if (p) (void)hipFree(p);
    if (e != hipSuccess) {
        free_all(w);
        (void)hipGetLastError();   // reported below, and no error of the caller's next launch
        return aq_fail(ctx, e == hipErrorOutOfMemory ? AQ_E_NOMEM : AQ_E_DEVICE, "aq_q4_upload: %s", hipGetErrorString(e));
    }
    *out = w;
    return AQ_OK;
}

aq_status aq_q4_forward(aq_ctx *ctx, const aq_q4 *w, int x_type, const void *x, int64_t x_ld, const float *x_scale,
                        int64_t x_group, int64_t M, int y_type, void *y, int64_t y_ld) {
    if (!ctx || !w) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_forward: null argument");
    if (w->device != ctx->device)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_forward: weights belong to another device");
    const bool eight = x_type == AQ_T_I8 || x_type == AQ_T_E4M3;
    if (!eight && x_type != AQ_T_F32 && x_type != AQ_T_F16 && x_type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_forward: unknown x_type %d", x_type);
    if (y_type != AQ_T_F32 && y_type != AQ_T_F16 && y_type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_forward: y_type %d is not F32, F16 or BF16", y_type);
    if (eight && x_group != 0 && x_group != 32 && x_group != 64 && x_group != 128)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_forward: x_group %lld is not 0, 32, 64 or 128", (long long)x_group);
    if (M < 0 || M > int64_t{1} << 20)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_q4_forward: M=%lld (0 to 2^20)", (long long)M);
    if (M == 0) return AQ_OK;
    if (!x || !y || eight != (x_scale != nullptr))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_q4_forward: null x or y, or x_scale without an 8-bit x");
    if (x_ld < w->K || y_ld < w->N)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_q4_forward: x_ld=%lld below in_features=%lld, or y_ld=%lld below out_features=%lld",
                       (long long)x_ld, (long long)w->K, (long long)y_ld, (long long)w->N);
    aq_device_guard g(ctx->device);
    const int xg = eight ? static_cast<int>(x_group) : 0;
    const aq_q4_impl::args a{w->codes, w->scale, w->zero, w->bias, x, x_scale, nullptr, y, x_ld, y_ld, static_cast<int>(M),
                             static_cast<int>(w->N), static_cast<int>(w->K), w->tiles, w->kblocks,
                             static_cast<int>(w->group), xg, xg ? static_cast<int>((w->K + xg - 1) / xg) : 1, y_type};
    switch (x_type) {
    case AQ_T_F32: return aq_q4_impl::launch_f32(ctx, a);
    case AQ_T_F16: return aq_q4_impl::launch_f16(ctx, a);
    case AQ_T_BF16: return aq_q4_impl::launch_bf16(ctx, a);
    case AQ_T_I8: return aq_q4_impl::launch_i8(ctx, a);
    default: return aq_q4_impl::launch_e4m3(ctx, a);
    }
}

aq_status aq_q4_release(aq_q4 *w) {
    if (!w) return AQ_E_INVALID_ARG;
    aq_device_guard g(w->device);
    free_all(w);
    return AQ_OK;
}

}  // extern "C"
