// The product with 4-bit weights (aq_q4_forward), one instantiation set per
// type of x (aq_q4_*.hip, so that they compile in parallel).
//
// Layout.  A tile is 16 rows of W, a k-block 128 columns: 1 KB, 16 bytes a
// lane.  Dword j of lane l holds row l % 16, columns 32 j + 8 (l / 16) ..+7 of
// the k-block, which is the operand of one 16x16x32 matrix instruction; the
// code of column c sits in nibble (c % 2) * 4 + c / 2 of its dword.  Scales
// and zeros are [tile][k-block][128 / group][16 rows].
//
// Floating x.  A code q becomes the 16-bit float 16 + q with one mask and one
// or: the nibble is moved to the top of the mantissa of 16.0.  The sum over a
// group starts from -(16 + zero) * sum(x), which the same instruction gives
// with a constant operand, so no code is converted or corrected on its own.
// The group's sum is scaled in fp32.  An fp32 x is split into three bf16
// parts (8 bits of the mantissa each, by truncation, exact).
//
// 8-bit x.  Whole numbers stay whole: the nibbles as bytes against x's bytes,
// started from -zero * sum(x).  e4m3 converts to f16 exactly.
#pragma once
#include "aq_internal.hpp"
#include "aq_q4.hpp"
#include "aq_types.hpp"

namespace aq_q4_impl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// x8 = 8 columns of a row of x from column k, zeros beyond K.
template <typename E>
__device__ inline void load_x8(const E *row, int k, int K, bool tail, E (&v)[8]) {
    if (!tail || k + 8 <= K) {
        std::memcpy(v, row + k, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : E(0);
    }
}

// What a type of x needs: its element, the operand fragment of 8 columns
// (PARTS of them for a split x), the operand of a dword of codes and of the
// correction, and the matrix instruction.
struct x_f16 {
    using elem = uint16_t;
    using frag = f16x8;
    using acc = f32x4;
    static constexpr int kParts = 1;
    static constexpr bool kScaled = false;
    static __device__ inline void x8(const elem (&v)[8], frag (&f)[kParts]) { std::memcpy(&f[0], v, 16); }
    static __device__ inline frag codes(uint32_t w) {
        constexpr uint32_t m = 0x03C003C0u, c = 0x4C004C00u;
        const uint4 r = make_uint4(((w << 6) & m) | c, ((w << 2) & m) | c, ((w >> 2) & m) | c, ((w >> 6) & m) | c);
        return __builtin_bit_cast(frag, r);
    }
    static __device__ inline frag less(float zero) {
        const _Float16 h = static_cast<_Float16>(-16.0f - zero);
        return frag{h, h, h, h, h, h, h, h};
    }
    static __device__ inline acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

struct x_bf16 {
    using elem = uint16_t;
    using frag = bf16x8;
    using acc = f32x4;
    static constexpr int kParts = 1;
    static constexpr bool kScaled = false;
    static __device__ inline void x8(const elem (&v)[8], frag (&f)[kParts]) { std::memcpy(&f[0], v, 16); }
    static __device__ inline frag codes(uint32_t w) {
        constexpr uint32_t m = 0x00780078u, c = 0x41804180u;
        const uint4 r = make_uint4(((w << 3) & m) | c, ((w >> 1) & m) | c, ((w >> 5) & m) | c, ((w >> 9) & m) | c);
        return __builtin_bit_cast(frag, r);
    }
    static __device__ inline frag less(float zero) {
        const __bf16 h = static_cast<__bf16>(-16.0f - zero);
        return frag{h, h, h, h, h, h, h, h};
    }
    static __device__ inline acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

struct x_f32 : x_bf16 {
    using elem = float;
    static constexpr int kParts = 3;
    static __device__ inline void x8(const elem (&v)[8], frag (&f)[kParts]) {
        uint32_t part[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t hi[2][3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float r = v[2 * i + h];
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    hi[h][p] = __float_as_uint(r) >> 16;
                    r -= __uint_as_float(hi[h][p] << 16);
                }
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) part[p][i] = hi[0][p] | (hi[1][p] << 16);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) std::memcpy(&f[p], part[p], 16);
    }
};

struct x_e4m3 : x_f16 {
    using elem = uint8_t;
    static constexpr bool kScaled = true;
    static __device__ inline void x8(const elem (&v)[8], frag (&f)[kParts]) {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        uint32_t w[2];
        std::memcpy(w, v, 8);
        pair p[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false);
            p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true);
        }
        std::memcpy(&f[0], p, 16);
    }
};

struct x_i8 {
    using elem = uint8_t;
    using frag = long;
    using acc = i32x4;
    static constexpr int kParts = 1;
    static constexpr bool kScaled = true;
    // The columns in the order of the codes' bytes below: 0 4 1 5, 2 6 3 7.
    static __device__ inline void x8(const elem (&v)[8], frag (&f)[kParts]) {
        uint32_t w[2];
        std::memcpy(w, v, 8);
        const uint32_t r[2] = {__builtin_amdgcn_perm(w[1], w[0], 0x05010400u), __builtin_amdgcn_perm(w[1], w[0], 0x07030602u)};
        std::memcpy(&f[0], r, 8);
    }
    static __device__ inline frag codes(uint32_t w) {
        const uint32_t r[2] = {w & 0x0F0F0F0Fu, (w >> 4) & 0x0F0F0F0Fu};
        return __builtin_bit_cast(frag, r);
    }
    static __device__ inline frag less(float zero) {
        const uint32_t b = static_cast<uint32_t>(-static_cast<int>(zero)) & 255u;
        const uint32_t r[2] = {b * 0x01010101u, b * 0x01010101u};
        return __builtin_bit_cast(frag, r);
    }
    static __device__ inline acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_i32_16x16x32_i8(a, b, c, 0, 0, 0); }
};

// A block: RT tiles of rows times 16 MT rows of x; its waves take the
// k-blocks in turn and their sums are joined in LDS, in the waves' order.
// SUBS: parts of a k-block with scales of their own (128 over the smaller of
// the two groups).
template <typename X, int SUBS, int RT, int MT>
__global__ __launch_bounds__(512) void q4_product_kernel(args a) {
    extern __shared__ float red[];   // [waves][RT * MT][64][4]
    using frag = typename X::frag;
    using acc_t = typename X::acc;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int tile0 = blockIdx.x * RT, m0 = blockIdx.y * 16 * MT;
    const int subs_w = 128 / a.group;   // scales of W in a k-block

    const typename X::elem *xrow[MT];
    const float *xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = min(m0 + 16 * t + col, a.M - 1);   // rows past the end repeat the last one; they are not written
        xrow[t] = static_cast<const typename X::elem *>(a.x) + m * a.x_ld;
        xs[t] = X::kScaled ? a.x_scale + static_cast<int64_t>(m) * a.x_groups : nullptr;
    }
    int tile[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) tile[r] = min(tile0 + r, a.tiles - 1);

    f32x4 sum[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[r][t] = f32x4{0, 0, 0, 0};

    for (int kb = wave; kb < a.kblocks; kb += waves) {
        const bool tail = kb * 128 + 128 > a.K;
        uint32_t w[RT][4];
#pragma unroll
        for (int r = 0; r < RT; ++r)
            std::memcpy(w[r], a.codes + ((static_cast<int64_t>(tile[r]) * a.kblocks + kb) * 64 + lane) * 16, 16);
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            const int sw = s * subs_w / SUBS;
            // Per row tile: the scales of this lane's four result rows, and the zero of its operand row.
            float ws[RT][4], zero[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int64_t at = ((static_cast<int64_t>(tile[r]) * a.kblocks + kb) * subs_w + sw) * 16;
                uint16_t h[4];
                std::memcpy(h, a.scale + at + 4 * quad, 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) ws[r][i] = aq_types::f16::load(h[i]);
                zero[r] = a.zero ? static_cast<float>(a.zero[at + col]) : 8.0f;
            }
            acc_t acc[RT][MT];
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[r][t] = acc_t{0, 0, 0, 0};
#pragma unroll
            for (int j = s * 4 / SUBS; j < (s + 1) * 4 / SUBS; ++j) {
                frag b[MT][X::kParts];
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    typename X::elem v[8];
                    load_x8(xrow[t], kb * 128 + 32 * j + 8 * quad, a.K, tail, v);
                    X::x8(v, b[t]);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const frag q = X::codes(w[r][j]), z = X::less(zero[r]);
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int p = 0; p < X::kParts; ++p) {
                            acc[r][t] = X::mma(z, b[t][p], acc[r][t]);
                            acc[r][t] = X::mma(q, b[t][p], acc[r][t]);
                        }
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float f = 1.0f;
                if (X::kScaled && a.x_group) f = xs[t][min(kb * 128 + s * (128 / SUBS), a.K - 1) / a.x_group];
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sum[r][t][i] = __fmaf_rn(X::kScaled ? ws[r][i] * f : ws[r][i], static_cast<float>(acc[r][t][i]),
                                                 sum[r][t][i]);
            }
        }
    }

    f32x4 *red4 = reinterpret_cast<f32x4 *>(red);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) red4[(wave * RT * MT + r * MT + t) * 64 + lane] = sum[r][t];
    __syncthreads();
    for (int i = wave; i < RT * MT; i += waves) {
        f32x4 v = red4[i * 64 + lane];
        for (int k = 1; k < waves; ++k) v += red4[(k * RT * MT + i) * 64 + lane];
        const int n = (tile0 + i / MT) * 16 + 4 * quad, m = m0 + 16 * (i % MT) + col;
        if (m >= a.M || n >= a.N) continue;
        if (X::kScaled && !a.x_group) v *= a.x_scale[m];
        float o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = a.bias && n + c < a.N ? v[c] + a.bias[n + c] : v[c];
        const int64_t at = m * a.y_ld + n;
        if (a.y_type == AQ_T_F32) {
            float *y = static_cast<float *>(a.y) + at;
            if (n + 4 <= a.N) std::memcpy(y, o, 16);
            else for (int c = 0; c < a.N - n; ++c) y[c] = o[c];
        } else {
            uint16_t h[4];
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                if (a.y_type == AQ_T_F16) aq_types::f16::store2(h + c, o[c], o[c + 1]);
                else aq_types::bf16::store2(h + c, o[c], o[c + 1]);
            }
            uint16_t *y = static_cast<uint16_t *>(a.y) + at;
            if (n + 4 <= a.N) std::memcpy(y, h, 8);
            else for (int c = 0; c < a.N - n; ++c) y[c] = h[c];
        }
    }
}

template <typename X, int SUBS, int RT, int MT>
aq_status launch_shape(aq_ctx *ctx, const args &a) {
    const int waves = a.kblocks < 8 ? a.kblocks : 8;
    const uint32_t lds = static_cast<uint32_t>(waves * RT * MT * 1024);
    auto kernel = q4_product_kernel<X, SUBS, RT, MT>;
    aq_status st = aq_launch_lds(ctx, reinterpret_cast<const void *>(kernel), lds, "aq_q4_forward");
    if (st != AQ_OK) return st;
    const dim3 grid(static_cast<uint32_t>((a.tiles + RT - 1) / RT), static_cast<uint32_t>((a.M + 16 * MT - 1) / (16 * MT)));
    aq_launch_timed(ctx, true, kernel, grid, dim3(static_cast<uint32_t>(64 * waves)), lds, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}

template <typename X, int SUBS>
aq_status launch_subs(aq_ctx *ctx, const args &a) {
    if (a.M <= 16) return launch_shape<X, SUBS, 1, 1>(ctx, a);
    if (a.M <= 32) return launch_shape<X, SUBS, 2, 2>(ctx, a);
    return launch_shape<X, SUBS, 2, 4>(ctx, a);
}

template <typename X>
aq_status launch(aq_ctx *ctx, const args &a) {
    int least = a.group;
    if (X::kScaled && a.x_group && a.x_group < least) least = a.x_group;
    if (least == 128) return launch_subs<X, 1>(ctx, a);
    if (least == 64) return launch_subs<X, 2>(ctx, a);
    return launch_subs<X, 4>(ctx, a);
}

}  // namespace aq_q4_impl
