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
// or: the nibble is moved to the top of the mantissa of 16.0.  A group's sum
// is then sum(x (16 + q)) - (16 + zero) sum(x), the second sum from the same
// instruction with ones for codes, shared by all tiles of rows: no code is
// converted or corrected on its own.  It is scaled in fp32.  An fp32 x is
// split into three bf16 parts (8 bits of the mantissa each, by truncation,
// exact).  The upper part's sums have few bits and are nearly exact; the lower
// parts have sums of their own, since next to the upper ones, which the offset
// of 16 + q makes several times the result, they would be rounded at that size
// (5 x 1000 x 4099, rows of mean 2: 1.4e-6 of the result, and 2e-7 apart).
//
// 8-bit x.  Whole numbers stay whole: the nibbles as bytes against x's bytes,
// and zero * sum(x) taken off (all below 2^24, so exact in fp32 as well).
// e4m3 converts to f16 exactly.
//
// What bounds it.  Up to 16 rows of x, the codes' way from memory: 8192 x
// 28672, one int8 row, 121 MB in 26 us, 4.7 TB/s, where a copy of 2 GB runs
// at 4.8.  Small matrices, latency: 1024 x 12288, one bf16 row, 5.6 us.  Many
// rows, x from the caches and few waves to wait for it: for 64 rows of f16 by
// 4096 x 16384 each of 512 blocks of two tiles reads all of the packed x, 268
// MB beside 38 MB from memory, with two waves a SIMD (196 registers): 19 us
// with 3 us of packing, the matrix instructions 37 % of it and the codes'
// conversion as much.  Groups of 64 and 32 columns hold more scales: their
// packed kernels have 280 to 320 registers there, one wave a SIMD, and take 36
// to 42 and 67 to 73 us.
#pragma once
#include "aq_internal.hpp"
#include "aq_q4.hpp"
#include "aq_types.hpp"

namespace aq_q4_impl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// N words in registers, and their load from any address.  (Vectors and single
// words: copied arrays are taken apart into bytes by the compiler.)
template <int N> struct words;
template <> struct words<1> {
    uint32_t v;
    __device__ inline void load(const void *p) {
        typedef uint32_t any __attribute__((aligned(1)));
        v = *static_cast<const any *>(p);
    }
    __device__ inline uint32_t operator[](int) const { return v; }
    __device__ inline void set(int, uint32_t w) { v = w; }
};
template <> struct words<2> {
    u32x2 v;
    __device__ inline void load(const void *p) {
        typedef u32x2 any __attribute__((aligned(1)));
        v = *static_cast<const any *>(p);
    }
    __device__ inline uint32_t operator[](int i) const { return v[i]; }
    __device__ inline void set(int i, uint32_t w) { v[i] = w; }
};
template <> struct words<4> {
    u32x4 v;
    __device__ inline void load(const void *p) {
        typedef u32x4 any __attribute__((aligned(1)));
        v = *static_cast<const any *>(p);
    }
    // Read once: an aligned load that is the first to leave the caches.
    __device__ inline void stream(const void *p) { v = __builtin_nontemporal_load(static_cast<const u32x4 *>(p)); }
    __device__ inline uint32_t operator[](int i) const { return v[i]; }
    __device__ inline void set(int i, uint32_t w) { v[i] = w; }
};
template <> struct words<8> {
    words<4> a, b;
    __device__ inline void load(const void *p) {
        a.load(p);
        b.load(static_cast<const char *>(p) + 16);
    }
    __device__ inline uint32_t operator[](int i) const { return i < 4 ? a[i] : b[i - 4]; }
    __device__ inline void set(int i, uint32_t w) {
        if (i < 4) a.set(i, w);
        else b.set(i - 4, w);
    }
};

// What a type of x needs: its element, the operand fragment of 8 columns
// (kParts of them for a split x, whose sums go to kSums accumulators: the
// first part to the first, the others to the last), the operand of a dword of
// codes and of the correction, and the matrix instruction.
struct x_f16 {
    using elem = uint16_t;
    using frag = f16x8;
    using acc = f32x4;
    static constexpr int kParts = 1, kSums = 1;
    static constexpr bool kScaled = false;
    static __device__ inline void x8(const words<4> &v, frag (&f)[kParts]) { f[0] = __builtin_bit_cast(frag, v.v); }
    static __device__ inline frag codes(uint32_t w) {
        uint32_t m = 0x03C003C0u;
        constexpr uint32_t c = 0x4C004C00u;
        asm("" : "+v"(m));   // in a vector register, so that mask and or are one instruction
        const u32x4 r = {((w << 6) & m) | c, ((w << 2) & m) | c, ((w >> 2) & m) | c, ((w >> 6) & m) | c};
        return __builtin_bit_cast(frag, r);
    }
    static constexpr float kBias = 16.0f;   // codes() gives q + kBias
    static __device__ inline frag ones() {
        const _Float16 h = static_cast<_Float16>(1.0f);
        return frag{h, h, h, h, h, h, h, h};
    }
    static __device__ inline acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

struct x_bf16 {
    using elem = uint16_t;
    using frag = bf16x8;
    using acc = f32x4;
    static constexpr int kParts = 1, kSums = 1;
    static constexpr bool kScaled = false;
    static __device__ inline void x8(const words<4> &v, frag (&f)[kParts]) { f[0] = __builtin_bit_cast(frag, v.v); }
    static __device__ inline frag codes(uint32_t w) {
        uint32_t m = 0x00780078u;
        constexpr uint32_t c = 0x41804180u;
        asm("" : "+v"(m));   // in a vector register, so that mask and or are one instruction
        const u32x4 r = {((w << 3) & m) | c, ((w >> 1) & m) | c, ((w >> 5) & m) | c, ((w >> 9) & m) | c};
        return __builtin_bit_cast(frag, r);
    }
    static constexpr float kBias = 16.0f;   // codes() gives q + kBias
    static __device__ inline frag ones() {
        const __bf16 h = static_cast<__bf16>(1.0f);
        return frag{h, h, h, h, h, h, h, h};
    }
    static __device__ inline acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

struct x_f32 : x_bf16 {
    using elem = float;
    static constexpr int kParts = 3, kSums = 2;
    static __device__ inline void x8(const words<8> &v, frag (&f)[kParts]) {
        u32x4 part[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t hi[2][3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float r = __uint_as_float(v[2 * i + h]);
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
        for (int p = 0; p < 3; ++p) f[p] = __builtin_bit_cast(frag, part[p]);
    }
};

struct x_e4m3 : x_f16 {
    using elem = uint8_t;
    static constexpr bool kScaled = true;
    static __device__ inline void x8(const words<2> &w, frag (&f)[kParts]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false));
            r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true));
        }
        f[0] = __builtin_bit_cast(frag, r);
    }
};

struct x_i8 {
    using elem = uint8_t;
    using frag = long;
    using acc = i32x4;
    static constexpr int kParts = 1, kSums = 1;
    static constexpr bool kScaled = true;
    // The columns in the order of the codes' bytes below: 0 4 1 5, 2 6 3 7.
    static __device__ inline void x8(const words<2> &w, frag (&f)[kParts]) {
        const u32x2 r = {__builtin_amdgcn_perm(w[1], w[0], 0x05010400u), __builtin_amdgcn_perm(w[1], w[0], 0x07030602u)};
        f[0] = __builtin_bit_cast(frag, r);
    }
    static __device__ inline frag codes(uint32_t w) {
        const u32x2 r = {w & 0x0F0F0F0Fu, (w >> 4) & 0x0F0F0F0Fu};
        return __builtin_bit_cast(frag, r);
    }
    static constexpr float kBias = 0.0f;
    static __device__ inline frag ones() { return 0x0101010101010101l; }
    static __device__ inline acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_i32_16x16x32_i8(a, b, c, 0, 0, 0); }
};

// A block: RT tiles of rows times 16 MT rows of x; its waves take the
// k-blocks in turn and their sums are joined in LDS, in the waves' order.
// SUBS: parts of a k-block with scales of their own (128 over the smaller of
// the two groups).  AHEAD: the codes and scales of two k-blocks are on their
// way or in use at any time, and J 32-column steps of x ahead of those in use
// (x comes from a near cache, the codes from memory); without it each wave has
// one k-block or two, and less code to fetch.
template <typename X, bool PACKED, int MT, int J>
struct x_step {
    // Words of 8 columns of x: as they are, or the operand fragments.
    static constexpr int kWords = PACKED ? sizeof(typename X::frag) / 4 : 2 * sizeof(typename X::elem);
    static constexpr int kPieces = PACKED ? X::kParts : 1;
    words<kWords> v[MT][J][kPieces];
};

// The scales and zeros of a group, of this lane's four result rows per tile,
// as they are stored, and the scales of its rows of x.
template <int RT, int MT, int SUMS>
struct scales {
    words<2> w[RT];
    words<1> zero[RT];
    float x[MT], x1[SUMS][MT];   // a packed x's scale, and its sums over the group
};

// PACKED: x and its sums are what q4_pack_kernel wrote.  STREAM: the codes pass
// the caches once (8192 x 28672: 26.2 us, 27.5 with plain loads); a small
// matrix, or one that several rows of blocks read, is better left in them.
// (Two waves a SIMD at least: left free, the packed kernel with two sums takes
// 268 registers with SUBS = 2, one wave a SIMD, and 220 so, without a spill.)
template <typename X, bool PACKED, bool AHEAD, bool STREAM, int SUBS, int RT, int MT, int J>
__global__ __launch_bounds__(PACKED || RT > 2 ? 256 : 512, PACKED && X::kSums == 2 ? 2 : 1) void q4_product_kernel(args a) {
    using x_t = x_step<X, PACKED, MT, J>;
    extern __shared__ float red[];   // [waves][RT * MT][64][4]
    using frag = typename X::frag;
    using acc_t = typename X::acc;
    using elem = typename X::elem;
    constexpr int kSteps = 4 / J, kPer = 4 / SUBS;   // loads of a k-block; 32-column steps with one scale
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    // An even share of the tiles, at most RT of them; the first blocks have one more.
    const int share = a.tiles / static_cast<int>(gridDim.x), more = a.tiles % static_cast<int>(gridDim.x);
    const int tile0 = static_cast<int>(blockIdx.x) * share + min(static_cast<int>(blockIdx.x), more);
    const int tiles = share + (static_cast<int>(blockIdx.x) < more ? 1 : 0), m0 = blockIdx.y * 16 * MT;
    const int subs_w = 128 / a.group;   // scales of W in a k-block

    const elem *xrow[MT];
    const float *xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = min(m0 + 16 * t + col, a.M - 1);   // rows past the end repeat the last one; they are not written
        if (!PACKED) xrow[t] = static_cast<const elem *>(a.x) + m * a.x_ld + 8 * quad;
        xs[t] = X::kScaled ? a.x_scale + static_cast<int64_t>(m) * a.x_groups : nullptr;
    }
    int64_t tile[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) tile[r] = static_cast<int64_t>(tile0 + min(r, tiles - 1)) * a.kblocks;   // past its share: the last again

    const auto load_codes = [&](int kb, words<4> (&w)[RT]) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const uint8_t *from = a.codes + ((tile[r] + kb) * 64 + lane) * 16;
            if constexpr (STREAM) w[r].stream(from);
            else w[r].load(from);
        }
    };
    const auto load_x = [&](int kb, int part, x_t &x) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if constexpr (PACKED) {
                    const int64_t at = (static_cast<int64_t>(m0 / 16 + t) * a.kblocks + kb) * 4 + part * J + j;
#pragma unroll
                    for (int p = 0; p < X::kParts; ++p)
                        x.v[t][j][p].load(static_cast<const frag *>(a.x) + (at * X::kParts + p) * 64 + lane);
                } else {
                    x.v[t][j][0].load(xrow[t] + kb * 128 + (part * J + j) * 32);
                }
            }
    };
    const auto load_scales = [&](int kb, int s, scales<RT, MT, X::kSums> &c) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int64_t at = ((tile[r] + kb) * subs_w + s * subs_w / SUBS) * 16 + 4 * quad;
            c.w[r].load(a.scale + at);
            if (a.zero) c.zero[r].load(a.zero + at);
            else c.zero[r].v = 0x08080808u;
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
        {
            c.x[t] = X::kScaled && a.x_group ? xs[t][min(kb * 128 + s * (128 / SUBS), a.K - 1) / a.x_group] : 1.0f;
            if (PACKED) {
                const int64_t at = ((static_cast<int64_t>(m0 / 16 + t) * a.kblocks + kb) * SUBS + s) * X::kSums;
#pragma unroll
                for (int i = 0; i < X::kSums; ++i) c.x1[i][t] = a.x_sum[(at + i) * 16 + col];
            }
        }
    };

    f32x4 sum[RT][MT];
    acc_t acc[X::kSums][RT][MT], all[X::kSums][MT];   // a group's sums of the codes' products, and of x
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[r][t] = f32x4{0, 0, 0, 0};
    const auto open = [&] {
#pragma unroll
        for (int i = 0; i < X::kSums; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                all[i][t] = acc_t{0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[i][r][t] = acc_t{0, 0, 0, 0};
            }
    };
    const auto add32 = [&](const words<4> (&w)[RT], int at, const x_t &x, int j) {
        frag q[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) q[r] = X::codes(w[r][at]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            frag b[X::kParts];
            if constexpr (PACKED) {
#pragma unroll
                for (int p = 0; p < X::kParts; ++p) b[p] = __builtin_bit_cast(frag, x.v[t][j][p].v);
            } else {
                X::x8(x.v[t][j][0], b);
            }
#pragma unroll
            for (int p = 0; p < X::kParts; ++p) {
                constexpr int kLast = X::kSums - 1;
                const int to = p < kLast ? p : kLast;
                if (!PACKED) all[to][t] = X::mma(X::ones(), b[p], all[to][t]);
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[to][r][t] = X::mma(q[r], b[p], acc[to][r][t]);
            }
        }
    };
    const auto close = [&](const scales<RT, MT, X::kSums> &c) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ws = aq_types::f16::load(static_cast<uint16_t>(c.w[r][i / 2] >> (i % 2 * 16)));
                const float less = -X::kBias - static_cast<float>((c.zero[r].v >> (8 * i)) & 255u);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    float v[X::kSums];
#pragma unroll
                    for (int p = 0; p < X::kSums; ++p)
                        v[p] = __fmaf_rn(less, PACKED ? c.x1[p][t] : static_cast<float>(all[p][t][0]),
                                         static_cast<float>(acc[p][r][t][i]));
                    if (X::kSums == 2) v[0] += v[X::kSums - 1];
                    sum[r][t][i] = __fmaf_rn(X::kScaled ? ws * c.x[t] : ws, v[0], sum[r][t][i]);
                }
            }
    };

    const int whole = PACKED ? a.kblocks : a.K / 128;   // k-blocks without columns past the end
    constexpr int kSets = AHEAD ? 2 : 1;
    words<4> w[kSets][RT];
    scales<RT, MT, X::kSums> c[kSets][SUBS];
    x_t x[2];
    const auto load_block = [&](int kb, int d) {
        load_codes(kb, w[d]);
#pragma unroll
        for (int s = 0; s < SUBS; ++s) load_scales(kb, s, c[d][s]);
    };
    if constexpr (AHEAD) {
        if (wave < whole) {
            load_x(wave, 0, x[0]);
            load_block(wave, 0);
        }
        if (wave + waves < whole) load_block(wave + waves, 1);
    }
#pragma unroll 1
    for (int kb0 = wave; kb0 < whole; kb0 += kSets * waves) {
        if constexpr (!AHEAD) {
            load_x(kb0, 0, x[0]);
            load_block(kb0, 0);
        }
#pragma unroll
        for (int d = 0; d < kSets; ++d) {
            const int kb = kb0 + d * waves;
            if (AHEAD && kb >= whole) break;
#pragma unroll
            for (int part = 0; part < kSteps; ++part) {
                x_t &next = x[(d * kSteps + part + 1) % 2];
                if (part + 1 < kSteps) load_x(kb, part + 1, next);
                else if (AHEAD && kb + waves < whole) load_x(kb + waves, 0, next);
                __builtin_amdgcn_sched_barrier(0);   // the loads go out before the arithmetic
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int at = part * J + j;   // 32-column step of the k-block
                    if (at % kPer == 0) open();
                    add32(w[d], at, x[(d * kSteps + part) % 2], j);
                    if ((at + 1) % kPer == 0) close(c[d][at / kPer]);
                }
            }
            if (AHEAD && kb + 2 * waves < whole) load_block(kb + 2 * waves, d);
        }
    }
    if (!PACKED && whole < a.kblocks && wave == whole % waves) {   // the last columns, one step at a time, zeros beyond K
#pragma unroll 1
        for (int at = 0; at < 4; ++at) {
            if (at % kPer == 0) {
                open();
                load_scales(whole, at / kPer, c[0][0]);
            }
            const int k0 = whole * 128 + 32 * at;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                words<1> one;
                one.load(a.codes + ((tile[r] + whole) * 64 + lane) * 16 + at * 4);
                w[0][r].set(0, one.v);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < x_t::kWords; ++i) {
                    constexpr int kIn = 4 / sizeof(elem);   // elements of a word
                    uint32_t word = 0;
#pragma unroll
                    for (int e = 0; e < kIn; ++e)
                        if (k0 + 8 * quad + i * kIn + e < a.K)
                            word |= aq_types::bits_of(xrow[t][k0 + i * kIn + e]) << (8 * static_cast<int>(sizeof(elem)) * e);
                    x[0].v[t][0][0].set(i, word);
                }
            add32(w[0], 0, x[0], 0);
            if ((at + 1) % kPer == 0) close(c[0][0]);
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
        if (m >= a.M || n >= a.N || i / MT >= tiles) continue;
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

// x in the order of the matrix instructions' operands, converted and with
// zeros past M and K: [16 rows][k-block][4 steps][parts][64 lanes].  A lane of
// the product reads 16 (or 8) bytes next to its neighbour's, where a row of x
// gives it 16 bytes of each of 16 rows: for many rows that, not the
// arithmetic, was what the product waited for (64 rows, 4096 x 16384: 39 us,
// and 19 with the packing).
// With them the sums of x over each of a k-block's `subs` parts, [16 rows]
// [k-block][subs][kSums][16], as the products' groups need them.
template <typename X>
__global__ __launch_bounds__(256) void q4_pack_kernel(args a, void *to, float *sums, int subs) {
    __shared__ float part[4][X::kSums][16];
    using elem = typename X::elem;
    using frag = typename X::frag;
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6;
    const int kb = blockIdx.x, m = blockIdx.y * 16 + (lane & 15), k = kb * 128 + 32 * j + 8 * (lane >> 4);
    const elem *row = static_cast<const elem *>(a.x) + m * a.x_ld;
    words<2 * sizeof(elem)> x;
    if (m < a.M && k + 8 <= a.K) {
        x.load(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(elem)); ++i) {
            constexpr int kIn = 4 / sizeof(elem);
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < kIn; ++e)
                if (m < a.M && k + i * kIn + e < a.K)
                    word |= aq_types::bits_of(row[k + i * kIn + e]) << (8 * static_cast<int>(sizeof(elem)) * e);
            x.set(i, word);
        }
    }
    frag f[X::kParts];
    X::x8(x, f);
    const int64_t at = (static_cast<int64_t>(blockIdx.y) * a.kblocks + kb) * 4 + j;
#pragma unroll
    for (int p = 0; p < X::kParts; ++p) static_cast<frag *>(to)[(at * X::kParts + p) * 64 + lane] = f[p];
    typename X::acc all[X::kSums];
#pragma unroll
    for (int i = 0; i < X::kSums; ++i) all[i] = typename X::acc{0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < X::kParts; ++p) {   // each lane: its row's 32 columns
        constexpr int kLast = X::kSums - 1;
        const int to_sum = p < kLast ? p : kLast;
        all[to_sum] = X::mma(X::ones(), f[p], all[to_sum]);
    }
    if (lane < 16) {
#pragma unroll
        for (int i = 0; i < X::kSums; ++i) part[j][i][lane] = static_cast<float>(all[i][0]);
    }
    __syncthreads();
    const int per = 4 / subs, s = threadIdx.x / 16;
    if (s < subs) {
#pragma unroll
        for (int i = 0; i < X::kSums; ++i) {
            float sum = 0.0f;
            for (int k32 = 0; k32 < per; ++k32) sum += part[s * per + k32][i][lane & 15];
            sums[(((static_cast<int64_t>(blockIdx.y) * a.kblocks + kb) * subs + s) * X::kSums + i) * 16 + (lane & 15)] = sum;
        }
    }
}

template <typename X, bool PACKED, bool AHEAD, bool STREAM, int SUBS, int RT, int MT, int J>
aq_status launch_shape(aq_ctx *ctx, const args &a, int waves) {
    if (waves > a.kblocks) waves = a.kblocks;
    const uint32_t lds = static_cast<uint32_t>(waves * RT * MT * 1024);
    auto kernel = q4_product_kernel<X, PACKED, AHEAD, STREAM, SUBS, RT, MT, J>;
    aq_status st = aq_launch_lds(ctx, reinterpret_cast<const void *>(kernel), lds, "aq_q4_forward");
    if (st != AQ_OK) return st;
    const dim3 grid(static_cast<uint32_t>((a.tiles + RT - 1) / RT), static_cast<uint32_t>((a.M + 16 * MT - 1) / (16 * MT)));
    aq_launch_timed(ctx, true, kernel, grid, dim3(static_cast<uint32_t>(64 * waves)), lds, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}

template <typename X, int SUBS>
aq_status launch_subs(aq_ctx *ctx, const args &a) {
    // Up to 16 rows of x.  Bound by the codes' way from memory, and where a
    // wave has few of them by latency: all in one, 8192 x 28672 takes an int8
    // row at 4.6 TB/s.  Several tiles a block load x once for all of them, but
    // leave fewer blocks.  In us, for 1 and 16 rows at K = 4096, group 128:
    //                        int8          bf16
    //    512 tiles, one     7.5  13.4     7.5  12.0
    //               two     7.5   9.6     8.3   9.5
    //   1024 tiles, two    10.7  15.4    11.3  14.5
    //               four   11.4  12.4    14.4  14.7
    // and at K = 8192, 1792 tiles: two 30.3 and 47.2, 33.3 and 43.0, four 28.4
    // and 31.8, 36.3 and 34.5: the bound for few rows follows int8, and a
    // floating row is 3 us slower there with four tiles than with two.  With 32 columns a scale four tiles' scales do
    // not fit the registers; there one row (bf16, 1792 tiles) takes 49 us with
    // one tile, 67 with two, 16 rows 74 and 70, fp32 96 and 96, 129 and 109.
    if (a.M <= 16) {
        const bool few = a.M <= 4;
        // A wave has one k-block: no loads ahead, less code to fetch (1000 x
        // 4099, five fp32 rows: 6.0 us, 8.2 with them).
        if (a.kblocks <= 8) return launch_shape<X, false, false, false, SUBS, 1, 1, 4>(ctx, a, 8);
        if (a.tiles < 512) return launch_shape<X, false, true, false, SUBS, 1, 1, 4>(ctx, a, 8);
        // Two tiles' sums of an fp32 x leave registers for half a k-block of it.
        constexpr int kJ = SUBS == 4 && X::kSums == 2 ? 2 : 4;
        if (a.tiles < (few ? 1536 : 1024)) return launch_shape<X, false, true, true, SUBS, 2, 1, kJ>(ctx, a, 8);
        if constexpr (SUBS < 4) return launch_shape<X, false, true, true, SUBS, 4, 1, 4>(ctx, a, 4);
        else if (few) return launch_shape<X, false, true, true, SUBS, 1, 1, 4>(ctx, a, 4);
        else return launch_shape<X, false, true, true, SUBS, 2, 1, kJ>(ctx, a, 4);
    }
    // Packed batches of rows, at most 64 MB of them (but 64 rows).
    const int64_t row_bytes = static_cast<int64_t>(a.kblocks) * 16 * sizeof(typename X::frag) * X::kParts;
    int64_t rows = (int64_t{64} << 20) / row_bytes / 64 * 64;
    if (rows < 64) rows = 64;
    if (rows > (a.M + 63) / 64 * 64) rows = (a.M + 63) / 64 * 64;
    char *packed = nullptr;
    const size_t bytes = static_cast<size_t>(rows * row_bytes);
    aq_status st = aq_ctx_scratch(ctx, 8, bytes + static_cast<size_t>(rows) * a.kblocks * SUBS * X::kSums * 4,
                                  reinterpret_cast<void **>(&packed));
    if (st != AQ_OK) return st;
    float *sums = reinterpret_cast<float *>(packed + bytes);
    for (int64_t m = 0; m < a.M; m += rows) {
        args b = a;
        b.M = static_cast<int>(a.M - m < rows ? a.M - m : rows);
        b.x = static_cast<const typename X::elem *>(a.x) + m * a.x_ld;
        b.x_scale = a.x_scale ? a.x_scale + m * a.x_groups : nullptr;
        b.y = static_cast<char *>(a.y) + m * a.y_ld * (a.y_type == AQ_T_F32 ? 4 : 2);
        const dim3 grid(static_cast<uint32_t>(a.kblocks), static_cast<uint32_t>((b.M + 63) / 64 * 4));
        aq_launch_timed(ctx, false, q4_pack_kernel<X>, grid, dim3(256), 0u, b, static_cast<void *>(packed), sums, SUBS);
        b.x = packed;
        b.x_sum = sums;
        // 64 rows of x at once where the registers hold their sums and the
        // grid has two blocks a compute unit, else 32: 64 rows, K = 4096, bf16:
        // 14.2 and 10.7 us for 4096 columns, 19.5 and 20.2 for 16384.  (With
        // 64 columns a scale only one of the two fits a compute unit at a time.)
        // With 32 columns a scale the two sums of an fp32 x leave registers
        // for one tile and 16 rows: in us for 4096 and 16384 columns, 64 rows
        // 30 and 93, 30 and 102 as the others have it, 256 rows 88 and 327, 105
        // and 384.
        constexpr bool kWide = SUBS != 4 && X::kParts == 1;
        constexpr int kTiles = SUBS == 4 && X::kSums == 2 ? 1 : 2;
        const int64_t blocks = static_cast<int64_t>((a.tiles + 1) / 2) * ((b.M + 63) / 64);
        bool wide = false;
        if constexpr (kWide) {
            wide = blocks >= 512 && b.M > 32;
            if (wide) st = launch_shape<X, true, true, false, SUBS, 2, 4, 1>(ctx, b, 4);
        }
        if (!wide) st = launch_shape<X, true, true, false, SUBS, kTiles, kTiles, X::kParts == 1 ? 2 : 1>(ctx, b, 4);
        if (st != AQ_OK) return st;
    }
    return AQ_OK;
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
