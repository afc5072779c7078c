// Attention to an encoder's states and over a shared prefix (aq_cross_attention,
// aq_prefix_attention).
//
// A row r of a head's group of G query heads is (token, head of the group).
// One pass over the keys with each row's running maximum m and weight l:
//   s = q . k,  m' = max(m, c max s),  p = 2^(c s - m'),
//   o = o 2^(m - m') + sum p v,  l = l 2^(m - m') + sum p,   out = o / l
// with c = scale log2(e).  m' stays m while it would grow by no more than 5:
// a p of up to 32 is as good as one of up to 1, and most tiles rescale nothing.
// m is c times a score.  Its rounding shifts all exponents of a row alike, which
// out does not see; where m is so large that the shift is not small beside 1
// (or has no value in fp32), they are c (s - score) instead.  That path is one
// branch of a tile (8 x 4096 rows over 1500 keys 449 -> 452 us, 16 x 512 over
// 8192 + 512 569 -> 577).
//
// Both products have the keys' side as the first operand, so that every lane
// works for one row: S^T = K Q^T has a row per column, the lane's own, with 16
// of a tile's 32 keys in its registers and the other 16 in lane ^ 32, and O^T =
// V^T P^T takes p from those registers as they are: the order of the keys in
// the second product is the one that the first leaves, and V is read from LDS
// in that order, by the loads that transpose (16-bit types) or one value a
// lane (fp32).  A row's m, l and rescaling are plain registers; one exchange
// per tile joins the two halves' maxima.
//
// Scores, m, l and o are fp32.  p is rounded to the 16-bit type of v (by at most
// 2^-8 of itself, 2^-11 for f16, with errors of either sign that the sum over
// the keys averages); an f16 p is 2^10 times the weight, so that small weights
// are not lost below its range.  fp32 inputs keep fp32 products throughout.
//
// What bounds it.  Many rows: 870 to 980 TFLOP/s (8 x 4096 rows of 16 heads over
// 1500 keys in 452 us, 16 x 512 rows over a prefix of 8192 in 577), where a
// large product of the library's reaches 1110 to 1270: the matrix instructions
// 45 % of the clocks and the vector instructions (two thirds of them for the
// exponentials) 51 %, on two waves a SIMD (227 registers) that
// cover each other's waits.  Few rows, the keys' way from memory: 64 streams over
// 1500 keys, 266 MB, 55 us (4.8 TB/s).  Both at once, a token of 128 streams
// over 16384 shared and up to 1024 own keys: 122 us with the joining, where the
// own keys' 368 MB take 72 alone and the prefix 44, in a launch of its kind of
// blocks.  Side by side they gain nothing, and not for want of caches: 451 MB
// are fetched, as by both alone, and three of four reads of the prefix hit.  In
// the launch for both kinds the prefix takes 69 beside own blocks without a key.
//
// A key that a row does not see is never multiplied into it: its score is
// -infinity whatever the product gave, keys that no row of the tile sees are
// zeros in LDS, and where a causal tile that some rows see in part holds values
// that are not finite, those are kept out of the products (0 * infinity is
// NaN) and reach the rows that see them at the end.
#pragma once
#include "aq_attn.hpp"
#include "aq_types.hpp"

#include <climits>
#include <type_traits>

namespace aq_attn_impl {

using namespace aq_types;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A tile of KT keys by DP columns in LDS, rows of 16-byte pieces.  A piece's
// place in its row is XORed with a number of the row's, so that the lanes that
// read together meet different banks.
template <typename T, int DP>
struct shape {
    static constexpr bool kF32 = sizeof(typename T::raw) == 4;
    static constexpr int kPer = 16 / sizeof(typename T::raw);   // elements of a piece
    static constexpr int kPieces = DP / kPer;                   // of a row
    static constexpr int kRow = kPieces * 16;                   // bytes of a row
    static __device__ inline int swz_k(int key) { return kRow >= 256 ? key & 15 : (key >> 1) & 7; }
    static __device__ inline int swz_v(int key) {
        if (kF32) return kRow >= 256 ? ((key >> 2) & 1) * 8 : 0;
        return kRow >= 256 ? (key & 3) * 4 : ((key >> 1) & 1) * 4;
    }
};

__device__ inline f32x16 mma(f16, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ inline f32x16 mma(bf16, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ inline f32x16 mma(f32, float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// Each element of a word that is not finite replaced by zero.
template <typename T>
__device__ inline uint32_t finite_bits(uint32_t v) {
    if (std::is_same<T, f32>::value) return (v & 0x7F800000u) == 0x7F800000u ? 0u : v;
    constexpr uint32_t kLow = std::is_same<T, f16>::value ? 0x7C00u : 0x7F80u, kHigh = kLow << 16;
    return ((v & kLow) == kLow ? 0u : v & 0xFFFFu) | ((v & kHigh) == kHigh ? 0u : v & 0xFFFF0000u);
}

// The lanes whose reference asks for the exponents of far ones: it is far, or
// it is the first and may be -infinity by its product with c alone.
__device__ inline uint64_t far_rows(float score, float c) { return __ballot(is_far(score, c) || (c > 1.0f && score == -INFINITY)); }

// A piece of a row, elements at.. of D; zeros from D on, and where !use.
template <typename T>
__device__ inline u32x4 load_piece(const typename T::raw *row, int at, int D, bool use) {
    typedef u32x4 any __attribute__((aligned(1)));
    constexpr int kPer = 16 / sizeof(typename T::raw);
    u32x4 r = {0, 0, 0, 0};
    if (!use || at >= D) return r;
    if (at + kPer <= D) return *reinterpret_cast<const any *>(row + at);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (at + i < D) {
            if (sizeof(typename T::raw) == 4) r[i] = bits_of(row[at + i]);
            else r[i / 2] |= bits_of(row[at + i]) << (16 * (i % 2));
        }
    return r;
}

// Sixteen bytes of zeros, for the pieces past D and the keys that no row sees.
static __device__ const u32x4 kZeros = {0, 0, 0, 0};

// The rows of one wave's 32 columns and what they have gathered.
template <typename T, int DP>
struct row_state {
    using S = shape<T, DP>;
    static constexpr int kQ = S::kF32 ? DP / 8 : DP / 16;   // pieces of q in a lane
    u32x4 q[kQ];
    f32x16 o[DP / 32];
    float m, l;        // the row's; l holds the half's keys
    float score;       // m = c score, rounded
    int b, t, h;       // the lane's row
    bool used;         // it exists
    int see;           // own keys that it sees
    uint64_t far;      // far_rows() of the wave
};

template <typename T, int DP, bool DIRECT>
__device__ inline void open_rows(const args &a, int walk, int b0, int r, int hk, row_state<T, DP> &w) {
    using S = shape<T, DP>;
    const int half = (threadIdx.x & 63) >> 5;
    const int tok = r / a.G;
    w.b = b0 + tok / a.T;
    w.t = tok % a.T;
    w.h = hk * a.G + r % a.G;
    // (for a stream's own walk b0 is the stream, and rows past its T tokens are no rows)
    w.used = w.b < a.B && (walk == kPrefix || tok < a.T);
    int rows = a.T, keys = a.S;
    if (w.used) {
        if (a.q_len) rows = max(0, min(a.q_len[w.b], a.T));
        if (a.kv_len) keys = max(0, min(a.kv_len[w.b], a.S));
    }
    w.used = w.used && w.t < rows;
    w.see = !w.used ? 0 : a.causal ? max(0, keys - rows + w.t + 1) : keys;
    const typename T::raw *row = static_cast<const typename T::raw *>(a.q);
    if (w.used) row += w.b * a.sq.batch + w.t * a.sq.row + w.h * a.sq.head;
    if constexpr (DIRECT) {   // whole pieces: one load each, and all on their way together
#pragma unroll
        for (int i = 0; i < row_state<T, DP>::kQ; ++i) {
            typedef u32x4 any __attribute__((aligned(1)));
            const int at = (2 * i + half) * S::kPer;
            const bool use = w.used && at < a.D;
            const u32x4 v = *reinterpret_cast<const any *>(use ? row + at : reinterpret_cast<const typename T::raw *>(&kZeros));
            w.q[i] = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < row_state<T, DP>::kQ; ++i) w.q[i] = load_piece<T>(row, (2 * i + half) * S::kPer, a.D, w.used);
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) w.o[d][i] = 0.0f;
    w.m = w.score = -INFINITY;
    w.l = 0.0f;
    w.far = far_rows(w.score, a.c);
}

// Steps of a chain of products whose operands come from LDS: kAhead of them are
// on their way before the first is used.  The scheduling barriers keep it so;
// left alone, the compiler loads each next to its use, or all at once.  Tiles
// of 32 keys are left to it: there the registers hold a tile on its way, and
// what a ring takes more is spilled (64 streams over 1500 keys: 65 us, 61 so).
template <int NT> constexpr int kAheadSteps = NT > 1 ? 4 : 0;

// S^T for a tile of 32 NT keys: s[n] += K q.
template <typename T, int DP, int NT>
__device__ inline void add_scores(const unsigned char *lk, f32x16 (&s)[NT], const row_state<T, DP> &w) {
    using S = shape<T, DP>;
    constexpr int kQ = row_state<T, DP>::kQ, kSteps = NT * kQ, kAhead = kAheadSteps<NT>, kRing = kAhead + 1;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const auto piece = [&](int e) {
        const int key = 32 * (e % NT) + col, i = e / NT;
        return *reinterpret_cast<const u32x4 *>(lk + key * S::kRow + (((2 * i + half) ^ S::swz_k(key)) << 4));
    };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
    u32x4 ring[kRing];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) ring[e] = piece(e);
#pragma unroll
    for (int e = 0; e < kSteps; ++e) {
        if (e + kAhead < kSteps) ring[(e + kAhead) % kRing] = piece(e + kAhead);
        if (kAhead) __builtin_amdgcn_sched_barrier(0);
        const u32x4 k = ring[e % kRing];
        if constexpr (S::kF32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[e % NT] = mma(f32(), __uint_as_float(k[j]), __uint_as_float(w.q[e / NT][j]), s[e % NT]);
        } else {
            s[e % NT] = mma(T(), k, w.q[e / NT], s[e % NT]);
        }
    }
}

// o += P V, with p = 2^(c s - from): the sum of the lane's p comes back.  16-bit
// types: the exponentials of 16 keys are taken between the products of the 16
// before them.
template <typename T, int DP, int NT>
__device__ inline float add_values(const unsigned char *lv, f32x16 (&s)[NT], float c, float from, row_state<T, DP> &w) {
    using S = shape<T, DP>;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    constexpr int kD = DP / 32;
    float sum = 0.0f;
    const auto weigh = [&](int n, int i) {
        s[n][i] = __builtin_amdgcn_exp2f(__fmaf_rn(s[n][i], c, -from));
        sum += s[n][i];
    };
    if constexpr (S::kF32) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) weigh(n, i);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = 32 * n + 8 * (i >> 2) + (i & 3) + 4 * half;   // this half's
#pragma unroll
                for (int d = 0; d < kD; ++d) {
                    const int at = 32 * d + col;
                    const uint32_t v = *reinterpret_cast<const uint32_t *>(lv + key * S::kRow + (((at >> 2) ^ S::swz_v(key)) << 4) +
                                                                           (at & 3) * 4);
                    w.o[d] = mma(f32(), __uint_as_float(v), s[n][i], w.o[d]);
                }
                if (DP > 128) __builtin_amdgcn_sched_barrier(0);   // (or loads run so far ahead that registers spill)
            }
    } else {
        constexpr int kGroups = 2 * NT, kSteps = kGroups * kD, kAhead = kAheadSteps<NT>, kRing = kAhead + 1;
        const int sub = (lane >> 2) & 3;   // of the four keys that 16 lanes load for each other
        const auto values = [&](int e) {   // keys 16 (e / kD) + 4 half + 0..3, and 8 on, of column 32 (e % kD) + col
            const int key = 16 * (e / kD) + 4 * half + sub, piece = 4 * (e % kD) + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
            const unsigned char *at = lv + key * S::kRow + ((piece ^ S::swz_v(key)) << 4) + (lane & 1) * 8;
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * S::kRow)));
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        const auto packed = [&](int g) {
            typename T::raw p[8];
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 8; i += 2) T::store2(p + i, s[g / 2][8 * (g % 2) + i], s[g / 2][8 * (g % 2) + i + 1]);
            std::memcpy(&r, p, 16);
            return r;
        };
#pragma unroll
        for (int i = 0; i < 8; ++i) weigh(0, i);
        u32x4 ring[kRing], p = packed(0);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) ring[e] = values(e);
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
            const int g = e / kD, d = e % kD;
            if (e + kAhead < kSteps) ring[(e + kAhead) % kRing] = values(e + kAhead);
            if (kAhead) __builtin_amdgcn_sched_barrier(0);
            w.o[d] = mma(T(), ring[e % kRing], p, w.o[d]);
            if (g + 1 < kGroups) {
#pragma unroll
                for (int i = 8 * d / kD; i < 8 * (d + 1) / kD; ++i) weigh((g + 1) / 2, 8 * ((g + 1) % 2) + i);
                if (d == kD - 1) p = packed(g + 1);
            }
        }
    }
    return sum;
}

// The larger of this lane's value and lane ^ 32's.
__device__ inline float both_halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// One tile of 32 NT keys from LDS.  vis: bit j is set where this lane's row
// sees key j of each 32; all: every lane sees every key.
template <typename T, int DP, int NT>
__device__ inline void add_tile(const unsigned char *lk, const unsigned char *lv, const uint32_t (&vis)[NT], bool all,
                                float c, row_state<T, DP> &w) {
    constexpr int kShift = std::is_same<T, f16>::value ? 10 : 0;   // p is 2^kShift times the weight
    constexpr float kSlack = 5.0f;
    const int half = (threadIdx.x & 63) >> 5;
    f32x16 s[NT];
    add_scores<T, DP, NT>(lk, s, w);
    // Of a SIMD's two waves the one with exponentials and products to mix goes
    // first, the one with products alone fills what is left (8 x 4096 rows over
    // 1500 keys: 462 -> 449 us, 16 x 512 over 8192 + 512: 598 -> 573).
    if (NT > 1) __builtin_amdgcn_s_setprio(1);
    if (!all) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t v = vis[n] >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = v >> (8 * (i >> 2) + (i & 3)) & 1u ? s[n][i] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
    top = both_halves_max(top);
    // The sums' reference moves only when a row's maximum has outgrown it by
    // 2^kSlack: until then the weights are that much above 1 at most.
    // (Row by row: a row's result does not depend on its neighbours'.)
    bool grown = top * c > w.m + kSlack;
    if ((__ballot(grown) | w.far) != 0) {
        if (is_far(w.score, c) || w.score == -INFINITY) grown = (top - w.score) * c > kSlack;
        const float keep = grown ? weight_of(w.score, top, c) : 1.0f;
        w.score = grown ? top : w.score;
        w.m = grown ? top * c : w.m;
        w.l *= keep;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) w.o[d] *= keep;
        w.far = far_rows(w.score, c);
    }
    float from = (w.m == -INFINITY ? 0.0f : w.m) - kShift;
    if (__builtin_expect(w.far != 0, 0)) {   // out of line; the exponents themselves, by distance where the row's reference is far
        const bool far = is_far(w.score, c);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = far ? __fmaf_rn(s[n][i] - w.score, c, kShift) : __fmaf_rn(s[n][i], c, -from);
        c = 1.0f;
        from = 0.0f;
    }
    w.l += add_values<T, DP, NT>(lv, s, c, from, w);
    if (NT > 1) __builtin_amdgcn_s_setprio(0);
}

// The keys that a walk meets one after the other: the prefix's tiles, then the
// stream's own.  Everything here is the same for all lanes that share a tile.
template <typename T>
struct key_walk {
    const typename T::raw *pk, *pv, *k, *v;
    const uint8_t *mask;
    int prefix_tiles, P, keys, own;   // keys: of the stream (for the staging); own: that the rows can see
    int64_t pk_row, pv_row, k_row, v_row;
};

template <typename T, int KT>
__device__ inline int open_walk(const args &a, int walk, int b, int hk, int most, key_walk<T> &w) {
    using E = typename T::raw;
    w.P = walk & kPrefix ? a.P : 0;
    w.prefix_tiles = (w.P + KT - 1) / KT;
    w.own = walk & kOwn ? most : 0;
    w.pk = static_cast<const E *>(a.pk) + hk * a.spk.head;
    w.pv = static_cast<const E *>(a.pv) + hk * a.spv.head;
    w.k = static_cast<const E *>(a.k) + b * a.sk.batch + hk * a.sk.head;
    w.v = static_cast<const E *>(a.v) + b * a.sv.batch + hk * a.sv.head;
    w.pk_row = a.spk.row;
    w.pv_row = a.spv.row;
    w.k_row = a.sk.row;
    w.v_row = a.sv.row;
    w.mask = a.mask ? a.mask + b * a.mask_ld : nullptr;
    return w.prefix_tiles + (w.own + KT - 1) / KT;
}

// Brings a tile's K and V to LDS.  DIRECT (rows that start and end at 16
// bytes): straight from memory, still on their way when load() returns; each
// wave's 64 pieces land next to each other, so the piece of a place is the one
// that the swizzle puts there.  Otherwise through registers.
template <typename T, int DP, int KT, int THREADS, bool DIRECT>
struct stager {
    using S = shape<T, DP>;
    using E = typename T::raw;
    static constexpr int kEach = KT * S::kPieces / THREADS;

    static __device__ inline void piece(const void *from, unsigned char *to) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                         (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    }

    // The keys of the tile that any row may see come back as bits.  wave: of
    // the block's, the same for all its lanes (0 where a wave has the tile to
    // itself).
    static __device__ inline uint64_t load(const args &a, const key_walk<T> &w, int tile, unsigned char *lk, unsigned char *lv,
                                           int wave) {
        const bool pre = tile < w.prefix_tiles;
        const int j0 = (pre ? tile : tile - w.prefix_tiles) * KT, n = (pre ? w.P : w.own) - j0;
        uint64_t bits = n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1;
        const int lane = threadIdx.x & 63, thread = wave * 64 + lane;
        if (!pre && w.mask) bits &= __ballot(lane < n && w.mask[j0 + min(lane, n - 1)] != 0);
        const int64_t kr = pre ? w.pk_row : w.k_row, vr = pre ? w.pv_row : w.v_row;
        const E *kp = (pre ? w.pk : w.k) + j0 * kr, *vp = (pre ? w.pv : w.v) + j0 * vr;
        if constexpr (DIRECT) {
            unsigned char *const k0 = lk + wave * 1024, *const v0 = lv + wave * 1024;
            constexpr uint64_t kAll = KT == 64 ? ~uint64_t{0} : (uint64_t{1} << (KT % 64)) - 1;
            // Offsets within a tile fit 32 bits (the host saw to it), so a
            // piece's address is one multiplication.
            const uint32_t kb = static_cast<uint32_t>(kr * sizeof(E)), vb = static_cast<uint32_t>(vr * sizeof(E));
            if ((bits & kAll) == kAll && a.D == DP) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const uint32_t at = i * THREADS + thread, key = at / S::kPieces, place = at % S::kPieces;
                    piece(reinterpret_cast<const char *>(kp) + (key * kb + ((place ^ S::swz_k(key)) << 4)), k0 + i * THREADS * 16);
                    piece(reinterpret_cast<const char *>(vp) + (key * vb + ((place ^ S::swz_v(key)) << 4)), v0 + i * THREADS * 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const uint32_t at = i * THREADS + thread, key = at / S::kPieces, place = at % S::kPieces;
                    const uint32_t pk = place ^ S::swz_k(key), pv = place ^ S::swz_v(key), end = a.D / S::kPer;
                    const bool use = bits >> key & 1;
                    const void *none = &kZeros;
                    piece(use && pk < end ? reinterpret_cast<const char *>(kp) + (key * kb + (pk << 4)) : none, k0 + i * THREADS * 16);
                    piece(use && pv < end ? reinterpret_cast<const char *>(vp) + (key * vb + (pv << 4)) : none, v0 + i * THREADS * 16);
                }
            }
        } else {
#pragma unroll 4
            for (int i = 0; i < kEach; ++i) {
                const int at = i * THREADS + thread, key = at / S::kPieces, piece = at % S::kPieces;
                const bool use = bits >> key & 1;
                const u32x4 k = load_piece<T>(kp + key * kr, piece * S::kPer, a.D, use);
                const u32x4 v = load_piece<T>(vp + key * vr, piece * S::kPer, a.D, use);
                *reinterpret_cast<u32x4 *>(lk + key * S::kRow + ((piece ^ S::swz_k(key)) << 4)) = k;
                *reinterpret_cast<u32x4 *>(lv + key * S::kRow + ((piece ^ S::swz_v(key)) << 4)) = v;
            }
        }
        return bits;
    }
};

// The same through registers, for a tile that one wave has to itself: the next
// tile's pieces are on their way in registers while one is used.  Such keys are
// read once (in fp32 up to three times, by products far slower than memory), so
// they are the first to leave the caches: a prefix stays there
// (a token of 128 streams over 16384 + 1024 keys: 137 us with plain loads, 130
// so; of 64 streams over 1500 keys, 61 and 55).
template <typename T, int DP, int KT, bool DIRECT>
struct carrier {
    using S = shape<T, DP>;
    using E = typename T::raw;
    static constexpr int kEach = KT * S::kPieces / 64;
    u32x4 k[kEach + !kEach], v[kEach + !kEach];
    uint64_t bits;

    __device__ inline void load(const args &a, const key_walk<T> &w, int tile, int lane) {
        const bool pre = tile < w.prefix_tiles;
        const int j0 = (pre ? tile : tile - w.prefix_tiles) * KT, n = (pre ? w.P : w.own) - j0;
        bits = n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1;
        if (!pre && w.mask) bits &= __ballot(lane < n && w.mask[j0 + min(lane, n - 1)] != 0);
        const int64_t kr = pre ? w.pk_row : w.k_row, vr = pre ? w.pv_row : w.v_row;
        const E *kp = (pre ? w.pk : w.k) + j0 * kr, *vp = (pre ? w.pv : w.v) + j0 * vr;
        if constexpr (DIRECT) {   // whole pieces: a load each, from zeros where there is none
            constexpr int kStep = 64 / S::kPieces;   // keys from one of a lane's pieces to the next
            const int key = lane / S::kPieces, piece = lane % S::kPieces * S::kPer;
            const E *kg = kp + key * kr + piece, *vg = vp + key * vr + piece;
            constexpr uint64_t kAll = (uint64_t{1} << (KT % 64)) - 1;
            if ((bits & kAll) == kAll && a.D == DP) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kg + i * kStep * kr));
                    v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vg + i * kStep * vr));
                }
            } else {
                const E *const none = reinterpret_cast<const E *>(&kZeros);
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const bool in = (bits >> (key + i * kStep) & 1) != 0 && piece < a.D;
                    k[i] = *reinterpret_cast<const u32x4 *>(in ? kg + i * kStep * kr : none);
                    v[i] = *reinterpret_cast<const u32x4 *>(in ? vg + i * kStep * vr : none);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int at = i * 64 + lane, key = at / S::kPieces, piece = at % S::kPieces * S::kPer;
                const bool use = bits >> key & 1;
                k[i] = load_piece<T>(kp + key * kr, piece, a.D, use);
                v[i] = load_piece<T>(vp + key * vr, piece, a.D, use);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    __device__ inline void store(unsigned char *lk, unsigned char *lv, int lane) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = i * 64 + lane, key = at / S::kPieces, piece = at % S::kPieces;
            *reinterpret_cast<u32x4 *>(lk + key * S::kRow + ((piece ^ S::swz_k(key)) << 4)) = k[i];
            *reinterpret_cast<u32x4 *>(lv + key * S::kRow + ((piece ^ S::swz_v(key)) << 4)) = v[i];
        }
    }
};

// What this wave sent to LDS has landed, and what it read from there has come.
__device__ inline void landed() { __builtin_amdgcn_s_waitcnt(0x0070); }   // vmcnt(0) lgkmcnt(0)

// A causal tile that not all rows of the block see, its V in LDS: values that
// are not finite become zeros there, so that they do not reach the rows that
// do not see them (0 * infinity is NaN); add_odd() gives them to the others.
// Each of THREADS threads looks at its part; whether any was found there.
template <typename T, int DP, int KT, int THREADS>
__device__ inline bool hide_odd(unsigned char *lv, int thread) {
    using S = shape<T, DP>;
    bool odd = false;
#pragma unroll 1
    for (int n = 0; n < KT * S::kPieces / THREADS; ++n) {
        const int i = n * THREADS + thread;
        u32x4 v = reinterpret_cast<const u32x4 *>(lv)[i];
        bool any = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t f = finite_bits<T>(v[j]);
            any = any || f != v[j];
            v[j] = f;
        }
        if (any) reinterpret_cast<u32x4 *>(lv)[i] = v;
        odd = odd || any;
    }
    return odd;
}

// The values that hide_odd() took out of own keys, to the rows that see them;
// first and end count from the walk's start, in tiles of `tile` keys.  A weight
// is above 0 and its product with such a value is that value again, which no
// finite sum changes: it is added as it is.
template <typename T, int DP>
__device__ inline void add_odd(const args &a, const key_walk<T> &walk, int first, int end, int tile, row_state<T, DP> &w) {
    first -= walk.prefix_tiles * tile;
    end = min(end - walk.prefix_tiles * tile, walk.own);   // no key past those that a row sees is read
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll 1
    for (int key = first; key < end; ++key) {
        int D = key < w.see ? a.D : 0;
        asm("" : "+v"(D));   // (compared anew for each key: 16 DP / 32 comparisons kept over the loop fill the scalar registers)
        const typename T::raw *row = walk.v + key * walk.v_row;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int at = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
                const float value = T::load(row[max(min(at, D - 1), 0)]);
                w.o[d][i] += at < D && !(__builtin_fabsf(value) < INFINITY) ? value : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// A staged tile for this wave's rows.
template <typename T, int DP, int NT>
__device__ inline void take_tile(const args &a, const key_walk<T> &walk, int tile, uint64_t bits, const unsigned char *lk,
                                 const unsigned char *lv, row_state<T, DP> &w) {
    constexpr int KT = 32 * NT;
    const bool pre = tile < walk.prefix_tiles;
    uint32_t vis[NT];
    bool mine = true;
    // Keys of the tile that the row sees, masks apart.  (A column without a row may see any.)
    const int n = pre || !w.used ? KT : w.see - (tile - walk.prefix_tiles) * KT;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int c = min(max(n - 32 * i, 0), 32);
        vis[i] = (c == 32 ? ~0u : (1u << c) - 1u) & static_cast<uint32_t>(bits >> (32 * i));
        mine = mine && vis[i] == ~0u;
    }
    add_tile<T, DP, NT>(lk, lv, vis, __ballot(mine) == ~uint64_t{0}, a.c, w);
}

// Where the lane's row starts, in `out` or among the parts; -1 if it has none.
template <typename T, int DP>
__device__ inline int64_t row_start(const args &a, int part, const row_state<T, DP> &w) {
    if (!w.used) return -1;
    if (!a.sums) return w.b * a.so.batch + w.t * a.so.row + w.h * a.so.head;
    return (part * a.rows + (static_cast<int64_t>(w.b) * a.T + w.t) * a.H + w.h) * a.D;
}

// A part's reference and weight, by one lane of the row.
__device__ inline void put_ml(const args &a, int64_t start, float m, float l) {
    if (start < 0 || !a.sums) return;
    a.ml[start / a.D * 2] = m;
    a.ml[start / a.D * 2 + 1] = l;
}

// What a row's sums are multiplied by: a part's stay as they are; no key at all gives 0.
__device__ inline float share_of(const args &a, float l) { return a.sums ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l; }

// Columns c..c + 3 of a row.
template <typename T, bool DIRECT>
__device__ inline void put4(const args &a, int64_t start, int c, f32x4 v) {
    if (start < 0 || c >= a.D) return;
    if (a.sums) {
        float *to = a.sums + start + c;
        if (DIRECT || c + 4 <= a.D) std::memcpy(to, &v, 16);   // (DIRECT: D is a multiple of 4)
        else
            for (int j = 0; j < a.D - c; ++j) to[j] = v[j];
        return;
    }
    typename T::raw *to = static_cast<typename T::raw *>(a.out) + start + c, y[4];
#pragma unroll
    for (int j = 0; j < 4; j += 2) T::store2(y + j, v[j], v[j + 1]);
    if (DIRECT || c + 4 <= a.D) std::memcpy(to, y, sizeof(y));
    else
        for (int j = 0; j < a.D - c; ++j) to[j] = y[j];
}

// The wave's rows, or their part of them, to memory.  l is whole here.  A lane
// holds a row's columns four by four; they go through LDS (`lds`, BYTES of the
// wave's own), so that lanes next to each other write next to each other.
template <typename T, int DP, int BYTES, bool DIRECT>
__device__ inline void close_rows(const args &a, int part, row_state<T, DP> &w, unsigned char *lds) {
    constexpr int kTurns = 32 * DP * 4 > BYTES ? 2 : 1, kCols = DP / kTurns, kPieces = kCols / 4;
    static_assert(32 * kCols * 4 <= BYTES, "the columns of a turn fit");
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int64_t start = row_start<T, DP>(a, part, w);
    if (half == 0) put_ml(a, start, w.score, w.l);
    const float by = share_of(a, w.l);
#pragma unroll
    for (int turn = 0; turn < kTurns; ++turn) {
#pragma unroll
        for (int d = 0; d < kCols / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = w.o[turn * (kCols / 32) + d][4 * g + i] * by;
                const int piece = 8 * d + 2 * g + half;
                *reinterpret_cast<f32x4 *>(lds + (col * kPieces + (piece ^ (col & 15))) * 16) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
        for (int i = 0; i < 32 * kPieces / 64; ++i) {
            const int at = i * 64 + lane, r = at / kPieces, piece = at % kPieces;
            const f32x4 v = *reinterpret_cast<const f32x4 *>(lds + (r * kPieces + (piece ^ (r & 15))) * 16);
            put4<T, DIRECT>(a, __shfl(start, r), turn * kCols + piece * 4, v);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// The most own keys that any row of the block (or wave) sees.
__device__ inline int most_of(int see) {
#pragma unroll
    for (int d = 32; d; d >>= 1) see = max(see, __shfl_xor(see, d));
    return see;
}

// The fewest own keys that any of the rows sees.
__device__ inline int least_of(int see) {
#pragma unroll
    for (int d = 32; d; d >>= 1) see = min(see, __shfl_xor(see, d));
    return see;
}

// Where a block stands in its job.  Row tiles are next to each other, since
// they read the same keys; the key head is outermost, so that blocks near each
// other share a prefix.
struct place {
    int hk, b, tile, split;   // b: 0 for the prefix alone
};

__device__ inline place place_of(const args &a, const job &j, int at) {
    place p;
    p.tile = at % j.tiles;
    at /= j.tiles;
    p.split = at % j.splits;
    at /= j.splits;
    const int streams = j.walk == kPrefix ? 1 : a.B;
    p.b = at % streams;
    p.hk = at / streams;
    return p;
}

// Many rows: 32 a wave, 128 a block, which brings each tile to LDS once, into
// one of two places while the other is used.
template <typename T, int DP, int NT, bool DIRECT>
__device__ inline void rows_body(const args &a, const job &j, const place &at, unsigned char *lds) {
    using S = shape<T, DP>;
    constexpr int KT = 32 * NT, kTile = KT * S::kRow;
    using stage = stager<T, DP, KT, 256, DIRECT>;
    __shared__ int see[2][4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    row_state<T, DP> w;
    open_rows<T, DP, DIRECT>(a, j.walk, at.b, at.tile * 128 + wave * 32 + (lane & 31), at.hk, w);
    const int high = most_of(w.see), low = least_of(w.used ? w.see : INT_MAX);
    if (lane == 0) {
        see[0][wave] = high;
        see[1][wave] = low;
    }
    if (__syncthreads_or(w.used) == 0) return;
    key_walk<T> walk;
    const int most = __builtin_amdgcn_readfirstlane(max(max(see[0][0], see[0][1]), max(see[0][2], see[0][3])));
    const int least = __builtin_amdgcn_readfirstlane(min(min(see[1][0], see[1][1]), min(see[1][2], see[1][3])));
    const int tiles = open_walk<T, KT>(a, j.walk, at.b, at.hk, most, walk);
    const int mixed = least < most ? walk.prefix_tiles + least / KT : INT_MAX;   // from here on tiles that not all rows see
    const int per = (tiles + j.splits - 1) / j.splits, first = at.split * per, end = min(tiles, first + per);
    uint64_t bits = 0;
    bool odd = false;
    if (first < end) bits = stage::load(a, walk, first, lds, lds + kTile, wave);
#pragma unroll 1
    for (int tile = first; tile < end; ++tile) {
        unsigned char *const now = lds + ((tile - first) & 1) * 2 * kTile, *const then = lds + ((tile - first + 1) & 1) * 2 * kTile;
        landed();
        __syncthreads();   // the tile is there, and all waves are done with the one before
        const uint64_t use = bits;
        if (tile + 1 < end) bits = stage::load(a, walk, tile + 1, then, then + kTile, wave);
        if (tile >= mixed) odd |= __syncthreads_or(hide_odd<T, DP, KT, 256>(now + kTile, threadIdx.x)) != 0;
        take_tile<T, DP, NT>(a, walk, tile, use, now, now + kTile, w);
    }
    if (odd) add_odd(a, walk, max(first, mixed) * KT, end * KT, KT, w);
    w.l += __shfl_xor(w.l, 32);
    __syncthreads();   // no tile is read any more
    close_rows<T, DP, kTile, DIRECT>(a, j.part + at.split, w, lds + wave * kTile);
}

// Few rows (fp32: up to 96 of a stream): 32 a block; each of its first WAVES
// waves takes every WAVES-th tile, with LDS of its own, and the waves' sums are
// joined in LDS, in the waves' order.
template <typename T, int DP, int WAVES, bool DIRECT>
__device__ inline void keys_body(const args &a, const job &j, const place &at, unsigned char *lds) {
    using S = shape<T, DP>;
    constexpr int KT = 32, kTile = KT * S::kRow;
    __shared__ float ml[WAVES][2][32];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    unsigned char *const own = lds + wave * 2 * kTile;
    row_state<T, DP> w;
    open_rows<T, DP, DIRECT>(a, j.walk, at.b, at.tile * 32 + (lane & 31), at.hk, w);
    if (__ballot(w.used) == 0) return;   // the same for all waves
    key_walk<T> walk;
    const int most = __builtin_amdgcn_readfirstlane(most_of(w.see));
    const int least = __builtin_amdgcn_readfirstlane(least_of(w.used ? w.see : INT_MAX));
    const int tiles = open_walk<T, KT>(a, j.walk, at.b, at.hk, most, walk);
    const int mixed = least < most ? walk.prefix_tiles + least / KT : INT_MAX;
    bool odd = false;
    const int per = (tiles + j.splits - 1) / j.splits, first = at.split * per;
    const int end = wave < WAVES ? min(tiles, first + per) : 0;
    constexpr bool kAhead = S::kRow <= 512 && DP <= 128;   // registers hold a tile on its way
    carrier<T, DP, kAhead ? KT : 0, DIRECT> next;
    int tile = first + wave;
    if (kAhead && tile < end) next.load(a, walk, tile, lane);
#pragma unroll 1
    for (; tile < end; tile += WAVES) {
        uint64_t bits;
        if constexpr (kAhead) {
            next.store(own, own + kTile, lane);
            bits = next.bits;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (tile + WAVES < end) next.load(a, walk, tile + WAVES, lane);
        } else {
            landed();   // the last tile's reads, before this one takes the place
            bits = stager<T, DP, KT, 64, DIRECT>::load(a, walk, tile, own, own + kTile, 0);
            landed();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (tile >= mixed && __ballot(hide_odd<T, DP, KT, 64>(own + kTile, lane)) != 0) {
            odd = true;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        take_tile<T, DP, 1>(a, walk, tile, bits, own, own + kTile, w);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (odd)   // of this wave's tiles
        for (tile = first + wave; tile < end; tile += WAVES)
            if (tile >= mixed) add_odd(a, walk, tile * KT, (tile + 1) * KT, KT, w);
    w.l += __shfl_xor(w.l, 32);
    if (wave < WAVES && lane < 32) {
        ml[wave][0][lane] = w.score;
        ml[wave][1][lane] = w.l;
    }
    __syncthreads();   // (the tiles are not used any more either)
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, ml[i][0][lane & 31]);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) l = __fmaf_rn(ml[i][1][lane & 31], weight_of(ml[i][0][lane & 31], m, a.c), l);
    const float keep = weight_of(w.score, m, a.c);
    f32x16 *const red = reinterpret_cast<f32x16 *>(lds);   // [WAVES][DP / 32][64]
    if (wave < WAVES) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) red[(wave * (DP / 32) + d) * 64 + lane] = w.o[d] * keep;
    }
    __syncthreads();
    // Each wave joins and writes a share of the columns.
    const int64_t start = row_start<T, DP>(a, j.part + at.split, w);
    const int half = lane >> 5;
    if (wave == 0 && half == 0) put_ml(a, start, m, l);
    const float by = share_of(a, l);
#pragma unroll 1
    for (int d = wave; d < DP / 32; d += 4) {
        f32x16 o = red[d * 64 + lane];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) o += red[(i * (DP / 32) + d) * 64 + lane];
#pragma unroll
        for (int g = 0; g < 4; ++g)
            put4<T, DIRECT>(a, start, 32 * d + 8 * g + 4 * half, f32x4{o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]} * by);
    }
}

// The blocks of one job, or of two at once, evenly mixed: a prefix's products
// and the streams' own keys, which wait for memory, share the compute units.
// KINDS: the kinds of blocks that the launch has (1: many rows, 2: few); a kind
// alone has its registers to itself.
template <typename T, int DP, int NT, int WAVES, bool DIRECT, int KINDS>
__global__ __launch_bounds__(256, sizeof(typename T::raw) * DP <= 256 ? 2 : 1) void attn_kernel(args a) {
    extern __shared__ __align__(16) unsigned char lds[];
    // Blocks are dealt to the eight dies in turn; each die gets a run of
    // neighbours of either job, which share keys, and so its cache serves
    // them.  Within a die the two jobs alternate while both last.
    const int die = blockIdx.x % 8, n = blockIdx.x / 8;
    const int n0 = a.jobs[0].blocks, n1 = a.jobs[1].blocks, more0 = n0 % 8, more1 = n1 % 8;
    const int mine0 = n0 / 8 + (die < more0), mine1 = n1 / 8 + ((die + 8 - more0) % 8 < more1);
    int from1 = 0;   // the second job's blocks of the dies before: its remainder goes to the dies that the first's left out
    for (int d = 0; d < die; ++d) from1 += n1 / 8 + ((d + 8 - more0) % 8 < more1);
    const int both = 2 * min(mine0, mine1);
    const bool one = n < both ? n % 2 == 0 : mine0 > mine1;
    const int nth = n < both ? n / 2 : n - both / 2;
    const job &j = one ? a.jobs[0] : a.jobs[1];
    const int at = one ? n0 / 8 * die + min(die, more0) + nth : from1 + nth;
    const place p = place_of(a, j, at);
    if constexpr ((KINDS & 2) != 0) {
        if (KINDS == 2 || !j.many) {
            keys_body<T, DP, WAVES, DIRECT>(a, j, p, lds);
            return;
        }
    }
    if constexpr ((KINDS & 1) != 0) rows_body<T, DP, NT, DIRECT>(a, j, p, lds);
}

template <typename T, int DP, int NT, int WAVES>
aq_status run(aq_ctx *ctx, const args &a) {
    constexpr uint32_t kRows = 4 * 32 * NT * shape<T, DP>::kRow, kKeys = WAVES * 2 * 32 * shape<T, DP>::kRow;
    static_assert(kKeys >= WAVES * 32 * DP * 4, "the waves' sums fit where the tiles were");
    uint32_t lds = 0;
    int64_t blocks = 0;
    int kinds = 0;
    for (const job &j : a.jobs) {
        if (!j.blocks) continue;
        kinds |= j.many ? 1 : 2;
        const uint32_t need = j.many ? kRows : kKeys;
        if (need > lds) lds = need;
        blocks += j.blocks;
    }
    auto kernel = a.direct ? attn_kernel<T, DP, NT, WAVES, true, 1> : attn_kernel<T, DP, NT, WAVES, false, 1>;
    if constexpr (WAVES > 0) {
        if (kinds == 2) kernel = a.direct ? attn_kernel<T, DP, NT, WAVES, true, 2> : attn_kernel<T, DP, NT, WAVES, false, 2>;
        if (kinds == 3) kernel = a.direct ? attn_kernel<T, DP, NT, WAVES, true, 3> : attn_kernel<T, DP, NT, WAVES, false, 3>;
    }
    aq_status st = aq_launch_lds(ctx, reinterpret_cast<const void *>(kernel), lds, "attention");
    if (st != AQ_OK) return st;
    aq_launch_timed(ctx, true, kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), lds, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}

template <typename T>
aq_status launch(aq_ctx *ctx, const args &a) {
    constexpr bool kWide = sizeof(typename T::raw) == 4;
    if (a.D <= 64) return run<T, 64, kWide ? 1 : 2, 4>(ctx, a);
    if (a.D <= 128) return run<T, 128, kWide ? 1 : 2, 4>(ctx, a);
    return run<T, 256, 1, kWide ? 0 : 4>(ctx, a);   // (no registers for an fp32 tile of that width on its way)
}

}  // namespace aq_attn_impl
