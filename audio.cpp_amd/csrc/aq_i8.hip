// Products with 8-bit whole-number weights, a scale for each row of W and
// each row of x (aq_i8_*).
//
// Layout.  A tile is 16 rows of W, a k-block 64 columns: 1 KB, 16 bytes a
// lane, in the order of the 16x16x64 matrix instruction's operand: lane l
// holds row l % 16, columns 16 (l / 16) ..+15 of the k-block.  Rows and
// columns past the end are zeros, so x may hold anything there.  A packed x
// has the same layout, by 16 rows of x.
//
// What bounds it.  Few rows of x, the weights' way from memory: 64 x 8192 x
// 16384, 134 MB, 26 us (5.1 TB/s; 36 with bringing bf16 rows to 8 bits).  128
// rows of that size take 44 us: W is read once for 64 of them.  Many
// rows, the matrix instructions: 16384 x 8192 x 8192 in 1.04 ms, 2.1 POP/s, as
// fast as the library's product of whole numbers (bf16 rows 1.17 ms: bringing
// them to 8 bits reads them twice, at half the rate of a copy).  One row of 1024 x 1536: 3 us
// in the kernel, latency of the loads, of the join and of the launch.
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
//
// 16 rows and a k-block are 1 KB, as a tile of W.  Rows past M hold anything:
// they are columns of the product that are not written.

// I8 rows are moved: 16 rows by 256 columns a block.
__global__ __launch_bounds__(256) void i8_pack_kernel(const uint8_t *x, int64_t x_ld, int M, int K, int kblocks, i32x4 *to) {
    const int r = threadIdx.x & 15, c = static_cast<int>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    const int64_t m = static_cast<int64_t>(blockIdx.y) * 16 + r;
    if (m >= M || c >= kblocks * 4) return;
    const uint8_t *row = x + m * x_ld;
    to[(static_cast<int64_t>(blockIdx.y) * kblocks + (c >> 2)) * 64 + (c & 3) * 16 + r] =
        16 * c + 16 <= K ? load16(row + 16 * c) : load_tail(row, 16 * c, K);
}

// A floating row is brought to 8 bits: its largest magnitude, then q = the
// whole number nearest to x * 127 / max, ties to even.  Twice the quotient is
// formed in 64 bits with an error below 2^-44; where it is not a whole number
// it is at least 2^-32 off one (x and max have 24 bits, and x is near or above
// max / 254 where it matters), so within 2^-40 it is one, and every q is exact.
//
// ROWS rows a block of ROWS * 64 * WAVES threads.  Many rows: 16 a block, one
// wave each, so that the 16 rows' pieces of a cache line are written together;
// few: one a block, whose time is the call's (64 rows of 8192: 22 us with 16
// rows a block).
template <typename T, int ROWS, int WAVES>
__global__ __launch_bounds__(ROWS * WAVES * 64) void i8_quantize_kernel(const typename T::raw *x, int64_t x_ld, int M, int K,
                                                                        int kblocks, i32x4 *to, float *scale) {
    constexpr int kThreads = WAVES * 64;
    const int thread = threadIdx.x % kThreads;
    const int64_t m = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / kThreads;
    uint32_t most = 0;   // magnitudes compare like their bits, with infinity and NaN above all others
    const typename T::raw *row = x + (m < M ? m : M - 1) * x_ld;
#pragma unroll 4
    for (int c = thread; 8 * c < K; c += kThreads) {
        float v[8];
        load8<T>(row, 8 * c, K, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
    if constexpr (WAVES > 1) {
        __shared__ uint32_t part[WAVES];
        static_assert(ROWS == 1, "one row's waves share it");
        if ((thread & 63) == 0) part[thread >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) most = max(most, part[i]);
    }
    if (m >= M) return;
    const bool finite = most < 0x7F800000u;
    const double top = static_cast<double>(__uint_as_float(most)), per = finite && most ? 254.0 / top : 0.0;
    i32x4 *const out = to + m / 16 * kblocks * 64 + m % 16;
    for (int c = thread; c < kblocks * 4; c += kThreads) {
        uint32_t w[4] = {};
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
        out[(c >> 2) * 64 + (c & 3) * 16] =
            i32x4{static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3])};
    }
    if (thread == 0) scale[m] = finite ? static_cast<float>(top / 127.0) : __uint_as_float(0x7FC00000u);
}

// ---- the product ---------------------------------------------------------------

// What the four columns from n on are scaled with; columns past the end repeat
// the last.  wide: a sum (up to 2^31) times one of the scales may pass fp32's end.
struct columns {
    float scale[4], bias[4];
    bool wide;
};

constexpr float kWideScale = 0x1p96f;

__device__ inline columns columns_of(const args &a, int n) {
    columns v;
    v.wide = false;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int at = min(n + c, a.N - 1);
        v.scale[c] = a.scale[at];
        v.bias[c] = a.bias ? a.bias[at] : 0.0f;
        v.wide = v.wide || __builtin_fabsf(v.scale[c]) > kWideScale;
    }
    return v;
}

// Four columns n.. of row m from their sums.
__device__ inline void store4(const args &a, int m, int n, i32x4 sum, const columns &v, float xs) {
    if (m >= a.M || n >= a.N) return;
    const int most = min(4, a.N - n);
    float o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = static_cast<float>(sum[c]) * v.scale[c] * xs;   // (the scales' product alone may be subnormal)
    if (v.wide) {   // such a scale comes last: beyond fp32 before it is beyond after it
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (__builtin_fabsf(v.scale[c]) > kWideScale) o[c] = static_cast<float>(sum[c]) * xs * v.scale[c];
    }
    if (a.bias) {
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += v.bias[c];
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
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[(wave * RT * MT + r * MT + t) * 64 + lane] = sum[r][t];
    __syncthreads();
    for (int i = wave; i < RT * MT; i += waves) {
        i32x4 v = red[i * 64 + lane];
        for (int k = 1; k < waves; ++k) v += red[(k * RT * MT + i) * 64 + lane];
        const int m = m0 + 16 * (i % MT) + col, n = (tile0 + i / MT) * 16 + 4 * quad;
        store4(a, m, n, v, columns_of(a, n), a.x_scale[min(m, a.M - 1)]);
    }
}

// Many rows: a block of eight waves takes 32 RT rows of W by 64 MT rows of x,
// each wave RT tiles by MT.  The k-blocks come to LDS straight from memory, in
// operand order, kStages places in turn: while one is used the next two are
// there or on their way, and one barrier per k-block keeps the waves together.
// x is packed, or rows that start and end at 16 bytes, whose pieces past K read
// the row's start instead (W is 0 there).
constexpr int kStages = 4;

template <bool PACKED, int RT, int MT>
__global__ __launch_bounds__(512, 2) void i8_gemm_kernel(args a) {
    constexpr int kW = 2 * RT, kX = 4 * MT, kStage = (kW + kX) * 1024, kPieces = (kW + kX) / 8;   // KB of a k-block; of a wave
    static_assert((kW + kX) % 8 == 0, "every wave brings as much");
    extern __shared__ __align__(16) uint8_t lds[];   // [kStages][W tiles, x tiles]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    // Blocks are dealt to the eight dies in turn; each die gets a run of
    // neighbours in bands of 8 tiles of rows of x, so that its cache serves both sides.
    const int total = gridDim.x, die = blockIdx.x % 8;
    const int at = die * (total / 8) + min(die, total % 8) + blockIdx.x / 8;
    const int across = (a.tiles + kW - 1) / kW, down = (a.M + 16 * kX - 1) / (16 * kX);
    const int band = at / (8 * across), high = min(8, down - band * 8), in = at - band * 8 * across;
    const int tile0 = in / high * kW, m0 = (band * 8 + in % high) * 16 * kX;
    const int wn = wave & 1, wm = wave >> 1;   // the wave's place in the block

    const uint8_t *from[kPieces];   // the wave's pieces of a k-block, this lane's 16 bytes
    bool is_x[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int p = i * 8 + wave;   // of W's tiles, then of x's
        is_x[i] = p >= kW;
        if (!is_x[i]) {
            from[i] = a.w + (static_cast<int64_t>(min(tile0 + p, a.tiles - 1)) * a.kblocks * 64 + lane) * 16;
        } else if (PACKED) {
            from[i] = a.x + (static_cast<int64_t>(min(m0 / 16 + p - kW, (a.M - 1) / 16)) * a.kblocks * 64 + lane) * 16;
        } else {
            from[i] = a.x + min(m0 + 16 * (p - kW) + col, a.M - 1) * a.x_ld;
        }
    }
    const auto stage = [&](int kb, int place) {
        kb = min(kb, a.kblocks - 1);   // past the end: the last again, into a place that nobody reads
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint8_t *g;
            if (PACKED || !is_x[i]) {
                g = from[i] + static_cast<int64_t>(kb) * 1024;
            } else {
                const int k = kb * 64 + quad * 16;
                g = from[i] + (k < a.K ? k : 0);
            }
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)g,
                                             (__attribute__((address_space(3))) void *)(lds + place * kStage + (i * 8 + wave) * 1024),
                                             16, 0, 0);
        }
    };
    i32x4 sum[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[r][t] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) stage(s, s);
    // vmcnt(n): all but the two youngest stages have landed; lgkmcnt(0): what was read is here
    constexpr int kYoung = 2 * kPieces, kWait = (kYoung & 15) | ((kYoung >> 4) << 14) | 0x0070;
    static_assert(kYoung < 64, "vmcnt holds 6 bits");
#pragma unroll 1
    for (int kb = 0; kb < a.kblocks; ++kb) {
        // The k-block is there, and all are done with the one before, whose
        // place is next.  (A barrier without the fence of __syncthreads, which
        // would wait for the younger stages too.)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(kWait);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        stage(kb + kStages - 1, (kb + kStages - 1) % kStages);
        const i32x4 *const w = reinterpret_cast<const i32x4 *>(lds + (kb % kStages) * kStage) + wn * RT * 64 + lane;
        const i32x4 *const x = reinterpret_cast<const i32x4 *>(lds + (kb % kStages) * kStage) + (kW + wm * MT) * 64 + lane;
        constexpr int kAhead = RT > 2 ? 2 : 1, kRing = kAhead + 1;
        i32x4 xv[MT], ring[kRing];
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[t] = x[t * 64];
#pragma unroll
        for (int r = 0; r < kAhead; ++r) ring[r] = w[r * 64];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if (r + kAhead < RT) ring[(r + kAhead) % kRing] = w[(r + kAhead) * 64];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < MT; ++t) sum[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ring[r % kRing], xv[t], sum[r][t], 0, 0, 0);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);   // nothing is on its way to LDS when the block ends
    // All scales on their way at once: one after the other, with their waits,
    // they took some 20 us.
    float xs[MT];
    columns v[RT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xs[t] = a.x_scale[min(m0 + (wm * MT + t) * 16 + col, a.M - 1)];
#pragma unroll
    for (int r = 0; r < RT; ++r) v[r] = columns_of(a, (tile0 + wn * RT + r) * 16 + 4 * quad);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t)
            store4(a, m0 + (wm * MT + t) * 16 + col, (tile0 + wn * RT + r) * 16 + 4 * quad, sum[r][t], v[r], xs[t]);
}

template <bool PACKED, int RT, int MT>
aq_status launch_gemm(aq_ctx *ctx, const args &a) {
    auto kernel = i8_gemm_kernel<PACKED, RT, MT>;
    constexpr uint32_t kLds = kStages * (2 * RT + 4 * MT) * 1024;
    aq_status st = aq_launch_lds(ctx, reinterpret_cast<const void *>(kernel), kLds, "aq_i8_forward");
    if (st != AQ_OK) return st;
    const int64_t grid = int64_t{(a.tiles + 2 * RT - 1) / (2 * RT)} * ((a.M + 64 * MT - 1) / (64 * MT));
    aq_launch_timed(ctx, true, kernel, dim3(static_cast<uint32_t>(grid)), dim3(512), kLds, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
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

// How a call's rows of x are multiplied: by blocks that share them in LDS, in
// two sizes, or by waves that split the k-blocks.
enum how : int { kLarge, kMedium, kSplit };

// A block of a size is taken where its tiles give three of four compute units
// one, or where there are so few k-blocks that splitting them gains nothing.
// In us, 8-bit x, large, medium, split, with weights that come from memory
// (matrices in turn, more than the caches hold):
//   K = 4096, N = 4096:    M = 512: 57, 27, 22;   1024: 56, 29, 36;   4096: 71, 98, 115
//   K = 8192, N = 16384:   M = 128: 94, 56, 44;    200: 101, 51, 69;  1024: 132, 196, 228
//   K = 1024, N = 1536:    M = 128: 21, 11, 9;    4096: 25, 18, 28
// and with the same matrix again: 53, 24, 20; 54, 27, 33; 71, 89, 113; 93, 42,
// 37; 94, 49, 64; 119, 172, 221; 20, 9.4, 9.5; 25, 19, 28.
how how_of(const aq_ctx *ctx, const args &a) {
    const int64_t large = int64_t{(a.tiles + 15) / 16} * ((a.M + 255) / 256);
    const int64_t medium = int64_t{(a.tiles + 7) / 8} * ((a.M + 127) / 128);
    if (large >= ctx->num_cus * 3 / 4) return kLarge;
    if (a.M > 64 && (medium >= ctx->num_cus * 3 / 4 || a.kblocks <= 16)) return kMedium;
    return kSplit;
}

template <bool PACKED>
aq_status launch_product(aq_ctx *ctx, const args &a, how h) {
    if (h == kLarge) return launch_gemm<PACKED, 8, 4>(ctx, a);
    if (h == kMedium) return launch_gemm<PACKED, 4, 2>(ctx, a);
    if constexpr (!PACKED) {
        return launch<false, 1, 1, 4>(ctx, a, 8);
    } else {
        if (a.M <= 16) return launch<true, 1, 1, 4>(ctx, a, 8);
        // Four tiles by 64 rows read the weights once for them, where there are
        // enough such blocks; in us, two tiles by 32 rows and these with eight and
        // with four waves, packing included, weights from memory: 64 x 8192 x
        // 16384 46, 34, 37; 128 rows 81, 56, 44; 64 x 4096 x 4096 10.5, 15, 18;
        // 64 x 8192 x 2048 14, 23, 29.
        const int64_t blocks = int64_t{(a.tiles + 3) / 4} * ((a.M + 63) / 64);
        if (a.M <= 32 || blocks < ctx->num_cus) return launch<true, 2, 2, 2>(ctx, a, 8);
        return launch<true, 4, 4, 1>(ctx, a, a.M <= 64 ? 8 : 4);
    }
}

template <typename T>
void launch_quantize(aq_ctx *ctx, const void *x, int64_t x_ld, const args &a, i32x4 *to, float *scales) {
    const auto *rows = static_cast<const typename T::raw *>(x);
    if (a.M <= ctx->num_cus && a.K > 2048)
        aq_launch_timed(ctx, false, i8_quantize_kernel<T, 1, 16>, dim3(static_cast<uint32_t>(a.M)), dim3(1024), 0u, rows, x_ld,
                        a.M, a.K, a.kblocks, to, scales);
    else if (a.M <= 2 * ctx->num_cus)
        aq_launch_timed(ctx, false, i8_quantize_kernel<T, 1, 4>, dim3(static_cast<uint32_t>(a.M)), dim3(256), 0u, rows, x_ld, a.M,
                        a.K, a.kblocks, to, scales);
    else
        aq_launch_timed(ctx, false, i8_quantize_kernel<T, 16, 1>, dim3(static_cast<uint32_t>((a.M + 15) / 16)), dim3(1024), 0u,
                        rows, x_ld, a.M, a.K, a.kblocks, to, scales);
}

// Rows of x at a time in operand order: 64 MB of them, but at least 64, and no
// more than a grid's second axis takes of 16.
constexpr int64_t kPackedBytes = int64_t{64} << 20, kPackedRows = int64_t{1} << 19;

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
    const how h = how_of(ctx, a);
    // 8-bit rows as they are: few, or whole pieces for the blocks that bring them to LDS.
    const bool pieces = w->K % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_ld % 16 == 0;
    if (x_type == AQ_T_I8 && (h == kSplit ? M <= 16 : pieces)) return launch_product<false>(ctx, a, h);
    int64_t rows = kPackedBytes / (int64_t{w->kblocks} * 64) / 64 * 64;
    if (rows < 64) rows = 64;
    if (rows > kPackedRows) rows = kPackedRows;
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
        if (x_type == AQ_T_I8)
            aq_launch_timed(ctx, false, i8_pack_kernel,
                            dim3(static_cast<uint32_t>((b.kblocks + 3) / 4), static_cast<uint32_t>((b.M + 15) / 16)), dim3(256), 0u,
                            from, x_ld, b.M, b.K, b.kblocks, to);
        else if (x_type == AQ_T_F32) launch_quantize<f32>(ctx, from, x_ld, b, to, scales);
        else if (x_type == AQ_T_F16) launch_quantize<f16>(ctx, from, x_ld, b, to, scales);
        else launch_quantize<bf16>(ctx, from, x_ld, b, to, scales);
        AQ_HIP(ctx, hipGetLastError());
        b.x = packed;
        b.x_scale = x_scale ? x_scale + m : scales;
        b.y = static_cast<char *>(y) + m * y_ld * y_size;
        st = launch_product<true>(ctx, b, how_of(ctx, b));
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
