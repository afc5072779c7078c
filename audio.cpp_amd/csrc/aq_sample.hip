// Sampling with temperature, top-k, top-p and min-p from given random numbers
// (aq_sample).
//
// The weights 2^z relative to the row's largest logit are whole numbers of
// 2^-31, so every sum is exact and no split of a row, order of atomics or
// number of blocks changes a result.  The filters keep a prefix of the row in
// the order (logit falling, index rising): a set {key > K} and of {key == K}
// the indices up to I, found by a radix selection on the logits' ordered bits.
// The draw then runs over the kept in index order: no sort.
#include "aq_internal.hpp"
#include "aq_types.hpp"

namespace {

using namespace aq_types;

struct sample_args {
    const void *logits;
    int64_t ld, rows;
    int V;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *token;
    float *logp;
};

constexpr int kMaxV = 1 << 20;
constexpr float kLog2e = 1.4426950408889634f;

// A row's parameters, as the kernels use them.
struct row_params {
    float per;        // log2(e) / temperature
    float min_e;      // min-p
    uint32_t k;       // 0: off
    uint32_t p;       // in 2^-24; 2^24: off
    uint32_t u;       // in 2^-24
};

__device__ inline row_params params_of(const sample_args &a, int64_t row) {
    row_params r;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(t > 0.0f);
    r.per = greedy ? kLog2e : fminf(kLog2e / t, 3.4e38f);
    const int k = a.top_k ? a.top_k[row] : 0;
    r.k = greedy ? 1u : k > 0 && k < a.V ? static_cast<uint32_t>(k) : 0u;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    r.p = p < 1.0f ? static_cast<uint32_t>(fmaxf(p, 0.0f) * 0x1p24f) : 1u << 24;
    const float m = a.min_p ? a.min_p[row] : 0.0f;
    r.min_e = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    const float u = a.u[row];
    r.u = static_cast<uint32_t>(fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f) * 0x1p24f);   // NaN: 0
    return r;
}

// floor(part * total / 2^24) for part <= 2^24 and total < 2^52.
__device__ inline uint64_t share(uint32_t part, uint64_t total) {
    return __umul64hi(static_cast<uint64_t>(part) << 39, total << 1);
}

__device__ inline float z_of(float l, float top, float per) { return (l == top ? 0.0f : l - top) * per; }

// e of a logit; 0 for -infinity and NaN.
__device__ inline float e_of(float l, float top, float per) {
    return l > -INFINITY ? __builtin_amdgcn_exp2f(z_of(l, top, per)) : 0.0f;
}

__device__ inline uint32_t w_of(float e) { return static_cast<uint32_t>(e * 0x1p31f); }

// ln(2^z / (total / 2^31)), rounded once: the two terms may nearly cancel, or
// the second be many times the first.
__device__ inline float logp_of(float z, uint64_t total) {
    return static_cast<float>(static_cast<double>(z) * 0.69314718055994530942 - log(static_cast<double>(total) * 0x1p-31));
}

// The bits of a logit in its order; -0 as 0.
__device__ inline uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

// Inclusive sum over the lanes up to this one.
__device__ inline uint64_t wave_scan(uint64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t other = __shfl_up(v, o);
        if (lane >= o) v += other;
    }
    return v;
}

__device__ inline uint64_t wave_total(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(sample_args a) {
    constexpr int kWaves = THREADS / 64;
    __shared__ uint64_t hist[256];
    __shared__ uint64_t part[kWaves];
    __shared__ uint64_t found[2];   // what a selection step hands on
    using raw = typename T::raw;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const raw *logits = static_cast<const raw *>(a.logits) + row * a.ld;
    const row_params r = params_of(a, row);
    // Each wave owns a run of whole 64s of the row, in index order.
    const int run = (a.V + 64 * kWaves - 1) / (64 * kWaves) * 64;
    const int begin = min(wave * run, a.V), end = min(begin + run, a.V);

    float top = -INFINITY;
    for (int i = threadIdx.x; i < a.V; i += THREADS) top = fmaxf(top, T::load(logits[i]));   // not a NaN
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) part[wave] = __float_as_uint(top);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, __uint_as_float(static_cast<uint32_t>(part[w])));
    __syncthreads();
    if (!(top > -INFINITY)) {
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            if (a.logp) a.logp[row] = -INFINITY;
        }
        return;
    }

    uint32_t K = 0;         // kept: key > K, or key == K and index <= I
    int I = a.V;
    const auto kept = [&](uint32_t key, int i) { return key > K || (key == K && i <= I); };
    // The sum over the block of each thread's value, known to all.
    const auto block_total = [&](uint64_t v) {
        v = wave_total(v);
        if (lane == 0) part[wave] = v;
        __syncthreads();
        uint64_t s = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) s += part[w];
        __syncthreads();
        return s;
    };
    // The first place in index order where the running sum of `amount`
    // exceeds t, -1 if none; all threads get it.
    const auto first_over = [&](auto &&amount, uint64_t t) {
        uint64_t mine = 0;
        for (int i = begin + lane; i < end; i += 64) mine += amount(i);
        mine = wave_total(mine);
        if (lane == 0) part[wave] = mine;
        if (threadIdx.x == 0) found[0] = ~0ull;
        __syncthreads();
        uint64_t before = 0;
        for (int w = 0; w < wave; ++w) before += part[w];
        if (before <= t && before + mine > t) {   // one wave
            for (int i = begin; i < end; i += 64) {
                const uint64_t upto = before + wave_scan(i + lane < end ? amount(i + lane) : 0);
                const uint64_t over = __ballot(upto > t);
                if (over) {
                    if (lane == 0) found[0] = static_cast<uint64_t>(i + __builtin_ctzll(over));
                    break;
                }
                before = __shfl(upto, 63);
            }
        }
        __syncthreads();
        const int at = static_cast<int>(found[0]);
        __syncthreads();
        return at;
    };
    // Narrows the kept set to its shortest prefix whose amounts (1, or the
    // weights) reach `need`; leaves it if they do not.
    const auto select = [&](bool by_weight, uint64_t need) {
        uint32_t prefix = 0, mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int b = threadIdx.x; b < 256; b += THREADS) hist[b] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < a.V; i += THREADS) {
                const float l = T::load(logits[i]);
                const uint32_t w = w_of(e_of(l, top, r.per)), key = key_of(l);
                if (w && (key & mask) == prefix && kept(key, i))
                    atomicAdd(reinterpret_cast<unsigned long long *>(&hist[(key >> shift) & 255u]), by_weight ? w : 1u);
            }
            __syncthreads();
            if (wave == 0) {   // bins from the top, four a lane
                uint64_t sum = 0;
                for (int b = 0; b < 4; ++b) sum += hist[255 - 4 * lane - b];
                const uint64_t upto = wave_scan(sum);
                const uint64_t over = __ballot(upto >= need);
                if (lane == 0) found[0] = over ? 1 : 0;
                if (over && lane == __builtin_ctzll(over)) {
                    uint64_t before = upto - sum;
                    int b = 255 - 4 * lane;
                    while (before + hist[b] < need) before += hist[b--];
                    found[0] = 2 + static_cast<uint64_t>(b);
                    found[1] = need - before;
                }
            }
            __syncthreads();
            const uint64_t f = found[0], rest = found[1];
            __syncthreads();
            if (f < 2) return;   // fewer than needed: all stay (on the first pass only)
            prefix |= static_cast<uint32_t>(f - 2) << shift;
            mask |= 255u << shift;
            need = rest;
        }
        // Of the equal logits of key `prefix`, the first that together reach what is left.
        uint64_t each = 1;
        if (by_weight) {
            const uint32_t b = prefix & 0x80000000u ? prefix ^ 0x80000000u : ~prefix;
            each = w_of(e_of(__uint_as_float(b), top, r.per));
        }
        const uint64_t count = (need + each - 1) / each;
        const int at = first_over([&](int i) -> uint64_t {
            const uint32_t key = key_of(T::load(logits[i]));
            return key == prefix && kept(key, i) ? 1u : 0u;
        }, count - 1);
        K = prefix;
        I = at;
    };

    if (r.k) select(false, r.k);
    if (r.p < 1u << 24) {
        uint64_t mine = 0;
        for (int i = threadIdx.x; i < a.V; i += THREADS) {
            const float l = T::load(logits[i]);
            if (kept(key_of(l), i)) mine += w_of(e_of(l, top, r.per));
        }
        const uint64_t need = share(r.p, block_total(mine));
        select(true, need ? need : 1);
    }
    const auto weight = [&](int i) -> uint64_t {
        const float l = T::load(logits[i]);
        const float e = e_of(l, top, r.per);
        return kept(key_of(l), i) && e >= r.min_e ? w_of(e) : 0u;
    };
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < a.V; i += THREADS) mine += weight(i);
    const uint64_t total = block_total(mine);
    const int at = first_over(weight, share(r.u, total));
    if (threadIdx.x == 0) {
        a.token[row] = at;
        if (a.logp) a.logp[row] = logp_of(z_of(T::load(logits[at]), top, r.per), total);
    }
}

template <typename T>
void launch(aq_ctx *ctx, const sample_args &a) {
    const dim3 grid(static_cast<uint32_t>(a.rows));
    if (a.V <= 4096) aq_launch_timed(ctx, true, sample_kernel<T, 256>, grid, dim3(256), 0u, a);
    else aq_launch_timed(ctx, true, sample_kernel<T, 1024>, grid, dim3(1024), 0u, a);
}

}  // namespace

extern "C" aq_status aq_sample(aq_ctx *ctx, int type, const void *logits, int64_t ld, int64_t rows, int64_t V,
                               const float *u, const float *temperature, const int32_t *top_k, const float *top_p,
                               const float *min_p, int32_t *token, float *logp) {
    if (!ctx) return AQ_E_INVALID_ARG;
    if (type != AQ_T_F32 && type != AQ_T_F16 && type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_sample: type %d is not F32, F16 or BF16", type);
    if (rows < 0 || rows > int64_t{1} << 21 || V < 1 || V > kMaxV)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_sample: rows=%lld V=%lld (rows up to 2^21, V from 1 to 2^20)",
                       (long long)rows, (long long)V);
    if (rows == 0) return AQ_OK;
    if (!logits || !u || !token) return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_sample: null logits, u or token");
    if (ld < V) return aq_fail(ctx, AQ_E_SHAPE, "aq_sample: row stride %lld is below V=%lld", (long long)ld, (long long)V);
    aq_device_guard g(ctx->device);
    const sample_args a{logits, ld, rows, static_cast<int>(V), u, temperature, top_p, min_p, top_k, token, logp};
    if (type == AQ_T_F32) launch<f32>(ctx, a);
    else if (type == AQ_T_F16) launch<f16>(ctx, a);
    else launch<bf16>(ctx, a);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}
