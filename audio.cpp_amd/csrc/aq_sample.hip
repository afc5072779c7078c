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

__device__ inline float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// The weight of a key; 0 for key 0 (no element).
__device__ inline uint32_t weight_of(uint32_t key, float top, float per) {
    const uint32_t w = w_of(e_of(logit_of(key), top, per));   // key 0 is a NaN: 0
    return key ? w : 0;
}

// Lane i gets lane i - n's value (rows of 16: n = 1, 2, 4, 8), or the last of
// the row(s) before (0x142, 0x143); 0 where there is none.  These are register
// moves, where a shuffle goes through LDS.
template <int CTRL, int ROWS>
__device__ inline uint32_t dpp(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}

template <int CTRL, int ROWS>
__device__ inline uint64_t scan_step(uint64_t v) {
    return v + (static_cast<uint64_t>(dpp<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32 |
                dpp<CTRL, ROWS>(static_cast<uint32_t>(v)));
}

// Inclusive sum over the lanes up to this one.
__device__ inline uint64_t wave_scan(uint64_t v) {
    v = scan_step<0x111, 0xF>(v);
    v = scan_step<0x112, 0xF>(v);
    v = scan_step<0x114, 0xF>(v);
    v = scan_step<0x118, 0xF>(v);
    v = scan_step<0x142, 0xA>(v);
    return scan_step<0x143, 0xC>(v);
}

__device__ inline uint32_t lane_value(uint32_t v, int lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

__device__ inline uint64_t lane_value(uint64_t v, int lane) {
    return static_cast<uint64_t>(lane_value(static_cast<uint32_t>(v >> 32), lane)) << 32 |
           lane_value(static_cast<uint32_t>(v), lane);
}

// A value that all lanes hold, as a scalar.
__device__ inline uint32_t uniform(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); }

__device__ inline uint64_t wave_total(uint64_t v) { return lane_value(wave_scan(v), 63); }

// The largest key of the wave (0 is below every key).
__device__ inline uint32_t wave_max(uint32_t v) {
    v = max(v, dpp<0x111, 0xF>(v));
    v = max(v, dpp<0x112, 0xF>(v));
    v = max(v, dpp<0x114, 0xF>(v));
    v = max(v, dpp<0x118, 0xF>(v));
    v = max(v, dpp<0x142, 0xA>(v));
    v = max(v, dpp<0x143, 0xC>(v));
    return lane_value(v, 63);
}

// The elements of a row that a block holds in registers, in index order:
// WAVES waves, E elements a thread, in vectors of 8: wave w, vector v, lane i
// hold elements ((w * E / 8 + v) * 64 + i) * 8 ..+7.  `key` is 0 where there
// is no element, or one that is never drawn; `w` is the weight.  Every wave
// takes every decision for itself from what lies in LDS, so a step needs no
// barrier for its result.
template <int WAVES>
struct list_lds {
    uint64_t bins[256];
    uint64_t part[WAVES];
    uint32_t key[64], index[64], weight[64];
    uint32_t count, hi, lo, at;
};

template <int WAVES, int E, bool GIVEN = false>   // GIVEN: the elements bring their indices
struct row_list {
    static constexpr int kThreads = 64 * WAVES;
    list_lds<WAVES> &s;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6));
    uint32_t key[E], w[E];
    uint32_t given[GIVEN ? E : 1];
    uint32_t K = 1, I = 0xFFFFFFFFu;   // kept: key > K, or key == K and index <= I

    __device__ explicit row_list(list_lds<WAVES> &lds) : s(lds) {}

    __device__ uint32_t place(int e) const {   // in the list
        return static_cast<uint32_t>(((wave * (E / 8) + e / 8) * 64 + lane) * 8 + e % 8);
    }
    __device__ uint32_t index(int e) const { return GIVEN ? given[e] : place(e); }
    // No branches in the tests of elements: they are a few comparisons, and
    // ROCm 7.2's compiler has dropped the copy of a 64-bit value that a
    // short-circuit left to one of its paths.
    __device__ bool kept(int e) const { return (key[e] > K) | ((key[e] == K) & (index(e) <= I)); }

    // Each wave's sum of `mine` in s.part; the sum over the block.
    __device__ uint64_t total(uint64_t mine) {
        mine = wave_total(mine);
        if (WAVES == 1) return mine;
        __syncthreads();
        if (lane == 0) s.part[wave] = mine;
        __syncthreads();
        uint64_t sum = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) sum += s.part[i];
        return sum;
    }

    // After total() of amount(e) summed over each thread's elements: `hit`
    // runs in the thread of the first element where the running sum in index
    // order exceeds t.
    template <typename A, typename H>
    __device__ void first_over(A &&amount, uint64_t t, uint64_t mine, H &&hit) {
        uint64_t before = 0;
        if (WAVES > 1) {
            for (int i = 0; i < wave; ++i) before += s.part[i];
            mine = s.part[wave];
        } else {
            mine = wave_total(mine);
        }
        if (t < before || t >= before + mine) return;   // not in this wave
#pragma unroll
        for (int v = 0; v < E / 8; ++v) {
            uint64_t eight = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) eight += amount(8 * v + i);
            const uint64_t upto = before + wave_scan(eight);
            const uint64_t over = __ballot(upto > t);
            if (over && t >= before) {
                if (lane == __builtin_ctzll(over)) {
                    uint64_t sum = upto - eight;
                    bool found = false;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        sum += amount(8 * v + i);
                        if (!found && sum > t) {
                            found = true;
                            hit(8 * v + i);
                        }
                    }
                }
            }
            before = lane_value(upto, 63);
        }
    }

    // Narrows the kept set to its shortest prefix (logit falling, index
    // rising) whose amounts (1, or the weights) reach `need` >= 1; leaves it
    // if they do not.
    //
    // 256 bins of the elements in question; the bin where the running amount
    // crosses `need` is what remains in question, until it holds at most 64
    // elements, which a wave orders by comparing all pairs.  The first bins
    // are an eighth of a bit of weight wide (`per`: bits per unit of logit), so
    // that a usual row needs no others; the next ones are linear in the key,
    // which tells any two different logits apart after three more.
    __device__ void select(bool by_weight, uint64_t need, float top, float per) {
        uint32_t hi = 0xFFFFFFFFu, lo = 1;
        int shift = -1;   // of the key, from the second level on
        const float scale = fminf(8.0f * per, 3.4e38f);
        for (;;) {
            __syncthreads();
            for (int b = threadIdx.x; b < 256; b += kThreads) s.bins[b] = 0;
            if (threadIdx.x == 0) {
                s.count = 0;
                s.hi = 0;
                s.lo = 0xFFFFFFFFu;
            }
            __syncthreads();
            uint32_t bin[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                bin[e] = 256;
                uint32_t b;
                if (shift < 0) {
                    const float l = logit_of(key[e]);
                    b = static_cast<uint32_t>(fminf((l == top ? 0.0f : top - l) * scale, 255.0f));
                } else {
                    b = (hi - key[e]) >> shift;
                }
                if ((key[e] >= lo) & (key[e] <= hi) & kept(e)) bin[e] = b;
                if (bin[e] < 256) atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[bin[e]]), by_weight ? w[e] : 1u);
            }
            __syncthreads();
            uint64_t four[4], sum = 0;   // bins 4 lane ..+3, the largest logits first
#pragma unroll
            for (int b = 0; b < 4; ++b) sum += four[b] = s.bins[4 * lane + b];
            const uint64_t upto = wave_scan(sum);
            const uint64_t over = __ballot(upto >= need);
            if (!over) return;   // on the first level only
            const int owner = __builtin_ctzll(over);
            uint64_t before = upto - sum;
            uint32_t b = 0;
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (b == static_cast<uint32_t>(i) && before + four[i] < need) {
                    before += four[i];
                    ++b;
                }
            const uint32_t chosen = 4 * owner + lane_value(b, owner);
            need -= lane_value(before, owner);
            // The bin's elements: the first 64 into the short list, and their range.
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (bin[e] != chosen) continue;
                const uint32_t at = atomicAdd(&s.count, 1u);
                if (at < 64) {
                    s.key[at] = key[e];
                    s.index[at] = index(e);
                    s.weight[at] = by_weight ? w[e] : 1u;
                } else {
                    atomicMax(&s.hi, key[e]);
                    atomicMin(&s.lo, key[e]);
                }
            }
            __syncthreads();
            const uint32_t n = uniform(s.count);
            const uint32_t k = static_cast<uint32_t>(lane) < n ? s.key[lane] : 0;
            if (n <= 64) {
                const uint32_t at = static_cast<uint32_t>(lane) < n ? s.index[lane] : 0;
                const uint32_t amount = static_cast<uint32_t>(lane) < n ? s.weight[lane] : 0;
                uint64_t ahead = 0;
                for (uint32_t i = 0; i < n; ++i) {
                    const uint32_t ki = lane_value(k, i), ai = lane_value(at, i);
                    ahead += ((ki > k) | ((ki == k) & (ai < at))) ? lane_value(amount, i) : 0u;
                }
                const int last = __builtin_ctzll(__ballot((ahead < need) & (ahead + amount >= need)));
                K = lane_value(k, last);
                I = lane_value(at, last);
                return;
            }
            hi = max(uniform(s.hi), wave_max(k));
            lo = min(uniform(s.lo), ~wave_max(~k));
            if (hi == lo) break;
            shift = max(0, 24 - __builtin_clz(hi - lo));
        }
        // More than 64 equal logits cross: the first of them in index order.
        const uint32_t equal = lo;
        const auto one = [&](int e) { return ((key[e] == equal) & kept(e)) ? 1u : 0u; };
        uint64_t each = 1;
        if (by_weight) each = uniform(s.weight[0]);
        const uint64_t count = (need + each - 1) / each;
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += one(e);
        total(mine);
        first_over(one, count - 1, mine, [&](int e) { s.at = index(e); });
        __syncthreads();
        K = equal;
        I = uniform(s.at);
    }

    __device__ uint64_t kept_weight() const {   // this thread's
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += kept(e) ? w[e] : 0u;
        return mine;
    }

    // Draws from what is kept and is not below min-p, and writes the outputs.
    __device__ void draw(const sample_args &a, int64_t row, const row_params &r, float top) {
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = kept(e) ? w[e] : 0u;
            if (r.min_e > 0.0f) w[e] = e_of(logit_of(key[e]), top, r.per) >= r.min_e ? w[e] : 0u;
            mine += w[e];
        }
        const uint64_t sum = total(mine);
        first_over([&](int e) { return w[e]; }, share(r.u, sum), mine, [&](int e) {
            a.token[row] = static_cast<int32_t>(index(e));
            if (a.logp) a.logp[row] = logp_of(z_of(logit_of(key[e]), top, r.per), sum);
        });
    }
};

// 8 logits of a row as keys, 0 for those that are never drawn (or past the end).
template <typename T>
__device__ inline void load_keys(const typename T::raw *logits, int at, int V, uint32_t *key) {
    float l[8];
    load8<T>(logits, at, V, l, T::store(-INFINITY));
#pragma unroll
    for (int i = 0; i < 8; ++i) key[i] = l[i] > -INFINITY ? key_of(l[i]) : 0;
}

__device__ inline void write_empty(const sample_args &a, int64_t row) {
    a.token[row] = -1;
    if (a.logp) a.logp[row] = -INFINITY;
}

// Rows that fit the registers of a block.
template <typename T, int WAVES, int E>
__global__ __launch_bounds__(64 * WAVES) void sample_short_kernel(sample_args a) {
    __shared__ list_lds<WAVES> lds;
    using raw = typename T::raw;
    const int64_t row = blockIdx.x;
    const raw *logits = static_cast<const raw *>(a.logits) + row * a.ld;
    row_list<WAVES, E> list(lds);
    uint32_t top_key = 0;
#pragma unroll
    for (int v = 0; v < E / 8; ++v) load_keys<T>(logits, static_cast<int>(list.index(8 * v)), a.V, list.key + 8 * v);
#pragma unroll
    for (int e = 0; e < E; ++e) top_key = max(top_key, list.key[e]);
    const row_params r = params_of(a, row);
    top_key = wave_max(top_key);
    if (WAVES > 1) {
        if (list.lane == 0) lds.part[list.wave] = top_key;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top_key = max(top_key, static_cast<uint32_t>(lds.part[i]));
    }
    if (!top_key) {
        if (threadIdx.x == 0) write_empty(a, row);
        return;
    }
    const float top = logit_of(top_key);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        list.w[e] = weight_of(list.key[e], top, r.per);
        if (!list.w[e]) list.key[e] = 0;
    }
    if (r.k) list.select(false, r.k, top, r.per);
    if (r.p < 1u << 24) {
        const uint64_t need = share(r.p, list.total(list.kept_weight()));
        list.select(true, need ? need : 1, top, r.per);
    }
    list.draw(a, row, r, top);
}

// Longer rows: chunks of 4096 elements, a block each, in three launches.
//
//  1. the largest logit of each chunk;
//  2. the weights, relative to the row's largest; their sum over the chunk;
//     and, for rows with filters, the chunk's candidates: the elements of its
//     largest logits, in index order, as many whole half-bits of weight as fit
//     its slots;
//  3. a block per row.  Without filters it finds the chunk that the draw falls
//     into from the sums, and draws in it.  With filters it works on the
//     candidates down to the least half-bit that every chunk has given whole,
//     which holds the kept set unless that is very wide; else it streams the
//     row.
constexpr int kChunk = 4096;          // 256 threads, 16 elements each
constexpr int kSlots = 8192;          // candidates of a row: 1024 threads, 8 each
constexpr int kRowsAtOnce = 1024;

struct chunk_store {
    uint32_t *top;      // [rows][chunks] largest key
    uint64_t *weight;   // [rows][chunks] sum of weights (of those that min-p leaves, for rows without other filters)
    int32_t *whole;     // [rows][chunks] the last half-bit given whole, -1: none
    uint32_t *count;    // [rows][chunks] candidates
    uint2 *slot;        // [rows][chunks][cap] key, index
    int chunks, cap;
};

// The half-bit of weight below the largest that a key falls into, 0 to 63.
__device__ inline uint32_t half_bit(uint32_t key, float top, float scale) {
    const float l = logit_of(key);
    return static_cast<uint32_t>(fminf((l == top ? 0.0f : top - l) * scale, 63.0f));
}

template <typename T>
__global__ __launch_bounds__(256) void sample_top_kernel(sample_args a, chunk_store c, int64_t row0) {
    __shared__ uint32_t part[4];
    const int64_t r = blockIdx.y;
    const typename T::raw *logits = static_cast<const typename T::raw *>(a.logits) + (row0 + r) * a.ld;
    const int at = static_cast<int>(blockIdx.x) * kChunk + static_cast<int>(threadIdx.x) * 8;
    uint32_t key[16], top = 0;
    load_keys<T>(logits, at, a.V, key);
    load_keys<T>(logits, at + 2048, a.V, key + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, key[e]);
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) c.top[r * c.chunks + blockIdx.x] = max(max(part[0], part[1]), max(part[2], part[3]));
}

// The largest key of a row from its chunks'; every wave for itself.
__device__ inline uint32_t row_top(const chunk_store &c, int64_t r) {
    uint32_t top = 0;
    for (int i = threadIdx.x & 63; i < c.chunks; i += 64) top = max(top, c.top[r * c.chunks + i]);
    return wave_max(top);
}

template <typename T>
__global__ __launch_bounds__(256) void sample_chunk_kernel(sample_args a, chunk_store c, int64_t row0) {
    __shared__ uint32_t bins[64];
    __shared__ uint64_t part[4];
    __shared__ uint32_t counts[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = blockIdx.y, row = row0 + r, chunk = r * c.chunks + blockIdx.x;
    const typename T::raw *logits = static_cast<const typename T::raw *>(a.logits) + row * a.ld;
    const int base = static_cast<int>(blockIdx.x) * kChunk + (wave * 128 + lane) * 8;   // vectors at +0 and +512
    uint32_t key[16], w[16];
    load_keys<T>(logits, base, a.V, key);
    load_keys<T>(logits, base + 512, a.V, key + 8);
    const row_params p = params_of(a, row);
    const uint32_t top_key = row_top(c, r);
    if (!top_key) return;   // the whole row is empty
    const float top = logit_of(top_key);
    const bool filtered = p.k || p.p < 1u << 24;

    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        w[e] = weight_of(key[e], top, p.per);
        if (!filtered && p.min_e > 0.0f) w[e] = e_of(logit_of(key[e]), top, p.per) >= p.min_e ? w[e] : 0u;
        mine += w[e];
    }
    mine = wave_total(mine);
    if (lane == 0) part[wave] = mine;
    if (threadIdx.x < 64) bins[threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x == 0) c.weight[chunk] = part[0] + part[1] + part[2] + part[3];
    if (!filtered) return;

    const float scale = fminf(2.0f * p.per, 3.4e38f);
    uint32_t bin[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        bin[e] = w[e] ? half_bit(key[e], top, scale) : 64u;
        if (w[e]) atomicAdd(&bins[bin[e]], 1u);
    }
    __syncthreads();
    const uint32_t upto = static_cast<uint32_t>(wave_scan(bins[lane]));
    const int whole = __popcll(__ballot(upto <= static_cast<uint32_t>(c.cap))) - 1;   // upto does not fall with the lane

    // This thread's candidates in both vectors, counted before it in the wave.
    uint32_t own = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) own += static_cast<int>(bin[e]) <= whole ? (e < 8 ? 1u : 0x10000u) : 0u;
    const uint32_t through = static_cast<uint32_t>(wave_scan(own));   // no carry between the halves: at most 512 each
    const uint32_t all = lane_value(through, 63);
    if (lane == 0) counts[wave] = (all & 0xFFFFu) + (all >> 16);
    __syncthreads();
    uint32_t first = 0;
    for (int i = 0; i < wave; ++i) first += counts[i];
    uint32_t at[2] = {first + ((through - own) & 0xFFFFu), first + (all & 0xFFFFu) + ((through - own) >> 16)};
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if (static_cast<int>(bin[e]) <= whole)
            c.slot[chunk * c.cap + at[e / 8]++] = make_uint2(key[e], static_cast<uint32_t>(base + (e / 8) * 512 + e % 8));
    if (threadIdx.x == 0) {
        c.count[chunk] = counts[0] + counts[1] + counts[2] + counts[3];
        c.whole[chunk] = whole;
    }
}

// A row streamed from memory by a block of 16 waves: wave w has the run of
// whole vectors of 512 elements from w * run on, so that the waves' sums in
// order give index order.
template <typename T>
struct row_stream {
    using raw = typename T::raw;
    struct lds {
        uint64_t bins[2048];
        uint64_t part[16];
        uint32_t key[64], index[64], weight[64];
        uint32_t count, hi, lo, chosen;
        uint64_t before;
    };
    lds &s;
    const raw *logits;
    const int V;
    const float top, per;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6));
    const int run, begin, end;
    uint32_t K = 1, I = 0xFFFFFFFFu;

    __device__ row_stream(lds &l, const raw *p, int n, float t, float f)
        : s(l), logits(p), V(n), top(t), per(f), run((n + 8191) / 8192 * 512), begin(min(wave * run, n)),
          end(min(begin + run, n)) {}

    __device__ bool kept(uint32_t key, int i) const {
        return (key > K) | ((key == K) & (static_cast<uint32_t>(i) <= I));
    }

    // f(key, index) of every element of this wave's run that is ever drawn's key, or 0.
    template <typename F>
    __device__ void each(F &&f) {
        for (int i = begin; i < end; i += 512) {
            uint32_t key[8];
            load_keys<T>(logits, i + lane * 8, V, key);
#pragma unroll
            for (int e = 0; e < 8; ++e) f(key[e], i + lane * 8 + e);
        }
    }

    // The sum over the block of amount(key, index); each wave's in s.part.
    template <typename A>
    __device__ uint64_t total(A &&amount) {
        uint64_t mine = 0;
        each([&](uint32_t key, int i) { mine += amount(key, i); });
        mine = wave_total(mine);
        __syncthreads();
        if (lane == 0) s.part[wave] = mine;
        __syncthreads();
        return wave_total(lane < 16 ? s.part[lane] : 0);
    }

    // After total(amount): hit(key, index) of the first element where the running sum exceeds t.
    template <typename A, typename H>
    __device__ void first_over(A &&amount, uint64_t t, H &&hit) {
        const uint64_t sums = wave_scan(lane < 16 ? s.part[lane] : 0);
        uint64_t before = wave ? lane_value(sums, wave - 1) : 0;
        if (t < before || t >= lane_value(sums, wave)) return;
        for (int i = begin; i < end; i += 512) {
            uint32_t key[8];
            load_keys<T>(logits, i + lane * 8, V, key);
            uint64_t eight = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) eight += amount(key[e], i + lane * 8 + e);
            const uint64_t upto = before + wave_scan(eight);
            const uint64_t over = __ballot(upto > t);
            if (over) {
                if (lane == __builtin_ctzll(over)) {
                    uint64_t sum = upto - eight;
                    bool found = false;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        sum += amount(key[e], i + lane * 8 + e);
                        if (!found & (sum > t)) {
                            found = true;
                            hit(key[e], i + lane * 8 + e);
                        }
                    }
                }
                return;
            }
            before = lane_value(upto, 63);
        }
    }

    // As row_list::select, with 2048 bins (the first 1/64 of a bit wide).
    __device__ void select(bool by_weight, uint64_t need) {
        uint32_t hi = 0xFFFFFFFFu, lo = 1;
        int shift = -1;
        const float scale = fminf(64.0f * per, 3.4e38f);
        const auto bin_of = [&](uint32_t key) {
            const float l = logit_of(key);
            return shift < 0 ? static_cast<uint32_t>(fminf((l == top ? 0.0f : top - l) * scale, 2047.0f))
                             : (hi - key) >> shift;
        };
        for (;;) {
            __syncthreads();
            s.bins[threadIdx.x] = 0;
            s.bins[threadIdx.x + 1024] = 0;
            if (threadIdx.x == 0) {
                s.count = 0;
                s.hi = 0;
                s.lo = 0xFFFFFFFFu;
                s.chosen = 0xFFFFFFFFu;
            }
            __syncthreads();
            each([&](uint32_t key, int i) {
                const uint32_t w = weight_of(key, top, per);
                if ((w != 0) & (key >= lo) & (key <= hi) & kept(key, i))
                    atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[bin_of(key)]), by_weight ? w : 1u);
            });
            __syncthreads();
            if (wave == 0) {   // 32 bins a lane, from the largest logits
                uint64_t sum = 0;
                for (int b = 0; b < 32; ++b) sum += s.bins[32 * lane + b];
                const uint64_t upto = wave_scan(sum);
                const uint64_t over = __ballot(upto >= need);
                if (over && lane == __builtin_ctzll(over)) {
                    uint64_t before = upto - sum;
                    uint32_t b = 32 * lane;
                    for (int i = 0; i < 31; ++i) {
                        const uint64_t next = before + s.bins[b];
                        const bool on = next < need;
                        before = on ? next : before;
                        b += on ? 1u : 0u;
                        if (!on) break;
                    }
                    s.chosen = b;
                    s.before = before;
                }
            }
            __syncthreads();
            const uint32_t chosen = uniform(s.chosen);
            if (chosen == 0xFFFFFFFFu) return;
            need -= lane_value(s.before, 0);
            uint32_t high = 0, low = 0xFFFFFFFFu;
            each([&](uint32_t key, int i) {
                const uint32_t w = weight_of(key, top, per);
                if ((w != 0) & (key >= lo) & (key <= hi) & kept(key, i) & (bin_of(key) == chosen)) {
                    high = max(high, key);
                    low = min(low, key);
                    const uint32_t at = atomicAdd(&s.count, 1u);
                    if (at < 64) {
                        s.key[at] = key;
                        s.index[at] = static_cast<uint32_t>(i);
                        s.weight[at] = by_weight ? w : 1u;
                    }
                }
            });
            high = wave_max(high);
            low = ~wave_max(~low);
            if (lane == 0) {
                atomicMax(&s.hi, high);
                atomicMin(&s.lo, low);
            }
            __syncthreads();
            const uint32_t n = uniform(s.count);
            if (n <= 64) {
                const bool there = static_cast<uint32_t>(lane) < n;
                const uint32_t k = there ? s.key[lane] : 0, at = there ? s.index[lane] : 0;
                const uint32_t amount = there ? s.weight[lane] : 0;
                uint64_t ahead = 0;
                for (uint32_t i = 0; i < n; ++i) {
                    const uint32_t ki = lane_value(k, i), ai = lane_value(at, i);
                    ahead += ((ki > k) | ((ki == k) & (ai < at))) ? lane_value(amount, i) : 0u;
                }
                const int last = __builtin_ctzll(__ballot((ahead < need) & (ahead + amount >= need)));
                K = lane_value(k, last);
                I = lane_value(at, last);
                return;
            }
            hi = uniform(s.hi);
            lo = uniform(s.lo);
            if (hi == lo) break;
            shift = max(0, 21 - __builtin_clz(hi - lo));
        }
        const uint32_t equal = lo;
        const uint64_t each_one = by_weight ? uniform(s.weight[0]) : 1u;
        const uint64_t count = (need + each_one - 1) / each_one;
        const auto one = [&](uint32_t key, int i) -> uint64_t { return ((key == equal) & kept(key, i)) ? 1u : 0u; };
        total(one);
        first_over(one, count - 1, [&](uint32_t, int i) { s.chosen = static_cast<uint32_t>(i); });
        __syncthreads();
        K = equal;
        I = uniform(s.chosen);
    }
};

template <typename T>
__global__ __launch_bounds__(1024) void sample_row_kernel(sample_args a, chunk_store c, int64_t row0) {
    using stream_t = row_stream<T>;
    __shared__ union {
        list_lds<16> list;
        typename stream_t::lds stream;
    } lds;
    __shared__ uint64_t found_before;
    __shared__ int found_chunk;
    const int lane = threadIdx.x & 63;
    const int64_t r = blockIdx.x, row = row0 + r, chunk0 = r * c.chunks;
    const typename T::raw *logits = static_cast<const typename T::raw *>(a.logits) + row * a.ld;
    const row_params p = params_of(a, row);
    const uint32_t top_key = row_top(c, r);
    if (!top_key) {
        if (threadIdx.x == 0) write_empty(a, row);
        return;
    }
    const float top = logit_of(top_key);
    const bool filtered = p.k || p.p < 1u << 24;

    // The row's weight, and for filtered rows the least half-bit given whole.
    int whole = 63;
    uint64_t weight = 0;
    for (int i = lane; i < c.chunks; i += 64) {
        weight += c.weight[chunk0 + i];
        if (filtered) whole = min(whole, c.whole[chunk0 + i]);
    }
    weight = wave_total(weight);
    whole = static_cast<int>(63u - wave_max(static_cast<uint32_t>(63 - whole)));

    if (!filtered) {
        // The chunk where the running weight exceeds t, and the draw in it: 4096 elements, 8 for each of 512 threads.
        const uint64_t t = share(p.u, weight);
        if (threadIdx.x < 64) {
            uint64_t before = 0;
            for (int i = 0; i < c.chunks; i += 64) {
                const uint64_t upto = before + wave_scan(i + lane < c.chunks ? c.weight[chunk0 + i + lane] : 0);
                const uint64_t over = __ballot(upto > t);
                if (over) {
                    const int owner = __builtin_ctzll(over);
                    if (lane == owner) {
                        found_chunk = i + lane;
                        found_before = upto - c.weight[chunk0 + i + lane];
                    }
                    break;
                }
                before = lane_value(upto, 63);
            }
        }
        __syncthreads();
        const int base = static_cast<int>(uniform(static_cast<uint32_t>(found_chunk))) * kChunk;
        const uint64_t rest = t - found_before;
        row_list<16, 8> list(lds.list);
        const int at = static_cast<int>(list.place(0));
        load_keys<T>(logits, base + at, at < kChunk ? a.V : 0, list.key);
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            list.w[e] = weight_of(list.key[e], top, p.per);
            if (p.min_e > 0.0f) list.w[e] = e_of(logit_of(list.key[e]), top, p.per) >= p.min_e ? list.w[e] : 0u;
            mine += list.w[e];
        }
        list.total(mine);
        list.first_over([&](int e) { return list.w[e]; }, rest, mine, [&](int e) {
            a.token[row] = base + static_cast<int>(list.place(e));
            if (a.logp) a.logp[row] = logp_of(z_of(logit_of(list.key[e]), top, p.per), weight);
        });
        return;
    }

    {
        row_list<16, 8, true> list(lds.list);
        const float scale = fminf(2.0f * p.per, 3.4e38f);
        uint64_t count = 0;
        const int place = static_cast<int>(list.place(0)), chunk = place / c.cap, first = place % c.cap;
        const int n = chunk < c.chunks ? static_cast<int>(c.count[chunk0 + chunk]) - first : 0;
        const uint2 *slot = c.slot + (chunk0 + chunk) * c.cap + first;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint2 s = e < n ? slot[e] : make_uint2(0, 0);
            list.key[e] = static_cast<int>(half_bit(s.x, top, scale)) > whole ? 0u : s.x;
            list.given[e] = s.y;
            list.w[e] = weight_of(s.x, top, p.per);
            count += list.key[e] ? 1u : 0u;
        }
        // Complete down to what the filters ask for?
        const bool all = whole == 63;
        bool enough = true;
        if (p.k) enough = all || list.total(count) >= p.k;
        uint64_t need = 0;
        if (!p.k) {
            need = share(p.p, weight);
            enough = all || list.total(list.kept_weight()) >= (need ? need : 1);
        }
        if (enough) {
            if (p.k) list.select(false, p.k, top, p.per);
            if (p.p < 1u << 24) {
                if (p.k) need = share(p.p, list.total(list.kept_weight()));
                list.select(true, need ? need : 1, top, p.per);
            }
            list.draw(a, row, p, top);
            return;
        }
    }

    __syncthreads();
    stream_t stream(lds.stream, logits, a.V, top, p.per);
    if (p.k) stream.select(false, p.k);
    if (p.p < 1u << 24) {
        const uint64_t of = p.k ? stream.total([&](uint32_t key, int i) -> uint64_t {
            return stream.kept(key, i) ? weight_of(key, top, p.per) : 0u;
        }) : weight;
        const uint64_t need = share(p.p, of);
        stream.select(true, need ? need : 1);
    }
    const auto amount = [&](uint32_t key, int i) -> uint64_t {
        const float e = e_of(logit_of(key), top, p.per);
        return ((key != 0) & stream.kept(key, i) & (e >= p.min_e)) ? w_of(e) : 0u;
    };
    const uint64_t total = stream.total(amount);
    stream.first_over(amount, share(p.u, total), [&](uint32_t key, int i) {
        a.token[row] = i;
        if (a.logp) a.logp[row] = logp_of(z_of(logit_of(key), top, p.per), total);
    });
}

template <typename T>
aq_status launch_long(aq_ctx *ctx, const sample_args &a) {
    chunk_store c{};
    c.chunks = (a.V + kChunk - 1) / kChunk;
    c.cap = kSlots / c.chunks / 8 * 8;
    const size_t rows = static_cast<size_t>(a.rows < kRowsAtOnce ? a.rows : kRowsAtOnce), n = rows * c.chunks;
    char *at = nullptr;
    const size_t slots = n * c.cap * sizeof(uint2);
    aq_status st = aq_ctx_scratch(ctx, 7, slots + n * 20, reinterpret_cast<void **>(&at));
    if (st != AQ_OK) return st;
    c.slot = reinterpret_cast<uint2 *>(at);
    c.weight = reinterpret_cast<uint64_t *>(at + slots);
    c.top = reinterpret_cast<uint32_t *>(c.weight + n);
    c.count = c.top + n;
    c.whole = reinterpret_cast<int32_t *>(c.count + n);
    for (int64_t row0 = 0; row0 < a.rows; row0 += kRowsAtOnce) {
        const uint32_t now = static_cast<uint32_t>(a.rows - row0 < kRowsAtOnce ? a.rows - row0 : kRowsAtOnce);
        const dim3 grid(static_cast<uint32_t>(c.chunks), now);
        aq_launch_timed(ctx, true, sample_top_kernel<T>, grid, dim3(256), 0u, a, c, row0);
        aq_launch_timed(ctx, true, sample_chunk_kernel<T>, grid, dim3(256), 0u, a, c, row0);
        aq_launch_timed(ctx, true, sample_row_kernel<T>, dim3(now), dim3(1024), 0u, a, c, row0);
    }
    return AQ_OK;
}

template <typename T>
aq_status launch(aq_ctx *ctx, const sample_args &a) {
    const dim3 grid(static_cast<uint32_t>(a.rows));
    const auto in_registers = [&](auto kernel, int waves) {
        aq_launch_timed(ctx, true, kernel, grid, dim3(static_cast<uint32_t>(64 * waves)), 0u, a);
    };
    if (a.V <= 512) in_registers(sample_short_kernel<T, 1, 8>, 1);
    else if (a.V <= 1024) in_registers(sample_short_kernel<T, 2, 8>, 2);
    else if (a.V <= 2048) in_registers(sample_short_kernel<T, 4, 8>, 4);
    else if (a.V <= 4096) in_registers(sample_short_kernel<T, 4, 16>, 4);
    else if (a.V <= 8192) in_registers(sample_short_kernel<T, 8, 16>, 8);
    else if (a.V <= 16384) in_registers(sample_short_kernel<T, 16, 16>, 16);
    else return launch_long<T>(ctx, a);
    return AQ_OK;
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
    const aq_status st = type == AQ_T_F32   ? launch<f32>(ctx, a)
                         : type == AQ_T_F16 ? launch<f16>(ctx, a)
                                            : launch<bf16>(ctx, a);
    if (st != AQ_OK) return st;
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}
