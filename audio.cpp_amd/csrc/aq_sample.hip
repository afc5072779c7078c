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
    // [rows] each; those that the caller left out point to u and have no bit in `given`
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    uint32_t given;
    int32_t *token;
    float *logp;
};

enum : uint32_t { kTemperature = 1, kTopK = 2, kTopP = 4, kMinP = 8 };

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

// (All five loads at once: behind tests of the pointers each would wait for
// the one before.)
__device__ inline row_params params_of(const sample_args &a, int64_t row) {
    const float u = a.u[row], temperature = a.temperature[row], top_p = a.top_p[row], min_p = a.min_p[row];
    const int32_t top_k = a.top_k[row];
    row_params r;
    const float degree = a.given & kTemperature ? temperature : 1.0f;
    const bool greedy = !(degree > 0.0f);
    r.per = greedy ? kLog2e : fminf(kLog2e / degree, 3.4e38f);
    const int32_t k = a.given & kTopK ? top_k : 0;
    r.k = greedy ? 1u : (k > 0) & (k < a.V) ? static_cast<uint32_t>(k) : 0u;
    const float p = a.given & kTopP ? top_p : 1.0f;
    r.p = p < 1.0f ? static_cast<uint32_t>(fmaxf(p, 0.0f) * 0x1p24f) : 1u << 24;
    const float m = a.given & kMinP ? min_p : 0.0f;
    r.min_e = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    r.u = static_cast<uint32_t>(fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f) * 0x1p24f);   // NaN: 0
    return r;
}

// floor(part * total / 2^24) for part <= 2^24 and total < 2^52.
__device__ inline uint64_t share(uint32_t part, uint64_t total) {
    return __umul64hi(static_cast<uint64_t>(part) << 39, total << 1);
}

// log2 of a logit's weight relative to the largest.  (A row whose largest is
// +infinity is mapped to 0 and -infinity first: finite_of.)
__device__ inline float z_of(float l, float top, float per) { return (l - top) * per; }

__device__ inline float e_of(float z) { return __builtin_amdgcn_exp2f(z); }

// To a whole number, downwards; a NaN or a negative number to 0.
__device__ inline uint32_t whole_of(float v) {
    uint32_t r;
    asm("v_cvt_u32_f32 %0, %1" : "=v"(r) : "v"(v));
    return r;
}

__device__ inline uint32_t w_of(float z) { return whole_of(e_of(z) * 0x1p31f); }

__device__ inline bool is_infinite(float top) { return !(top < INFINITY); }

// A logit of a row whose largest is +infinity, the largest being 0 then.
__device__ inline float finite_of(float l) { return l == INFINITY ? 0.0f : -INFINITY; }

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

__device__ inline uint32_t wave_scan(uint32_t v) {
    v += dpp<0x111, 0xF>(v);
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    v += dpp<0x118, 0xF>(v);
    v += dpp<0x142, 0xA>(v);
    return v + dpp<0x143, 0xC>(v);
}

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
// is no element, or one that is never drawn; `w` is the weight.
//
// The filters.  Bins by weight (of count and weight at once: 16 bits and 48
// of a word, 8192 elements of at most 2^31); the bin where the running count
// or weight crosses what is needed holds the end of the kept prefix.  If it
// has at most 64 elements, a wave orders them by comparing all pairs; else it
// is divided again, in bins linear in the key, which tells any two different
// logits apart after at most four times; more than 64 equal ones are counted
// off in index order.  There are two bins a thread: with 256 for 8192 elements
// their atomics meet in the same words and the ordering has dozens of elements.
//
// A block's time is its steps' latency, barriers and the fetch of code that
// runs once, not memory or arithmetic: 12 rows of 1024 fp32 logits 6.4 us, 512
// rows of 2048 bf16 7.6.  So steps that look alike share one loop's code.
constexpr int kCountShift = 48;
constexpr uint64_t kWeightMask = (uint64_t{1} << kCountShift) - 1;

constexpr int bins_of(int waves) { return waves < 2 ? 256 : 128 * waves; }

template <int WAVES>
struct list_lds {
    uint64_t bins[bins_of(WAVES)];
    uint64_t part[WAVES];
    uint32_t part_n[WAVES];
    uint32_t key[2][64], index[2][64], weight[2][64];
    uint32_t count[2], hi[2], lo[2], at, each;
    // What one thread or wave found for all.
    uint32_t bin[2], K, I;
    uint64_t need[2], before, through;
};

template <int WAVES, int E, bool GIVEN = false>   // GIVEN: the elements bring their indices
struct row_list {
    static constexpr int kThreads = 64 * WAVES, kBins = bins_of(WAVES), kPer = kBins / kThreads;
    static constexpr float kBinsPerBit = kBins / 32.0f;   // weights span 31 bits
    list_lds<WAVES> &s;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6));
    uint32_t key[E], w[E], bin[E];
    uint32_t given[GIVEN ? E : 1], base = 0;
    uint32_t K = 1, I = 0xFFFFFFFFu;   // kept: key > K, or key == K and index <= I

    // Clears the bins: a barrier has to follow before filter().
    __device__ explicit row_list(list_lds<WAVES> &lds) : s(lds) {
        clear();
        if (threadIdx.x < 2) {
            s.count[threadIdx.x] = 0;
            s.hi[threadIdx.x] = 0;
            s.lo[threadIdx.x] = 0xFFFFFFFFu;
        }
    }

    __device__ void clear() {
#pragma unroll
        for (int b = 0; b < kPer; ++b) s.bins[threadIdx.x + b * kThreads] = 0;
    }

    __device__ uint32_t place(int e) const {   // in the list
        return static_cast<uint32_t>(((wave * (E / 8) + e / 8) * 64 + lane) * 8 + e % 8);
    }
    __device__ uint32_t index(int e) const { return GIVEN ? given[e] : base + place(e); }

    // No branches in the tests of elements: they are a few comparisons, and
    // ROCm 7.2's compiler has dropped the copy of a 64-bit value that a
    // short-circuit left to one of its paths.
    __device__ bool kept(int e) const { return (key[e] > K) | ((key[e] == K) & (index(e) <= I)); }

    // Element e: its bin is (-z - z0) * scale.
    __device__ void set(int e, float l, float top, float per, float z0, float scale) {
        const float z = z_of(l, top, per);
        w[e] = w_of(z);
        key[e] = w[e] ? key_of(l) : 0;
        bin[e] = min(whole_of((-z - z0) * scale), kBins - 1u);
    }

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

    // After total() of amount(e) summed over each thread's elements: true in
    // the thread of the first element where the running sum in index order
    // exceeds t, with its index and key.
    template <typename A>
    __device__ bool first_over(A &&amount, uint64_t t, uint64_t mine, uint32_t &its_index, uint32_t &its_key) {
        uint64_t before = 0;
        if (WAVES > 1) {
            for (int i = 0; i < wave; ++i) before += s.part[i];
            mine = s.part[wave];
        } else {
            mine = wave_total(mine);
        }
        if (t < before || t >= before + mine) return false;   // not in this wave
        bool found = false;
#pragma unroll
        for (int v = 0; v < E / 8; ++v) {
            uint64_t eight = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) eight += amount(8 * v + i);
            const uint64_t upto = before + wave_scan(eight);
            uint64_t sum = upto - eight;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint64_t next = sum + amount(8 * v + i);
                const bool at = (sum <= t) & (next > t);   // one element of one lane
                its_index = at ? index(8 * v + i) : its_index;
                its_key = at ? key[8 * v + i] : its_key;
                found |= at;
                sum = next;
            }
            before = lane_value(upto, 63);
        }
        return found;
    }

    // Into LDS: the elements that `in` names, up to 64, and the range of the
    // others' keys.  One store of code for all of a thread's elements, taken in
    // turn: code that runs once costs its fetch.
    template <typename P>
    __device__ void gather(int phase, P &&in) {
        uint32_t left = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) left |= in(e) ? 1u << e : 0u;
        while (__ballot(left != 0)) {
            uint32_t k = 0, i = 0, weight = 0;
            const uint32_t lowest = left & (0u - left);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool it = lowest == 1u << e;
                k = it ? key[e] : k;
                i = it ? index(e) : i;
                weight = it ? w[e] : weight;
            }
            if (left) {
                const uint32_t at = atomicAdd(&s.count[phase], 1u);
                if (at < 64) {
                    s.key[phase][at] = k;
                    s.index[phase][at] = i;
                    s.weight[phase][at] = weight;
                } else {
                    atomicMax(&s.hi[phase], k);
                    atomicMin(&s.lo[phase], k);
                }
            }
            left &= left - 1;
        }
    }

    // Puts the end of the kept prefix into bin `chosen`, where `need` of the
    // amounts (1, or the weights) are still to come; returns the weight kept
    // of that bin.  `phase`: 0 and 1, each once after a clear.
    __device__ uint64_t resolve(uint32_t chosen, int phase, bool by_weight, uint64_t need) {
        gather(phase, [&](int e) { return (bin[e] == chosen) & kept(e); });
        __syncthreads();
        const uint32_t n = uniform(s.count[phase]);
        if (n <= 64) return order(phase, n, by_weight, need);
        const uint32_t k = s.key[phase][lane];
        refine(by_weight, need, max(uniform(s.hi[phase]), wave_max(k)), min(uniform(s.lo[phase]), ~wave_max(~k)));
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += ((bin[e] == chosen) & kept(e)) ? w[e] : 0u;
        return total(mine);
    }

    // The end of the kept prefix among the n <= 64 elements of the short
    // list.  Every wave finds it, or where they would share their SIMDs the
    // first one for all.
    __device__ uint64_t order(int phase, uint32_t n, bool by_weight, uint64_t need) {
        uint64_t inside = 0;
        if (WAVES <= 4 || wave == 0) {
            const bool there = static_cast<uint32_t>(lane) < n;
            const uint32_t k = there ? s.key[phase][lane] : 0, at = there ? s.index[phase][lane] : 0;
            const uint32_t weight = there ? s.weight[phase][lane] : 0;
            uint64_t through_w = weight;
            uint32_t through_n = 1;
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t ki = lane_value(k, i), ai = lane_value(at, i), wi = lane_value(weight, i);
                const bool first = (ki > k) | ((ki == k) & (ai < at));
                through_w += first ? wi : 0u;
                through_n += first ? 1u : 0u;
            }
            // The last one kept is the first through which the amount reaches `need`.
            const uint64_t through = by_weight ? through_w : through_n, before = through - (by_weight ? weight : 1u);
            const int last = __builtin_ctzll(__ballot(there & (before < need) & (through >= need)));
            K = lane_value(k, last);
            I = lane_value(at, last);
            inside = lane_value(through_w, last);
        }
        if (WAVES > 4) {
            if (threadIdx.x == 0) {
                s.K = K;
                s.I = I;
                s.through = inside;
            }
            __syncthreads();
            K = uniform(s.K);
            I = uniform(s.I);
            inside = lane_value(s.through, 0);
        }
        return inside;
    }

    // This thread's bins, the largest logits first: the sums of weight and
    // count through the bins of the threads before it, and its own.
    struct bin_sums {
        uint64_t w[kPer], before_w, own_w, all_w;
        uint32_t n[kPer], before_n, own_n, all_n;
    };
    __device__ void scan_bins(bin_sums &b) {
        b.own_w = 0;
        b.own_n = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint64_t v = s.bins[threadIdx.x * kPer + i];
            b.own_w += b.w[i] = v & kWeightMask;
            b.own_n += b.n[i] = static_cast<uint32_t>(v >> kCountShift);
        }
        const uint64_t w = wave_scan(b.own_w);
        const uint32_t n = wave_scan(b.own_n);
        b.before_w = w - b.own_w;
        b.before_n = n - b.own_n;
        b.all_w = lane_value(w, 63);
        b.all_n = lane_value(n, 63);
        if (WAVES > 1) {
            if (lane == 63) {
                s.part[wave] = w;
                s.part_n[wave] = n;
            }
            __syncthreads();
            b.all_w = 0;
            b.all_n = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                b.before_w += i < wave ? s.part[i] : 0;
                b.before_n += i < wave ? s.part_n[i] : 0;
                b.all_w += s.part[i];
                b.all_n += s.part_n[i];
            }
            b.all_w = lane_value(b.all_w, 0);
            b.all_n = uniform(b.all_n);
        }
    }

    // Where the running count (or weight) crosses `need`, which it reaches:
    // the bin, what of `need` is left in it, and the weight before it.
    __device__ void crossing(const bin_sums &b, int phase, bool by_weight, uint64_t &need, uint32_t &bin_at, uint64_t &weight) {
        const uint64_t before = by_weight ? b.before_w : b.before_n, own = by_weight ? b.own_w : b.own_n;
        if ((before < need) & (before + own >= need)) {
            uint64_t sum = before, w_sum = b.before_w;
            uint32_t at = 0;
#pragma unroll
            for (int i = 0; i + 1 < kPer; ++i) {
                const uint64_t next = sum + (by_weight ? b.w[i] : b.n[i]);
                const bool on = (at == static_cast<uint32_t>(i)) & (next < need);
                sum = on ? next : sum;
                w_sum += on ? b.w[i] : 0;
                at += on ? 1u : 0u;
            }
            s.bin[phase] = threadIdx.x * kPer + at;
            s.need[phase] = need - sum;
            s.before = w_sum;
        }
        __syncthreads();
        bin_at = uniform(s.bin[phase]);
        need = lane_value(s.need[phase], 0);
        weight = lane_value(s.before, 0);
    }

    // As resolve(), for more than 64 elements: the kept ones with keys from lo to hi.
    __device__ void refine(bool by_weight, uint64_t need, uint32_t hi, uint32_t lo) {
        constexpr int kBits = 31 - __builtin_clz(static_cast<unsigned>(kBins));
        while (hi != lo) {
            const int shift = max(0, 32 - kBits - __builtin_clz(hi - lo));
            __syncthreads();
            clear();
            if (threadIdx.x == 0) {
                s.count[0] = 0;
                s.hi[0] = 0;
                s.lo[0] = 0xFFFFFFFFu;
            }
            __syncthreads();
            const auto in = [&](int e) { return (key[e] >= lo) & (key[e] <= hi) & kept(e); };
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (in(e))
                    atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[(hi - key[e]) >> shift]),
                              (uint64_t{1} << kCountShift) + w[e]);
            __syncthreads();
            bin_sums b;
            scan_bins(b);
            uint32_t chosen;
            uint64_t unused;
            crossing(b, 0, by_weight, need, chosen, unused);
            gather(0, [&](int e) { return in(e) & ((hi - key[e]) >> shift == chosen); });
            __syncthreads();
            const uint32_t n = uniform(s.count[0]);
            if (n <= 64) {
                order(0, n, by_weight, need);
                return;
            }
            const uint32_t k = s.key[0][lane];
            hi = max(uniform(s.hi[0]), wave_max(k));
            lo = min(uniform(s.lo[0]), ~wave_max(~k));
        }
        // Equal logits: the first of them in index order.
        uint64_t mine = 0, each = 1;
        uint32_t some = 0;
        const uint32_t equal = lo;
        const auto one = [&](int e) { return ((key[e] == equal) & kept(e)) ? 1u : 0u; };
#pragma unroll
        for (int e = 0; e < E; ++e) {
            mine += one(e);
            some = max(some, one(e) ? w[e] : 0u);
        }
        if (some) s.each = some;   // their weight, from whoever has one
        total(mine);
        __syncthreads();
        if (by_weight) each = uniform(s.each);
        uint32_t at = 0, unused = 0;
        if (first_over(one, (need + each - 1) / each - 1, mine, at, unused)) s.at = at;
        __syncthreads();
        K = equal;
        I = uniform(s.at);
    }

    // Top-k (k > 0), then top-p of the weight that leaves (p < 2^24), or
    // until `need` > 0 of the count or weight is reached.
    __device__ uint64_t filter(uint32_t k, uint32_t p, uint64_t need, bool by_weight = true) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (kept(e))
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[bin[e]]),
                          (uint64_t{1} << kCountShift) + w[e]);
        __syncthreads();
        bin_sums b;
        scan_bins(b);
        uint64_t weight = b.all_w;   // kept
        // Phase 0: top-k's end; phase 1: top-p's (or that of `need`).  (The sums
        // of bins behind top-k's end are too large then, but it is crossed
        // before.)  One loop, so that the code is there, and fetched, once.
#pragma unroll 1
        for (int phase = 0; phase < 2; ++phase) {
            uint64_t rest = need;
            if (phase == 0) rest = k;
            else if (p < 1u << 24) rest = max(share(p, weight), uint64_t{1});
            const bool weights = phase && by_weight;
            if (!rest || rest > (weights ? b.all_w : b.all_n)) continue;
            uint32_t chosen = 0;
            uint64_t before = 0;
            crossing(b, phase, weights, rest, chosen, before);
            weight = before + resolve(chosen, phase, weights, rest);
        }
        return weight;
    }

    __device__ uint64_t kept_weight() const {   // this thread's
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += kept(e) ? w[e] : 0u;
        return mine;
    }

    // The weights of what is not kept, or is below min-p, to 0; this thread's sum.
    __device__ uint64_t drop(float min_e, float top, float per) {
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = kept(e) ? w[e] : 0u;
            if (min_e > 0.0f) w[e] = e_of(z_of(logit_of(key[e]), top, per)) >= min_e ? w[e] : 0u;
            mine += w[e];
        }
        return mine;
    }

    // Draws among the weights and writes the outputs: from all of them, or
    // (sum > 0) as a part of a row whose kept weight is `sum`, t into this part.
    __device__ void draw(const sample_args &a, int64_t row, const row_params &r, float top, uint64_t mine, uint64_t sum,
                         uint64_t t) {
        const uint64_t all = total(mine);
        if (!sum) {
            sum = all;
            t = share(r.u, sum);
        }
        uint32_t at = 0, its_key = 0;
        if (!first_over([&](int e) { return w[e]; }, t, mine, at, its_key)) return;
        a.token[row] = static_cast<int32_t>(at);
        if (a.logp) a.logp[row] = logp_of(z_of(logit_of(its_key), top, r.per), sum);
    }
};

// 8 logits of a row, -infinity past the end.
template <typename T>
__device__ inline void load_logits(const typename T::raw *logits, int at, int V, float (&l)[8]) {
    load8<T>(logits, at, V, l, T::store(-INFINITY));
}

// The same in two steps, so that loads can be ahead of what is done with them.
template <typename T>
struct raw8 {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    typedef words any __attribute__((aligned(1)));
    static constexpr int kWords = sizeof(typename T::raw) / 2;   // 16 bytes each
    words w[kWords];
    __device__ void load(const typename T::raw *logits, int at, int V) {
        if (at + 8 <= V) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const any *>(logits + at)[i];
        } else {
            float l[8];
            load_logits<T>(logits, at, V, l);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t bits = bits_of(T::store(l[i]));
                if (kWords == 2) w[i / 4][i % 4] = bits;
                else w[0][i / 2] = i % 2 ? w[0][i / 2] | bits << 16 : bits;
            }
        }
    }
    __device__ void get(float (&l)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (kWords == 2) l[i] = __uint_as_float(w[i / 4][i % 4]);
            else l[i] = T::load(static_cast<typename T::raw>(w[0][i / 2] >> (i % 2 * 16)));
        }
    }
};

__device__ inline uint32_t largest_key(const float (&l)[8]) {
    float top = l[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, l[i]);   // not a NaN, unless there is no other
    return top > -INFINITY ? key_of(top) : 0;
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
    float l[E / 8][8];
    uint32_t top_key = 0;
#pragma unroll
    for (int v = 0; v < E / 8; ++v) load_logits<T>(logits, static_cast<int>(list.place(8 * v)), a.V, l[v]);
    const row_params r = params_of(a, row);
#pragma unroll
    for (int v = 0; v < E / 8; ++v) top_key = max(top_key, largest_key(l[v]));
    top_key = wave_max(top_key);
    if (list.lane == 0) lds.part[list.wave] = top_key;
    __syncthreads();
    if (WAVES > 1) {
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top_key = max(top_key, static_cast<uint32_t>(lds.part[i]));
        top_key = uniform(top_key);
    }
    if (!top_key) {
        if (threadIdx.x == 0) write_empty(a, row);
        return;
    }
    float top = logit_of(top_key);
    if (is_infinite(top)) {
        top = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) l[e / 8][e % 8] = finite_of(l[e / 8][e % 8]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) list.set(e, l[e / 8][e % 8], top, r.per, 0.0f, list.kBinsPerBit);
    if (r.k || r.p < 1u << 24) list.filter(r.k, r.p, 0);
    list.draw(a, row, r, top, list.drop(r.min_e, top, r.per), 0, 0);
}

// Longer rows: chunks of 8192 elements, a block each, in four launches.  (A row
// of 8192 itself takes 7.5 us as above, 20 in these; 1024 of them 29 and 100.
// Twice as many elements a thread do not fit the registers.)
//
//  1. the largest logit of each chunk, and the row's parameters;
//  2. the weights, relative to the row's largest, and their sum over the
//     chunk; for rows with filters also the chunk's count and weight per
//     quarter of a bit of weight, and its candidates: the elements of its
//     largest quarters, in index order, as many whole ones as fit its slots;
//  3. a small block per row.  Without filters it finds the chunk that the draw
//     falls into from the sums, and draws in it.  With filters it works on the
//     candidates down to the least quarter that every chunk has given whole,
//     which hold the kept set unless that is wide;
//  4. where a row may be filtered, a large block per row that is left, if any.
//     A wide set ends in a quarter that the sums tell (top-k's end, then
//     top-p's): its elements are collected from the chunks and decide where,
//     and the sums over what lies above it decide the chunk to draw in.  What
//     is left even then (min-p's end in a wide set, more than 8192 elements in
//     a quarter) streams the row.
//
// 256 rows of 160000 bf16 logits under top-p take 14, 31, 12 and 45 us (82 MB,
// 17 us at a copy's rate): the first reads at 6 TB/s; the second's time is
// vector instructions, some 20 an element; the third's and fourth's the
// latency of one block's steps, the fourth's with the row read again.  One row
// of 131071: 2.5, 6, 9 and 1.  In the first two and in the draw a thread's
// four loads wait for each other (each tests the row's end in its lanes),
// which many blocks a compute unit hide and one row does not.
// Without filters, or with min-p alone, 43 and 13 us.  A row that is streamed
// is read five times or more by its one block: 320 and 147 us where min-p
// ends in a wide nucleus, 428 and 224 where its quarter has more than 8192
// elements, 703 and 384 with top-k too.
constexpr int kChunk = 8192;          // 256 threads, 32 elements each
constexpr int kSlots = 2048;          // candidates of a row: 256 threads, 8 each
constexpr int kWideWaves = 8;         // of a block in the fourth launch: with twice as many its registers spill
constexpr int kGathered = 8192;       // elements of a quarter: 16 for each of its threads
constexpr int kMostChunks = kMaxV / kChunk;
constexpr int kRowsAtOnce = 256;

struct chunk_store {
    uint64_t *bins;     // [rows][chunks][kBinned] count and weight of each quarter, as kCountShift has them
    uint64_t *weight;   // [rows][chunks] sum of weights (of those that min-p leaves, for rows without other filters)
    uint2 *slot;        // [rows][chunks][cap] logit's bits, index
    uint32_t *top;      // [rows][chunks] largest key
    uint32_t *count;    // [rows][chunks] candidates
    int32_t *whole;     // [rows][chunks] the last quarter given whole, -1: none
    uint32_t *left;     // [rows] 1: for the fourth launch
    row_params *params; // [rows]
    int chunks, cap;
};

// The quarter of a bit of weight below the largest, counted from below: 125 for
// the largest itself, 124 for those above -1/4, down to 1 from -31 on; 0: no
// weight (or a NaN).  One fused product and sum, and it does not fall with z.
// Quarter 0 is the largest itself, 124 the last with weights.
constexpr int kQuarters = 125, kBinned = 128;   // bins, two a lane; the last ones stay empty
__device__ inline uint32_t step_of(float z) { return whole_of(__fmaf_rn(z, 4.0f, 125.0f)); }
__device__ inline uint32_t quarter(float z) { return kQuarters - step_of(z); }

// Elements that a wave picks from 2048 of a row, in index order: bit 31 - (8 v +
// e) of `in` is element e of this lane's 8 in vector v, and vector v's come
// before v + 1's.  `to`: the places of each vector's first one of this lane.
// Returns how many the wave has.  (Sums of two vectors in a word: no carry, at
// most 512 each.)
__device__ inline uint32_t places_of(uint32_t in, uint32_t (&to)[4]) {
    const uint32_t own01 = static_cast<uint32_t>(__popc(in >> 24) | __popc(in >> 16 & 255u) << 16);
    const uint32_t own23 = static_cast<uint32_t>(__popc(in >> 8 & 255u) | __popc(in & 255u) << 16);
    const uint32_t to01 = wave_scan(own01), to23 = wave_scan(own23);
    const uint32_t all01 = lane_value(to01, 63), all23 = lane_value(to23, 63);
    const uint32_t n0 = all01 & 0xFFFFu, n1 = n0 + (all01 >> 16), n2 = n1 + (all23 & 0xFFFFu);
    to[0] = (to01 - own01) & 0xFFFFu;
    to[1] = n0 + ((to01 - own01) >> 16);
    to[2] = n1 + ((to23 - own23) & 0xFFFFu);
    to[3] = n2 + ((to23 - own23) >> 16);
    return n2 + (all23 >> 16);
}

// f(place, offset of the element from the wave's first) for each of them.
template <typename F>
__device__ inline void each_picked(uint32_t in, const uint32_t (&to)[4], F &&f) {
    const uint32_t lane8 = (threadIdx.x & 63) * 8;
    uint32_t left = in;
    while (__ballot(left != 0)) {
        if (left) {
            const uint32_t bit = 31u - static_cast<uint32_t>(__builtin_clz(left)), v = 3 - bit / 8;
            const uint32_t before = static_cast<uint32_t>(__popc(in >> bit & (255u >> bit % 8))) - 1;   // own of this vector
            f((v == 0 ? to[0] : v == 1 ? to[1] : v == 2 ? to[2] : to[3]) + before, v * 512 + lane8 + 7 - bit % 8);
            left ^= 1u << bit;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void sample_top_kernel(sample_args a, chunk_store c, int64_t row0) {
    __shared__ uint32_t part[4];
    const int64_t r = blockIdx.y;
    const typename T::raw *logits = static_cast<const typename T::raw *>(a.logits) + (row0 + r) * a.ld;
    const int at = static_cast<int>(blockIdx.x) * kChunk + static_cast<int>(threadIdx.x) * 8;
    float l[4][8];
#pragma unroll
    for (int v = 0; v < 4; ++v) load_logits<T>(logits, at + 2048 * v, a.V, l[v]);
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) top = max(top, largest_key(l[v]));
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x != 0) return;
    c.top[r * c.chunks + blockIdx.x] = max(max(part[0], part[1]), max(part[2], part[3]));
    if (blockIdx.x == 0) c.params[r] = params_of(a, row0 + r);
}

// The largest key of a row from its chunks'; every wave for itself.
__device__ inline uint32_t row_top(const chunk_store &c, int64_t r) {
    uint32_t top = 0;
    for (int i = threadIdx.x & 63; i < c.chunks; i += 64) top = max(top, c.top[r * c.chunks + i]);
    return wave_max(top);
}

template <typename T>
__global__ __launch_bounds__(256) void sample_chunk_kernel(sample_args a, chunk_store c, int64_t row0) {
    // Copies of the bins for every eighth lane, since lanes of one wave often
    // meet in a bin, and a row's length that puts its neighbours into other
    // banks.  256 rows of 160000 bf16 logits: 31 us; with 16 copies 39, for the
    // room that they take, and 45 without the added word.
    constexpr int kCopies = 8;
    __shared__ uint64_t bins[kBinned][kCopies + 1];
    __shared__ uint64_t part[4];
    __shared__ uint32_t counts[4];
    __shared__ int whole;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6));
    const int64_t r = blockIdx.y, row = row0 + r, chunk = r * c.chunks + blockIdx.x;
    const typename T::raw *logits = static_cast<const typename T::raw *>(a.logits) + row * a.ld;
    const int base = static_cast<int>(blockIdx.x) * kChunk + (wave * 256 + lane) * 8;   // four vectors, 512 apart
    float l[4][8];
#pragma unroll
    for (int v = 0; v < 4; ++v) load_logits<T>(logits, base + 512 * v, a.V, l[v]);
    const row_params p = c.params[r];
    const uint32_t top_key = row_top(c, r);
    if (!top_key) return;   // the whole row is empty
    float top = logit_of(top_key);
    if (is_infinite(top)) {
        top = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) l[e / 8][e % 8] = finite_of(l[e / 8][e % 8]);
    }
    const bool filtered = p.k || p.p < 1u << 24;

    uint64_t mine = 0;
    if (!filtered) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const float weight = e_of(z_of(l[e / 8][e % 8], top, p.per));
            mine += whole_of(weight >= p.min_e ? weight * 0x1p31f : 0.0f);
        }
        mine = wave_total(mine);
        if (lane == 0) part[wave] = mine;
        __syncthreads();
        if (threadIdx.x == 0) c.weight[chunk] = part[0] + part[1] + part[2] + part[3];
        return;
    }
    // Vector instructions are what this takes its time for, so what is not for
    // an element is for 32 of them, or left to one wave.
#pragma unroll
    for (int i = 0; i < kBinned * kCopies / 256; ++i) bins[lane + i % 2 * 64][wave * (kCopies / 4) + i / 2] = 0;
    __syncthreads();
    uint32_t step[32];
    char *own = reinterpret_cast<char *>(&bins[0][lane % kCopies]);
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const float z = z_of(l[e / 8][e % 8], top, p.per);
        const uint32_t w = w_of(z);
        step[e] = step_of(z);
        if (step[e])
            atomicAdd(reinterpret_cast<unsigned long long *>(own + __umul24(step[e], sizeof(bins[0]))),
                      (uint64_t{1} << kCountShift) + w);
    }
    __syncthreads();
    if (wave == 0) {
        const int q = 2 * lane;   // and q + 1
        ulonglong2 sum = make_ulonglong2(0, 0);
        if (q < kQuarters) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                sum.x += bins[kQuarters - q][(i + lane) % kCopies];
                sum.y += q + 1 < kQuarters ? bins[kQuarters - q - 1][(i + lane) % kCopies] : 0;
            }
        }
        *reinterpret_cast<ulonglong2 *>(c.bins + chunk * kBinned + q) = sum;
        const uint64_t all = wave_total((sum.x & kWeightMask) + (sum.y & kWeightMask));
        const uint32_t n1 = static_cast<uint32_t>(sum.y >> kCountShift);
        const uint32_t upto = wave_scan(static_cast<uint32_t>(sum.x >> kCountShift) + n1);   // through q + 1; it does not fall
        const uint32_t cap = static_cast<uint32_t>(c.cap);
        const int last = __popcll(__ballot(upto <= cap)) + __popcll(__ballot(upto - n1 <= cap)) - 1;
        if (lane == 0) {
            c.weight[chunk] = all;
            c.whole[chunk] = last;
            whole = last;
        }
    }
    __syncthreads();
    const uint32_t least = static_cast<uint32_t>(max(kQuarters - whole, 1));   // step of the last quarter given

    // The candidates.
    uint32_t in = 0, to[4];
#pragma unroll
    for (int e = 0; e < 32; ++e) in = in + in + (step[e] >= least ? 1u : 0u);
    const uint32_t n = places_of(in, to);
    if (lane == 0) counts[wave] = n;
    __syncthreads();
    uint2 *slot = c.slot + chunk * c.cap;
    for (int i = 0; i < wave; ++i) slot += counts[i];
    const uint32_t index0 = blockIdx.x * kChunk + static_cast<uint32_t>(wave) * 2048;
    each_picked(in, to, [&](uint32_t at, uint32_t offset) {
        slot[at] = make_uint2(bits_of(static_cast<float>(T::load(logits[index0 + offset]))), index0 + offset);
    });
    if (threadIdx.x == 0) c.count[chunk] = counts[0] + counts[1] + counts[2] + counts[3];
}

// A row streamed from memory by a block of 8 waves: wave w has the run of
// whole vectors of 512 elements from w * run on, so that the waves' sums in
// order give index order.
template <typename T>
struct row_stream {
    using raw = typename T::raw;
    struct lds {
        uint64_t bins[2048];
        uint64_t part[kWideWaves];
        uint32_t key[64], index[64], weight[64];
        uint32_t count, hi, lo, chosen;
        uint64_t before;
    };
    lds &s;
    const raw *logits;
    const int V;
    const float top, per;
    const bool infinite;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6));
    const int run, begin, end;
    uint32_t K = 1, I = 0xFFFFFFFFu;

    __device__ row_stream(lds &l, const raw *p, int n, float t, float f, bool inf)
        : s(l), logits(p), V(n), top(t), per(f), infinite(inf), run((n + 512 * kWideWaves - 1) / (512 * kWideWaves) * 512), begin(min(wave * run, n)),
          end(min(begin + run, n)) {}

    __device__ bool kept(uint32_t key, int i) const {
        return (key > K) | ((key == K) & (static_cast<uint32_t>(i) <= I));
    }

    __device__ void load(int i, float (&l)[8]) {
        load_logits<T>(logits, i + lane * 8, V, l);
        if (infinite) {
#pragma unroll
            for (int e = 0; e < 8; ++e) l[e] = finite_of(l[e]);
        }
    }

    // f(logit, index) of every element of this wave's run.
    template <typename F>
    __device__ void each(F &&f) {
        for (int i = begin; i < end; i += 512) {
            float l[8];
            load(i, l);
#pragma unroll
            for (int e = 0; e < 8; ++e) f(l[e], i + lane * 8 + e);
        }
    }

    // The sum over the block of amount(logit, index); each wave's in s.part.
    template <typename A>
    __device__ uint64_t total(A &&amount) {
        uint64_t mine = 0;
        each([&](float l, int i) { mine += amount(l, i); });
        mine = wave_total(mine);
        __syncthreads();
        if (lane == 0) s.part[wave] = mine;
        __syncthreads();
        return wave_total(lane < kWideWaves ? s.part[lane] : 0);
    }

    // After total(amount): true in the thread of the first element where the
    // running sum exceeds t, with its index and logit.
    template <typename A>
    __device__ bool first_over(A &&amount, uint64_t t, int &its_index, float &its_logit) {
        const uint64_t sums = wave_scan(lane < kWideWaves ? s.part[lane] : 0);
        uint64_t before = wave ? lane_value(sums, wave - 1) : 0;
        if (t < before || t >= lane_value(sums, wave)) return false;
        for (int i = begin; i < end; i += 512) {
            float l[8];
            load(i, l);
            uint64_t eight = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) eight += amount(l[e], i + lane * 8 + e);
            const uint64_t upto = before + wave_scan(eight);
            before = lane_value(upto, 63);
            if (before <= t) continue;
            uint64_t sum = upto - eight;
            bool found = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint64_t next = sum + amount(l[e], i + lane * 8 + e);
                const bool at = (sum <= t) & (next > t);
                its_index = at ? i + lane * 8 + e : its_index;
                its_logit = at ? l[e] : its_logit;
                found |= at;
                sum = next;
            }
            return found;
        }
        return false;
    }

    // Narrows the kept set to its shortest prefix whose amounts (1, or the
    // weights) reach `need`, as row_list does, with 2048 bins (the first 1/64
    // of a bit wide); leaves it if they do not.
    __device__ void select(bool by_weight, uint64_t need) {
        uint32_t hi = 0xFFFFFFFFu, lo = 1;
        int shift = -1;
        const auto bin_of = [&](uint32_t key, float z) {
            return shift < 0 ? min(whole_of(z * -64.0f), 2047u) : (hi - key) >> shift;
        };
        for (;;) {
            __syncthreads();
            for (int b = threadIdx.x; b < 2048; b += 64 * kWideWaves) s.bins[b] = 0;
            if (threadIdx.x == 0) {
                s.count = 0;
                s.hi = 0;
                s.lo = 0xFFFFFFFFu;
                s.chosen = 0xFFFFFFFFu;
            }
            __syncthreads();
            each([&](float l, int i) {
                const float z = z_of(l, top, per);
                const uint32_t w = w_of(z), key = key_of(l);
                if ((w != 0) & (key >= lo) & (key <= hi) & kept(key, i))
                    atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[bin_of(key, z)]), by_weight ? w : 1u);
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
            each([&](float l, int i) {
                const float z = z_of(l, top, per);
                const uint32_t w = w_of(z), key = key_of(l);
                if ((w != 0) & (key >= lo) & (key <= hi) & kept(key, i) & (bin_of(key, z) == chosen)) {
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
        const auto one = [&](float l, int i) -> uint64_t {
            const uint32_t key = key_of(l);
            return ((key == equal) & kept(key, i)) ? 1u : 0u;
        };
        total(one);
        int at = 0;
        float unused = 0.0f;
        if (first_over(one, count - 1, at, unused)) s.chosen = static_cast<uint32_t>(at);
        __syncthreads();
        K = equal;
        I = uniform(s.chosen);
    }
};

// The weight and count of a row's quarters through 2 * lane and the next, from
// its chunks; every wave of a block takes part.
struct quarter_lds {
    uint64_t weight[kBinned];
    uint32_t count[kBinned];
};
struct quarter_sums {
    uint64_t w_even, w_odd;
    uint32_t n_even, n_odd;
    __device__ inline __attribute__((always_inline)) quarter_sums(const chunk_store &c, int64_t chunk0, quarter_lds &s) {
        const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6)), waves = blockDim.x >> 6;
        if (threadIdx.x < kBinned) {
            s.weight[threadIdx.x] = 0;
            s.count[threadIdx.x] = 0;
        }
        __syncthreads();
        uint64_t w0 = 0, w1 = 0;
        uint32_t n0 = 0, n1 = 0;
        for (int i = wave; i < c.chunks; i += waves) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(c.bins + (chunk0 + i) * kBinned + 2 * lane);
            w0 += v.x & kWeightMask;
            w1 += v.y & kWeightMask;
            n0 += static_cast<uint32_t>(v.x >> kCountShift);
            n1 += static_cast<uint32_t>(v.y >> kCountShift);
        }
        if (n0 + n1) {
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.weight[2 * lane]), w0);
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.weight[2 * lane + 1]), w1);
            atomicAdd(&s.count[2 * lane], n0);
            atomicAdd(&s.count[2 * lane + 1], n1);
        }
        __syncthreads();
        w1 = s.weight[2 * lane + 1];
        n1 = s.count[2 * lane + 1];
        w_odd = wave_scan(s.weight[2 * lane] + w1);
        n_odd = wave_scan(s.count[2 * lane] + n1);
        w_even = w_odd - w1;
        n_even = n_odd - n1;
    }
    // Through quarter b.
    __device__ uint64_t weight(int b) const {
        const uint64_t even = lane_value(w_even, b >> 1), odd = lane_value(w_odd, b >> 1);
        return b & 1 ? odd : even;
    }
    __device__ uint32_t count(int b) const {
        const uint32_t even = lane_value(n_even, b >> 1), odd = lane_value(n_odd, b >> 1);
        return b & 1 ? odd : even;
    }
};

// Where a wide set ends by count (top-k) or by weight (top-p of `weight`):
// the quarter, what is needed of it, and whether it can be worked on, with
// nothing kept that min-p may drop.
struct wide_end {
    uint64_t rest = 0;
    uint32_t quarter = 0, count = 0;
    bool usable = false;
    __device__ inline __attribute__((always_inline)) wide_end(const row_params &p, uint64_t weight, const quarter_sums &sums, const quarter_lds &s, bool by_weight) {
        rest = by_weight ? max(share(p.p, weight), uint64_t{1}) : p.k;
        const uint64_t over0 = by_weight ? __ballot(sums.w_even >= rest) : __ballot(sums.n_even >= rest);
        const uint64_t over1 = by_weight ? __ballot(sums.w_odd >= rest) : __ballot(sums.n_odd >= rest);
        if (!over1) return;
        const int in1 = 2 * __builtin_ctzll(over1) + 1, in0 = over0 ? 2 * __builtin_ctzll(over0) : in1;
        const int b = min(in0, in1);
        quarter = static_cast<uint32_t>(b);
        count = uniform(s.count[b]);
        usable = (count <= kGathered) &
                 !((p.min_e > 0.0f) & (e_of(-0.25f * static_cast<float>(b)) <= p.min_e * 1.0001f));
        if (b) rest -= by_weight ? sums.weight(b - 1) : sums.count(b - 1);
    }
};

// The draw in the chunk where the running weight over `sums` (device or LDS,
// one per chunk) exceeds share(u, weight), among what K and I keep.
template <typename T, int WAVES, int E>
__device__ inline void draw_in_chunk(const sample_args &a, const chunk_store &c, int64_t row, const row_params &p,
                                     const uint64_t *sums, uint64_t weight, float top, bool infinite, uint32_t K,
                                     uint32_t I, list_lds<WAVES> &lds) {
    static_assert(64 * WAVES * E == kChunk, "");
    row_list<WAVES, E> list(lds);
    // Every wave finds the chunk for itself.
    const uint64_t t = share(p.u, weight);
    uint64_t before = 0;
    int chunk = 0;
    for (int i = 0; i < c.chunks; i += 64) {
        const uint64_t v = i + list.lane < c.chunks ? sums[i + list.lane] : 0;
        const uint64_t upto = before + wave_scan(v);
        const uint64_t over = __ballot(upto > t);
        if (over) {
            const int owner = __builtin_ctzll(over);
            chunk = i + owner;
            before = lane_value(upto - v, owner);
            break;
        }
        before = lane_value(upto, 63);
    }
    const int base = chunk * kChunk;
    const typename T::raw *logits = static_cast<const typename T::raw *>(a.logits) + row * a.ld;
#pragma unroll
    for (int v = 0; v < E / 8; ++v) {
        float l[8];
        load_logits<T>(logits, base + static_cast<int>(list.place(8 * v)), a.V, l);
#pragma unroll
        for (int e = 0; e < 8; ++e) list.set(8 * v + e, infinite ? finite_of(l[e]) : l[e], top, p.per, 0.0f, list.kBinsPerBit);
    }
    list.base = static_cast<uint32_t>(base);
    list.K = K;
    list.I = I;
    list.draw(a, row, p, top, list.drop(p.min_e, top, p.per), weight, t - before);
}

template <typename T>
__global__ __launch_bounds__(256) void sample_row_kernel(sample_args a, chunk_store c, int64_t row0) {
    __shared__ list_lds<4> lds;
    __shared__ quarter_lds quarters;
    const int lane = threadIdx.x & 63;
    const int64_t r = blockIdx.x, row = row0 + r, chunk0 = r * c.chunks;
    const row_params p = c.params[r];
    const uint32_t top_key = row_top(c, r);
    if (threadIdx.x == 0) c.left[r] = 0;
    if (!top_key) {
        if (threadIdx.x == 0) write_empty(a, row);
        return;
    }
    const bool infinite = is_infinite(logit_of(top_key));
    const float top = infinite ? 0.0f : logit_of(top_key);
    const bool filtered = p.k || p.p < 1u << 24;

    // The row's weight, and for filtered rows the least quarter given whole.
    int whole = kBinned - 1;
    uint64_t weight = 0;
    for (int i = lane; i < c.chunks; i += 64) {
        weight += c.weight[chunk0 + i];
        if (filtered) whole = min(whole, c.whole[chunk0 + i]);
    }
    weight = wave_total(weight);
    whole = kBinned - 1 - static_cast<int>(wave_max(static_cast<uint32_t>(kBinned - 1 - whole)));
    if (!filtered) {
        draw_in_chunk<T, 4, 32>(a, c, row, p, c.weight + chunk0, weight, top, infinite, 1, 0xFFFFFFFFu, lds);
        return;
    }

    // The candidates.
    row_list<4, 8, true> list(lds);
    const int place = static_cast<int>(list.place(0)), chunk = place / c.cap, first = place % c.cap;
    const int n = chunk < c.chunks ? static_cast<int>(c.count[chunk0 + chunk]) - first : 0;
    const uint4 *slot = reinterpret_cast<const uint4 *>(c.slot + (chunk0 + min(chunk, c.chunks - 1)) * c.cap + first);
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = slot[i];
    // Do they hold the kept set?  They do if top-k ends in them; without
    // top-k, if top-p does, or if min-p lets nothing below them through.
    const quarter_sums sums(c, chunk0, quarters);
    const uint64_t need = p.k ? p.k : max(share(p.p, weight), uint64_t{1});
    bool enough = whole >= kQuarters - 1;
    if (whole >= 0) enough |= (p.k ? sums.count(whole) : sums.weight(whole)) >= need;
    enough |= !p.k && e_of(-0.25f * static_cast<float>(whole)) * 1.0001f < p.min_e;
    if (!enough) {
        if (threadIdx.x == 0) c.left[r] = 1;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float l = __uint_as_float(e % 2 ? v[e / 2].z : v[e / 2].x);
        if (infinite) l = finite_of(l);
        l = e < n ? l : -INFINITY;
        list.set(e, l, top, p.per, 0.0f, list.kBinsPerBit);
        list.given[e] = e % 2 ? v[e / 2].w : v[e / 2].y;
        if (static_cast<int>(quarter(z_of(l, top, p.per))) > whole) list.key[e] = 0;
    }
    list.filter(p.k, p.k ? p.p : 1u << 24, p.k ? 0 : need);
    list.draw(a, row, p, top, list.drop(p.min_e, top, p.per), 0, 0);
}

template <typename T>
struct wide_lds {
    list_lds<kWideWaves> list;
    uint64_t sums[kMostChunks];   // kept weight of each chunk
    union {
        typename row_stream<T>::lds stream;
        struct {
            uint32_t slot[kGathered];   // indices
            uint32_t offset[kMostChunks];
            quarter_lds quarters;
        } wide;
    };
};

template <typename T>
__global__ __launch_bounds__(64 * kWideWaves) void sample_wide_kernel(sample_args a, chunk_store c, int64_t row0) {
    __shared__ wide_lds<T> s;
    const int64_t r = blockIdx.x;
    if (!c.left[r]) return;
    using raw = typename T::raw;
    const int lane = threadIdx.x & 63, wave = static_cast<int>(uniform(threadIdx.x >> 6));
    const int64_t row = row0 + r, chunk0 = r * c.chunks;
    const raw *logits = static_cast<const raw *>(a.logits) + row * a.ld;
    const row_params p = c.params[r];
    const uint32_t top_key = row_top(c, r);
    const bool infinite = is_infinite(logit_of(top_key));
    const float top = infinite ? 0.0f : logit_of(top_key);

    uint64_t weight = 0;
    for (int i = lane; i < c.chunks; i += 64) {
        const uint64_t w = c.weight[chunk0 + i];
        weight += w;
        if (wave == 0) s.sums[i] = w;
    }
    weight = wave_total(weight);
    const quarter_sums sums(c, chunk0, s.wide.quarters);
    uint32_t K = 1, I = 0xFFFFFFFFu;
    {
        // A wide set.  Phase 0: top-k's end; phase 1: top-p's.  (Where the sums
        // cross, so there is one: both are at most the row's.)
        bool done = true;
#pragma unroll 1
        for (int phase = 0; phase < 2; ++phase) {
            const bool by_weight = phase != 0;
            if (by_weight ? p.p >= 1u << 24 : !p.k) continue;
            if (!by_weight && p.k > sums.count(kQuarters - 1)) {   // top-k leaves everything, and the sums are of everything
                done = !(p.min_e > 0.0f);
                if (!done) break;
                continue;
            }
            const wide_end ends(p, weight, sums, s.wide.quarters, by_weight);
            done = ends.usable;
            if (!done) break;
            const uint32_t b = ends.quarter, n_all = ends.count;
            const uint64_t rest = ends.rest;
            auto &wide = s.wide;
            const uint64_t above = b ? sums.weight(static_cast<int>(b) - 1) : 0;
            // Each chunk's weight above the quarter, and where its elements of it go.
            for (int i = wave; i < c.chunks; i += kWideWaves) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(c.bins + (chunk0 + i) * kBinned + 2 * lane);
                const uint32_t q = 2 * static_cast<uint32_t>(lane);
                const uint64_t sum = wave_total((q < b ? v.x & kWeightMask : 0) + (q + 1 < b ? v.y & kWeightMask : 0));
                if (lane == 0) s.sums[i] = sum;
                if (q == (b & ~1u)) wide.offset[i] = static_cast<uint32_t>((b & 1 ? v.y : v.x) >> kCountShift);
            }
            __syncthreads();
            if (wave == 0) {
                uint32_t before = 0;
                for (int i = 0; i < c.chunks; i += 64) {
                    const uint32_t v = i + lane < c.chunks ? wide.offset[i + lane] : 0;
                    const uint32_t through = before + wave_scan(v);
                    if (i + lane < c.chunks) wide.offset[i + lane] = through - v;
                    before = lane_value(through, 63);
                }
            }
            __syncthreads();
            for (int i = wave; i < c.chunks; i += kWideWaves) {
                uint32_t at = uniform(wide.offset[i]);
                const uint32_t end = i + 1 < c.chunks ? uniform(wide.offset[i + 1]) : n_all;
                raw8<T> ahead[4];
                const auto load4 = [&](int v0) {
#pragma unroll
                    for (int v = 0; v < 4; ++v) ahead[v].load(logits, i * kChunk + (v0 + v) * 512 + lane * 8, a.V);
                };
                load4(0);
                for (int v0 = 0; v0 < kChunk / 512 && at < end; v0 += 4) {
                    float l[4][8];
#pragma unroll
                    for (int v = 0; v < 4; ++v) ahead[v].get(l[v]);
                    if (v0 + 4 < kChunk / 512) load4(v0 + 4);
                    if (infinite) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) l[e / 8][e % 8] = finite_of(l[e / 8][e % 8]);
                    }
                    uint32_t in = 0;   // 8 bits a vector from the highest down
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        in = in + in + (step_of(z_of(l[e / 8][e % 8], top, p.per)) == kQuarters - b ? 1u : 0u);
                    uint32_t to[4];
                    const uint32_t n = places_of(in, to);
                    const uint32_t index0 = static_cast<uint32_t>(i * kChunk + v0 * 512);
                    each_picked(in, to, [&](uint32_t place, uint32_t offset) { wide.slot[at + place] = index0 + offset; });
                    at += n;
                }
            }
            __syncthreads();
            row_list<kWideWaves, 16, true> part(s.list);
            __syncthreads();
            float l[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                part.given[e] = wide.slot[min(part.place(e), n_all - 1)];
                l[e] = T::load(logits[part.given[e]]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (infinite) l[e] = finite_of(l[e]);
                l[e] = part.place(e) < n_all ? l[e] : -INFINITY;
                // the bins over this quarter's part of z: -b/4 <= z < (1 - b)/4
                part.set(e, l[e], top, p.per, 0.25f * (static_cast<float>(b) - 1.0f), 128.0f * part.kBinsPerBit);
            }
            part.K = K;
            part.I = I;
            weight = above + part.filter(0, 1u << 24, rest, by_weight);
            K = part.K;
            I = part.I;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (part.kept(e))
                    atomicAdd(reinterpret_cast<unsigned long long *>(&s.sums[part.given[e] / kChunk]), part.w[e]);
            __syncthreads();
        }
        if (!done) {
            __syncthreads();
            row_stream<T> whole_row(s.stream, logits, a.V, top, p.per, infinite);
            uint64_t total = 0;
            float min_e = 0.0f;
            const auto amount = [&](float l, int i) -> uint64_t {
                const float e = e_of(z_of(l, top, p.per));
                return (whole_row.kept(key_of(l), i) & (e >= min_e)) ? whole_of(e * 0x1p31f) : 0u;
            };
#pragma unroll 1
            for (int phase = 0; phase < 3; ++phase) {   // top-k, top-p, the draw
                if (phase == 2) min_e = p.min_e;
                if (phase) total = whole_row.total(amount);
                const uint64_t rest = phase == 0 ? p.k : phase == 1 && p.p < 1u << 24 ? max(share(p.p, total), uint64_t{1}) : 0;
                if (rest) whole_row.select(phase != 0, rest);
            }
            int at = 0;
            float its = 0.0f;
            if (!whole_row.first_over(amount, share(p.u, total), at, its)) return;
            a.token[row] = at;
            if (a.logp) a.logp[row] = logp_of(z_of(its, top, p.per), total);
            return;
        }
    }

    __syncthreads();
    draw_in_chunk<T, kWideWaves, 16>(a, c, row, p, s.sums, weight, top, infinite, K, I, s.list);
}

template <typename T>
aq_status launch_long(aq_ctx *ctx, const sample_args &a) {
    chunk_store c{};
    c.chunks = (a.V + kChunk - 1) / kChunk;
    c.cap = kSlots / c.chunks / 8 * 8;
    const size_t rows = static_cast<size_t>(a.rows < kRowsAtOnce ? a.rows : kRowsAtOnce), n = rows * c.chunks;
    char *at = nullptr;
    aq_status st = aq_ctx_scratch(ctx, 7, n * (kBinned * 8 + 8 + c.cap * 8 + 12) + rows * (4 + sizeof(row_params)), reinterpret_cast<void **>(&at));
    if (st != AQ_OK) return st;
    c.bins = reinterpret_cast<uint64_t *>(at);
    c.weight = c.bins + n * kBinned;
    c.slot = reinterpret_cast<uint2 *>(c.weight + n);
    c.top = reinterpret_cast<uint32_t *>(c.slot + n * c.cap);
    c.count = c.top + n;
    c.whole = reinterpret_cast<int32_t *>(c.count + n);
    c.left = c.count + 2 * n;
    c.params = reinterpret_cast<row_params *>(c.left + rows);
    for (int64_t row0 = 0; row0 < a.rows; row0 += kRowsAtOnce) {
        const uint32_t now = static_cast<uint32_t>(a.rows - row0 < kRowsAtOnce ? a.rows - row0 : kRowsAtOnce);
        const dim3 grid(static_cast<uint32_t>(c.chunks), now);
        aq_launch_timed(ctx, true, sample_top_kernel<T>, grid, dim3(256), 0u, a, c, row0);
        aq_launch_timed(ctx, true, sample_chunk_kernel<T>, grid, dim3(256), 0u, a, c, row0);
        aq_launch_timed(ctx, true, sample_row_kernel<T>, dim3(now), dim3(256), 0u, a, c, row0);
        if (a.given & (kTemperature | kTopK | kTopP))   // a temperature of 0 is a top-k of 1
            aq_launch_timed(ctx, true, sample_wide_kernel<T>, dim3(now), dim3(64 * kWideWaves), 0u, a, c, row0);
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
    else if (a.V <= 4096) in_registers(sample_short_kernel<T, 8, 8>, 8);
    else if (a.V <= 8192) in_registers(sample_short_kernel<T, 8, 16>, 8);
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
    const sample_args a{logits,
                        ld,
                        rows,
                        static_cast<int>(V),
                        u,
                        temperature ? temperature : u,
                        top_p ? top_p : u,
                        min_p ? min_p : u,
                        top_k ? top_k : reinterpret_cast<const int32_t *>(u),
                        (temperature ? kTemperature : 0u) | (top_k ? kTopK : 0u) | (top_p ? kTopP : 0u) | (min_p ? kMinP : 0u),
                        token,
                        logp};
    const aq_status st = type == AQ_T_F32   ? launch<f32>(ctx, a)
                         : type == AQ_T_F16 ? launch<f16>(ctx, a)
                                            : launch<bf16>(ctx, a);
    if (st != AQ_OK) return st;
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}
