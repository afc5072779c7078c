// Element types of the operators that take more than fp32 (aq_dtype): the
// conversions to and from fp32, and 8-element row loads and stores that need
// no more than the element's own alignment (gfx950 runs with unaligned
// access mode on, so a 16-byte access at any element is one instruction).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>

#include "aq_mi355x.h"

namespace aq_types {

typedef float float2v __attribute__((ext_vector_type(2)));

// Each type: its bits `raw`, both conversions (to the nearest, ties to even;
// NaN stays NaN), and a pair's conversion, which is one instruction.
struct f16 {
    using raw = uint16_t;
    typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
    static __device__ inline float load(raw v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
    static __device__ inline raw store(float v) { return __builtin_bit_cast(raw, static_cast<_Float16>(v)); }
    static __device__ inline void store2(raw *to, float a, float b) {
        const pair_t p = __builtin_convertvector((float2v{a, b}), pair_t);
        std::memcpy(to, &p, sizeof(p));
    }
};

struct bf16 {
    using raw = uint16_t;
    typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
    static __device__ inline float load(raw v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
    static __device__ inline raw store(float v) { return __builtin_bit_cast(raw, static_cast<__bf16>(v)); }
    static __device__ inline void store2(raw *to, float a, float b) {
        const pair_t p = __builtin_convertvector((float2v{a, b}), pair_t);
        std::memcpy(to, &p, sizeof(p));
    }
};

struct f32 {
    using raw = float;
    static __device__ inline float load(raw v) { return v; }
    static __device__ inline raw store(float v) { return v; }
    static __device__ inline void store2(raw *to, float a, float b) {
        to[0] = a;
        to[1] = b;
    }
};

__device__ inline uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ inline uint32_t bits_of(uint16_t v) { return v; }
__device__ inline uint32_t bits_of(uint8_t v) { return v; }

// v[0..7] = p[at..at+7], with `fill` from column `end` on.
template <typename T>
__device__ inline void load8(const typename T::raw *p, int64_t at, int64_t end, float (&v)[8],
                             typename T::raw fill = typename T::raw(0)) {
    typename T::raw r[8];
    if (at + 8 <= end) {
        std::memcpy(r, p + at, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = at + i < end ? p[at + i] : fill;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = T::load(r[i]);
}

// p[at..at+7] = v[0..7], up to column `end`.
template <typename T>
__device__ inline void store8(typename T::raw *p, int64_t at, int64_t end, const float (&v)[8]) {
    typename T::raw r[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) T::store2(r + i, v[i], v[i + 1]);
    if (at + 8 <= end) {
        std::memcpy(p + at, r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < end) p[at + i] = r[i];
    }
}

}  // namespace aq_types
