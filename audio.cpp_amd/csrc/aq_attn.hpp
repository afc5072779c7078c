// Arguments of the attention kernels, and their launches per element type.
#pragma once
#include "aq_internal.hpp"

namespace aq_attn_impl {

// Which keys a launch walks: the shared prefix's, a stream's own, or the
// prefix's and then the stream's own.
enum walk : int { kPrefix = 1, kOwn = 2, kBoth = 3 };

struct strides {
    int64_t batch, row, head;   // elements
};

// A set of blocks: rows of all streams over the prefix, or of each stream over
// its own keys, or over both.
struct job {
    int walk;
    int many;      // 128 rows a block, whose waves share the keys; or 32, whose waves split them
    int tiles;     // row tiles: of a stream, or of all streams' rows for the prefix alone
    int splits;    // parts of the keys, by blocks
    int part;      // the first of them in `sums`
    int blocks;
};

struct args {
    const void *q, *pk, *pv, *k, *v;   // pk, pv: the shared prefix (no batch)
    void *out;
    strides sq, spk, spv, sk, sv, so;
    const int32_t *q_len, *kv_len;   // [B] or null: T, S
    const uint8_t *mask;             // [B, S] or null
    int64_t mask_ld;
    float c;       // scale * log2(e)
    int B, T, S, P, H, Hkv, G, D;
    int causal;    // own keys up to the row's own
    int direct;    // rows of keys and values start and end at 16 bytes, and any row is a whole number of such pieces
    job jobs[2];   // of the launch; the second may be empty
    // Parts that another launch joins (null: the launch writes `out`): sums
    // [part][row][D] and their references (scores) and weights [part][row][2],
    // row = (b T + t) H + h.
    float *sums, *ml;
    int64_t rows;   // B T H
};

// Whether a reference, given as the score that it is c times, is so large that
// its rounding (by up to 2^-25 of it) is not small in an exponent.  Scores of
// that size have been rounded by as much themselves.
__device__ inline bool is_far(float score, float c) { return __builtin_fabsf(score * c) > 0x1p16f && score > -INFINITY; }

// 2^(c (score - top)), what sums with one reference are multiplied by beside
// those with a larger one; 0 for sums of nothing.
__device__ inline float weight_of(float score, float top, float c) {
    const float near = score * c - (top == -INFINITY ? 0.0f : top * c), far = (score - top) * c;
    return __builtin_amdgcn_exp2f(is_far(top, c) ? far : near);
}

aq_status launch_f32(aq_ctx *ctx, const args &a);
aq_status launch_f16(aq_ctx *ctx, const args &a);
aq_status launch_bf16(aq_ctx *ctx, const args &a);

}  // namespace aq_attn_impl
