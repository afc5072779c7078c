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
    int direct;    // rows of keys and values start and end at 16 bytes
    // Work of a launch.
    int walk;
    int splits;    // parts of the keys, by blocks
    int tiles;     // row tiles: of a stream, or of all streams' rows for the prefix alone
    // Parts that another launch joins (null: the launch writes `out`): sums
    // [part][row][D] and their largest scores and weights [part][row][2], row
    // = (b T + t) H + h; this launch's parts start at `part`.
    float *sums, *ml;
    int part;
    int64_t rows;   // B T H
};

// The launches: many rows (128 a block, its waves share the keys) and few
// rows (32 a block, its waves share the rows and split the keys).
aq_status launch_rows_f32(aq_ctx *ctx, const args &a);
aq_status launch_rows_f16(aq_ctx *ctx, const args &a);
aq_status launch_rows_bf16(aq_ctx *ctx, const args &a);
aq_status launch_keys_f32(aq_ctx *ctx, const args &a);
aq_status launch_keys_f16(aq_ctx *ctx, const args &a);
aq_status launch_keys_bf16(aq_ctx *ctx, const args &a);

}  // namespace aq_attn_impl
