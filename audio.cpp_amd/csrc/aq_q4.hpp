// Arguments of the product with 4-bit weights, and its launch per type of x.
#pragma once
#include "aq_internal.hpp"

namespace aq_q4_impl {

struct args {
    const uint8_t *codes;    // [tiles][kblocks][64 lanes][16 B]
    const uint16_t *scale;   // [tiles][kblocks][128 / group][16] f16
    const uint8_t *zero;     // like scale, or null: 8
    const float *bias;       // [N] or null
    const void *x;
    const float *x_scale;    // [M, x_groups], 8-bit x
    const float *x_sum;      // of a packed x
    void *y;
    int64_t x_ld, y_ld;
    int M, N, K, tiles, kblocks, group, x_group, x_groups, y_type;
};

aq_status launch_f32(aq_ctx *ctx, const args &a);
aq_status launch_f16(aq_ctx *ctx, const args &a);
aq_status launch_bf16(aq_ctx *ctx, const args &a);
aq_status launch_i8(aq_ctx *ctx, const args &a);
aq_status launch_e4m3(aq_ctx *ctx, const args &a);

}  // namespace aq_q4_impl
