// Attention for bf16 elements.
#include "aq_attn_kernels.hpp"

namespace aq_attn_impl {
aq_status launch_bf16(aq_ctx *ctx, const args &a) { return launch<aq_types::bf16>(ctx, a); }
}  // namespace aq_attn_impl
