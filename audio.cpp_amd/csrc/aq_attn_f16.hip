// Attention for f16 elements.
#include "aq_attn_kernels.hpp"

namespace aq_attn_impl {
aq_status launch_f16(aq_ctx *ctx, const args &a) { return launch<aq_types::f16>(ctx, a); }
}  // namespace aq_attn_impl
