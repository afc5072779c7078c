// Attention for f16 elements.
#include "aq_attn_kernels.hpp"

namespace aq_attn_impl {
aq_status launch_rows_f16(aq_ctx *ctx, const args &a) { return launch_rows<aq_types::f16>(ctx, a); }
aq_status launch_keys_f16(aq_ctx *ctx, const args &a) { return launch_keys<aq_types::f16>(ctx, a); }
}  // namespace aq_attn_impl
