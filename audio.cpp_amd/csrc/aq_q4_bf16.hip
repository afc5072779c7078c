#include "aq_q4_kernels.hpp"

aq_status aq_q4_impl::launch_bf16(aq_ctx *ctx, const args &a) { return launch<x_bf16>(ctx, a); }
