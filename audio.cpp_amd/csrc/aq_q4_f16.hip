#include "aq_q4_kernels.hpp"

aq_status aq_q4_impl::launch_f16(aq_ctx *ctx, const args &a) { return launch<x_f16>(ctx, a); }
