#include "aq_q4_kernels.hpp"

aq_status aq_q4_impl::launch_i8(aq_ctx *ctx, const args &a) { return launch<x_i8>(ctx, a); }
