#include "aq_q4_kernels.hpp"

aq_status aq_q4_impl::launch_e4m3(aq_ctx *ctx, const args &a) { return launch<x_e4m3>(ctx, a); }
