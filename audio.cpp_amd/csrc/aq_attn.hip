// Attention to an encoder's states and over a shared prefix: the C ABI, how a
// call is cut into launches, and the joining of parts.  The kernels are in
// aq_attn_kernels.hpp.
#include "aq_attn.hpp"
#include "aq_types.hpp"

#include <algorithm>
#include <cmath>

namespace {

using aq_attn_impl::args;

struct join_args {
    const float *sums, *ml;
    void *out;
    const int32_t *q_len;
    int64_t rows, batch, row, head;   // strides of out
    int T, H, D, parts;
};

// One wave a row: out = sum over parts of 2^(m_part - m) sums_part, over the
// same sum of the weights.  In the parts' order.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(join_args a) {
    const int lane = threadIdx.x & 63;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (r >= a.rows) return;
    const int h = static_cast<int>(r % a.H);
    const int64_t bt = r / a.H, b = bt / a.T, t = bt % a.T;
    if (a.q_len && t >= a.q_len[b]) return;
    float m = -INFINITY;
    for (int p = lane; p < a.parts; p += 64) m = fmaxf(m, a.ml[(p * a.rows + r) * 2]);
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float from = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[4] = {};
    for (int p = 0; p < a.parts; ++p) {
        const int64_t at = p * a.rows + r;
        const float by = __builtin_amdgcn_exp2f(a.ml[at * 2] - from);
        l = __fmaf_rn(a.ml[at * 2 + 1], by, l);
        if (by == 0.0f) continue;   // (a part without a key for this row holds zeros)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < a.D) o[i] = __fmaf_rn(a.sums[at * a.D + lane + 64 * i], by, o[i]);
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    typename T::raw *to = static_cast<typename T::raw *>(a.out) + b * a.batch + t * a.row + h * a.head;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.D) to[lane + 64 * i] = T::store(o[i] * by);
}

// Scratch of the parts, at most.
constexpr int64_t kPartBytes = int64_t{256} << 20;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct plan {
    bool rows;      // which kernel
    int tiles, splits;
};

// A launch over `rows` rows (of each of `groups` groups) and `keys` keys: the
// kernel, and in how many parts the keys are taken so that the card is full.
plan plan_of(const aq_ctx *ctx, int64_t groups, int64_t rows, int64_t keys, int64_t most_parts) {
    plan p;
    p.rows = rows > 32;
    p.tiles = static_cast<int>(ceil_div(rows, p.rows ? 128 : 32));
    const int64_t blocks = groups * p.tiles, want = 2 * ctx->num_cus;
    // at least 256 keys a part
    const int64_t most = std::min(most_parts, ceil_div(keys, 256));
    p.splits = static_cast<int>(std::max<int64_t>(1, std::min(most, want / std::max<int64_t>(blocks, 1))));
    return p;
}

aq_status launch(aq_ctx *ctx, int type, const args &a, bool rows) {
    switch (type) {
    case AQ_T_F32: return rows ? aq_attn_impl::launch_rows_f32(ctx, a) : aq_attn_impl::launch_keys_f32(ctx, a);
    case AQ_T_F16: return rows ? aq_attn_impl::launch_rows_f16(ctx, a) : aq_attn_impl::launch_keys_f16(ctx, a);
    default: return rows ? aq_attn_impl::launch_rows_bf16(ctx, a) : aq_attn_impl::launch_keys_bf16(ctx, a);
    }
}

aq_status attend(aq_ctx *ctx, int type, args a) {
    const int64_t per_stream = static_cast<int64_t>(a.T) * a.G;   // rows of a stream and key head
    a.rows = static_cast<int64_t>(a.B) * a.T * a.H;
    const int64_t part_bytes = a.rows * (a.D + 2) * 4, most_parts = std::max<int64_t>(kPartBytes / part_bytes, 1);
    // The streams' rows go over the prefix together where a stream alone would
    // not fill a tile of rows; then its own keys are a part of their own.
    const bool apart = a.P > 0 && a.B > 1 && per_stream < 64 && most_parts >= 2;
    plan first, second{};
    int parts;
    if (apart) {
        first = plan_of(ctx, a.Hkv, per_stream * a.B, a.P, most_parts / 2);
        second = plan_of(ctx, static_cast<int64_t>(a.B) * a.Hkv, per_stream, a.S, most_parts / 2);
        parts = first.splits + second.splits;
    } else {
        first = plan_of(ctx, static_cast<int64_t>(a.B) * a.Hkv, per_stream, static_cast<int64_t>(a.P) + a.S, most_parts);
        parts = first.splits;
    }
    if (parts > 1) {
        void *p = nullptr;
        aq_status st = aq_ctx_scratch(ctx, 9, static_cast<size_t>(parts) * static_cast<size_t>(part_bytes), &p);
        if (st != AQ_OK) return st;
        a.sums = static_cast<float *>(p);
        a.ml = a.sums + static_cast<int64_t>(parts) * a.rows * a.D;
    }
    a.walk = apart ? aq_attn_impl::kPrefix : aq_attn_impl::kBoth;
    a.tiles = first.tiles;
    a.splits = first.splits;
    aq_status st = launch(ctx, type, a, first.rows);
    if (st == AQ_OK && apart) {
        a.walk = aq_attn_impl::kOwn;
        a.tiles = second.tiles;
        a.splits = second.splits;
        a.part = first.splits;
        st = launch(ctx, type, a, second.rows);
    }
    if (st != AQ_OK || parts == 1) return st;
    const join_args j{a.sums, a.ml, a.out, a.q_len, a.rows, a.so.batch, a.so.row, a.so.head, a.T, a.H, a.D, parts};
    const dim3 grid(static_cast<uint32_t>(ceil_div(a.rows, 4)));
    if (type == AQ_T_F32) aq_launch_timed(ctx, false, attn_join_kernel<aq_types::f32>, grid, dim3(256), 0u, j);
    else if (type == AQ_T_F16) aq_launch_timed(ctx, false, attn_join_kernel<aq_types::f16>, grid, dim3(256), 0u, j);
    else aq_launch_timed(ctx, false, attn_join_kernel<aq_types::bf16>, grid, dim3(256), 0u, j);
    AQ_HIP(ctx, hipGetLastError());
    return AQ_OK;
}

aq_attn_impl::strides strides_of(const aq_heads &t) { return {t.batch_ld, t.row_ld, t.head_ld}; }

bool negative(const aq_heads &t) { return t.batch_ld < 0 || t.row_ld < 0 || t.head_ld < 0; }

// Whether two of the rows [batch, row, head] of D elements share one.
bool overlaps(const aq_heads &t, int64_t B, int64_t T, int64_t H, int64_t D) {
    int64_t ld[3] = {t.batch_ld, t.row_ld, t.head_ld}, n[3] = {B, T, H}, reach = D;
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (ld[j] < ld[i]) {
                std::swap(ld[i], ld[j]);
                std::swap(n[i], n[j]);
            }
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        if (ld[i] < reach) return true;
        if (ld[i] > (int64_t{1} << 60) / n[i]) return true;   // no such tensor
        reach += ld[i] * (n[i] - 1);
    }
    return false;
}

// Rows that start and end at 16 bytes.
bool pieces(const aq_heads &t, int64_t D, int64_t size) {
    return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && D * size % 16 == 0 && t.batch_ld * size % 16 == 0 &&
           t.row_ld * size % 16 == 0 && t.head_ld * size % 16 == 0;
}

constexpr int64_t kMost = int64_t{1} << 30;

// The checks that both entry points share.
aq_status checked(aq_ctx *ctx, const char *name, int type, int64_t B, int64_t T, int64_t keys, int64_t S, int64_t heads,
                  int64_t kv_heads, int64_t D, const aq_heads &q, const aq_heads &k, const aq_heads &v, float scale,
                  const aq_heads &out) {
    if (!ctx) return AQ_E_INVALID_ARG;
    if (type != AQ_T_F32 && type != AQ_T_F16 && type != AQ_T_BF16)
        return aq_fail(ctx, AQ_E_INVALID_ARG, "%s: type %d is not F32, F16 or BF16", name, type);
    if (!(scale > 0.0f) || !std::isfinite(scale))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "%s: scale %g is not above 0 and finite", name, static_cast<double>(scale));
    if (B < 0 || T < 0 || keys < 0 || S < 0 || keys > kMost || S > kMost || heads < 1 || kv_heads < 1 || heads > kMost ||
        heads % kv_heads != 0 || D < 1 || D > 256)
        return aq_fail(ctx, AQ_E_SHAPE, "%s: B=%lld T=%lld keys=%lld + %lld (up to 2^30) heads=%lld kv_heads=%lld D=%lld (1 to 256)",
                       name, (long long)B, (long long)T, (long long)keys, (long long)S, (long long)heads, (long long)kv_heads,
                       (long long)D);
    if (B > 0 && T > 0 && (B > kMost / heads || T > kMost / heads / B))
        return aq_fail(ctx, AQ_E_SHAPE, "%s: B=%lld T=%lld heads=%lld: more than 2^30 rows", name, (long long)B, (long long)T,
                       (long long)heads);
    if (B == 0 || T == 0) return AQ_OK;
    if (!q.data || !out.data || (S > 0 && (!k.data || !v.data)))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "%s: null q, k, v or out", name);
    if (negative(q) || negative(k) || negative(v) || negative(out))
        return aq_fail(ctx, AQ_E_SHAPE, "%s: a stride is negative", name);
    if (overlaps(out, B, T, heads, D)) return aq_fail(ctx, AQ_E_SHAPE, "%s: rows of out overlap", name);
    return AQ_OK;
}

}  // namespace

extern "C" {

aq_status aq_cross_attention(aq_ctx *ctx, int type, int64_t B, int64_t T, int64_t S, int64_t heads, int64_t kv_heads, int64_t D,
                             aq_heads q, aq_heads k, aq_heads v, const int32_t *q_len, const int32_t *kv_len,
                             const uint8_t *mask, int64_t mask_ld, float scale, aq_heads out) {
    aq_status st = checked(ctx, "aq_cross_attention", type, B, T, 0, S, heads, kv_heads, D, q, k, v, scale, out);
    if (st != AQ_OK || B == 0 || T == 0) return st;
    if (mask && (mask_ld < 0 || (B > 1 && mask_ld != 0 && mask_ld < S)))
        return aq_fail(ctx, AQ_E_SHAPE, "aq_cross_attention: mask_ld=%lld is neither 0 nor at least S=%lld", (long long)mask_ld,
                       (long long)S);
    aq_device_guard g(ctx->device);
    const int64_t size = type == AQ_T_F32 ? 4 : 2;
    args a{};
    a.q = q.data;
    a.k = k.data;
    a.v = v.data;
    a.out = out.data;
    a.sq = strides_of(q);
    a.sk = strides_of(k);
    a.sv = strides_of(v);
    a.so = strides_of(out);
    a.q_len = q_len;
    a.kv_len = kv_len;
    a.mask = mask;
    a.mask_ld = mask_ld;
    a.c = scale * 1.4426950408889634f;
    a.B = static_cast<int>(B);
    a.T = static_cast<int>(T);
    a.S = static_cast<int>(S);
    a.H = static_cast<int>(heads);
    a.Hkv = static_cast<int>(kv_heads);
    a.G = a.H / a.Hkv;
    a.D = static_cast<int>(D);
    a.direct = pieces(k, D, size) && pieces(v, D, size);
    return attend(ctx, type, a);
}

aq_status aq_prefix_attention(aq_ctx *ctx, int type, int64_t B, int64_t T, int64_t P, int64_t S, int64_t heads, int64_t kv_heads,
                              int64_t D, aq_heads q, aq_heads prefix_k, aq_heads prefix_v, aq_heads k, aq_heads v,
                              const int32_t *q_len, const int32_t *kv_len, float scale, aq_heads out) {
    aq_status st = checked(ctx, "aq_prefix_attention", type, B, T, P, S, heads, kv_heads, D, q, k, v, scale, out);
    if (st != AQ_OK || B == 0 || T == 0) return st;
    if (P > 0 && (!prefix_k.data || !prefix_v.data))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "aq_prefix_attention: null prefix_k or prefix_v");
    if (prefix_k.row_ld < 0 || prefix_k.head_ld < 0 || prefix_v.row_ld < 0 || prefix_v.head_ld < 0)
        return aq_fail(ctx, AQ_E_SHAPE, "aq_prefix_attention: a stride of the prefix is negative");
    aq_device_guard g(ctx->device);
    const int64_t size = type == AQ_T_F32 ? 4 : 2;
    prefix_k.batch_ld = prefix_v.batch_ld = 0;
    args a{};
    a.q = q.data;
    a.pk = prefix_k.data;
    a.pv = prefix_v.data;
    a.k = k.data;
    a.v = v.data;
    a.out = out.data;
    a.sq = strides_of(q);
    a.spk = strides_of(prefix_k);
    a.spv = strides_of(prefix_v);
    a.sk = strides_of(k);
    a.sv = strides_of(v);
    a.so = strides_of(out);
    a.q_len = q_len;
    a.kv_len = kv_len;
    a.c = scale * 1.4426950408889634f;
    a.B = static_cast<int>(B);
    a.T = static_cast<int>(T);
    a.S = static_cast<int>(S);
    a.P = static_cast<int>(P);
    a.H = static_cast<int>(heads);
    a.Hkv = static_cast<int>(kv_heads);
    a.G = a.H / a.Hkv;
    a.D = static_cast<int>(D);
    a.causal = 1;
    a.direct = (S == 0 || (pieces(k, D, size) && pieces(v, D, size))) &&
               (P == 0 || (pieces(prefix_k, D, size) && pieces(prefix_v, D, size)));
    return attend(ctx, type, a);
}

}  // extern "C"
