// Attention to an encoder's states and over a shared prefix: the C ABI, how a
// call is cut into launches, and the joining of parts.  The kernels are in
// aq_attn_kernels.hpp.
#include "aq_attn.hpp"
#include "aq_types.hpp"

#include <algorithm>

namespace {

using aq_attn_impl::args;

struct join_args {
    const float *sums, *ml;
    void *out;
    const int32_t *q_len;
    int64_t rows, batch, row, head;   // strides of out
    int T, H, D, parts;
    float c;
};

// One wave a row: out = sum over parts of 2^(m_part - m) sums_part, over the
// same sum of the weights.  Four columns a lane; where that leaves lanes, 64 /
// LANES parts are taken at once, in an order that the sizes alone decide.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void attn_join_kernel(join_args a) {
    constexpr int kAt = 64 / LANES;
    const int lane = threadIdx.x & 63, at = (lane % LANES) * 4, set = lane / LANES;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (r >= a.rows) return;
    const int h = static_cast<int>(r % a.H);
    const int64_t bt = r / a.H, b = bt / a.T, t = bt % a.T;
    if (a.q_len && t >= a.q_len[b]) return;
    float m = -INFINITY;
    for (int p = lane; p < a.parts; p += 64) m = fmaxf(m, a.ml[(p * a.rows + r) * 2]);
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    float l = 0.0f, o[4] = {};
    const auto add = [&](int p, auto load) {
        const int64_t row = p * a.rows + r;
        const float by = aq_attn_impl::weight_of(a.ml[row * 2], m, a.c);
        l = __fmaf_rn(a.ml[row * 2 + 1], by, l);
        float v[4];
        load(a.sums + row * a.D, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __fmaf_rn(v[i], by, o[i]);
    };
    if (a.D % 4 == 0) {   // one load each without a condition (lanes past the end repeat the last): several are on their way
        const int from4 = min(at, a.D - 4);
#pragma unroll 8
        for (int p = set; p < a.parts; p += kAt) add(p, [&](const float *sums, float(&v)[4]) { std::memcpy(v, sums + from4, 16); });
    } else {
        for (int p = set; p < a.parts; p += kAt)
            add(p, [&](const float *sums, float(&v)[4]) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = sums[min(at + i, a.D - 1)];
            });
    }
#pragma unroll
    for (int d = LANES; d < 64; d <<= 1) {
        l += __shfl_xor(l, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], d);
    }
    if (set != 0 || at >= a.D) return;
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    typename T::raw *to = static_cast<typename T::raw *>(a.out) + b * a.batch + t * a.row + h * a.head + at;
    typename T::raw y[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) T::store2(y + i, o[i] * by, o[i + 1] * by);
    if (at + 4 <= a.D) std::memcpy(to, y, sizeof(y));
    else
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < a.D) to[i] = y[i];
}

template <typename T>
void launch_join(aq_ctx *ctx, const join_args &j) {
    const dim3 grid(static_cast<uint32_t>((j.rows + 3) / 4));
    if (j.D <= 64) aq_launch_timed(ctx, false, attn_join_kernel<T, 16>, grid, dim3(256), 0u, j);
    else if (j.D <= 128) aq_launch_timed(ctx, false, attn_join_kernel<T, 32>, grid, dim3(256), 0u, j);
    else aq_launch_timed(ctx, false, attn_join_kernel<T, 64>, grid, dim3(256), 0u, j);
}

// Scratch of the parts, at most.
constexpr int64_t kPartBytes = int64_t{256} << 20;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A job over `rows` rows (of each of `groups` groups) and `keys` keys: the keys
// are taken in so many parts that there are `want` blocks.
aq_attn_impl::job job_of(int64_t want, int walk, int type, int D, int64_t groups, int64_t rows, int64_t keys, int64_t most_parts) {
    aq_attn_impl::job j{};
    j.walk = walk;
    // fp32 products bound either kind of block, so what counts is how few rows
    // the last tile wastes.  (Of more than 128 columns there is the first kind only.)
    const bool f32 = type == AQ_T_F32;
    j.many = rows > (f32 ? 96 : 32) || (f32 && D > 128);
    j.tiles = static_cast<int>(ceil_div(rows, j.many ? 128 : 32));
    const int64_t blocks = groups * j.tiles;
    // At least this many keys a part: fp32 products are slow enough for one
    // tile, or one of each wave's (3 x 111 rows over 333 keys: 19 us, 31 with 128
    // keys a part, 60 with 512); 16-bit ones are not worth the joining.
    const int64_t least = !f32 ? 256 : j.many ? 32 : 128;
    const int64_t most = std::min(most_parts, ceil_div(keys, least));
    j.splits = static_cast<int>(std::max<int64_t>(1, std::min(most, want / std::max<int64_t>(blocks, 1))));
    j.blocks = static_cast<int>(blocks * j.splits);
    return j;
}

aq_status attend(aq_ctx *ctx, int type, args a) {
    const int64_t per_stream = static_cast<int64_t>(a.T) * a.G;   // rows of a stream and key head
    const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
    a.rows = static_cast<int64_t>(a.B) * a.T * a.H;
    const int64_t part_bytes = a.rows * (a.D + 2) * 4, most_parts = std::max<int64_t>(kPartBytes / part_bytes, 1);
    // The streams' rows go over the prefix together where a stream alone would
    // not fill half a tile of rows; then its own keys are a part of their own.
    // In us, alone and together: 16 streams over 8192 + 512 keys, bf16, 32 rows
    // each 58, 53; 64 rows 101, 83; 80 rows 103, 115; 64 streams over 4096 + 600,
    // 64 rows 104, 100; 80 rows 104, 117; fp32, 16 rows 112, 108; 32 rows 105, 197.
    const bool apart = a.P > 0 && a.B > 1 && per_stream <= (type == AQ_T_F32 ? 16 : 64) && most_parts >= 2;
    int parts;
    // A compute unit holds two blocks.  A prefix's jobs share it with the own
    // keys', and each of its parts is written and joined: one block a unit, and
    // three for four units where the own keys outnumber the prefix's.  In us,
    // one token, 32/8 heads of 128, for 192, 256 and 512 blocks: 128 streams over
    // 16384 + 1024 keys 124, 134, 129; over 4096 + 1024 94, 97, 105; over 65536 +
    // 64 313, 256, 268; 32 streams over 16384 + 1024 51, 54, 65; over 16384 + 16
    // 38, 37, 51.
    // Other jobs: one block a unit too (in us, with 256 and 512 blocks: one row
    // of 32/8 heads over 65536 keys 54, 58; 4 streams over 8192 31, 34; 16 rows of
    // 2 streams over 8192 28, 31; fp32, of which a unit holds one block, 200 rows
    // over 2000 54, 65), but two where so many 16-bit rows share each key that
    // products bound it (512 rows of 8 heads over 16384: 59, 54).
    const bool wide = per_stream > 256 && type != AQ_T_F32 && a.D <= 128;
    const int64_t full = wide ? 2 * ctx->num_cus : ctx->num_cus;
    const int64_t beside = static_cast<int64_t>(a.B) * a.S >= a.P ? ctx->num_cus * 3 / 4 : ctx->num_cus;
    if (apart) {
        a.jobs[0] = job_of(beside, aq_attn_impl::kPrefix, type, a.D, a.Hkv, per_stream * a.B, a.P, most_parts / 2);
        a.jobs[1] = job_of(full, aq_attn_impl::kOwn, type, a.D, heads, per_stream, a.S, most_parts / 2);
        a.jobs[1].part = a.jobs[0].splits;
        parts = a.jobs[0].splits + a.jobs[1].splits;
    } else {
        a.jobs[0] = job_of(full, aq_attn_impl::kBoth, type, a.D, heads, per_stream, static_cast<int64_t>(a.P) + a.S, most_parts);
        parts = a.jobs[0].splits;
    }
    if (int64_t{a.jobs[0].blocks} + a.jobs[1].blocks >= int64_t{1} << 24)
        return aq_fail(ctx, AQ_E_SHAPE, "attention: %lld streams' heads of %lld rows each need more than 2^24 blocks",
                       (long long)heads, (long long)per_stream);
    if (parts > 1) {
        void *p = nullptr;
        aq_status st = aq_ctx_scratch(ctx, 9, static_cast<size_t>(parts) * static_cast<size_t>(part_bytes), &p);
        if (st != AQ_OK) return st;
        a.sums = static_cast<float *>(p);
        a.ml = a.sums + static_cast<int64_t>(parts) * a.rows * a.D;
    }
    aq_status st = type == AQ_T_F32   ? aq_attn_impl::launch_f32(ctx, a)
                   : type == AQ_T_F16 ? aq_attn_impl::launch_f16(ctx, a)
                                      : aq_attn_impl::launch_bf16(ctx, a);
    if (st != AQ_OK || parts == 1) return st;
    const join_args j{a.sums, a.ml, a.out, a.q_len, a.rows, a.so.batch, a.so.row, a.so.head, a.T, a.H, a.D, parts, a.c};
    if (type == AQ_T_F32) launch_join<aq_types::f32>(ctx, j);
    else if (type == AQ_T_F16) launch_join<aq_types::f16>(ctx, j);
    else launch_join<aq_types::bf16>(ctx, j);
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

// Rows that start and end at 16 bytes, with 64 of them within 2^31 bytes.
bool pieces(const aq_heads &t, int64_t D, int64_t size) {
    return t.row_ld < (int64_t{1} << 25) / size &&
           reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && D * size % 16 == 0 && t.batch_ld * size % 16 == 0 &&
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
    if (!(scale > 0.0f) || !(scale < 1e38f))
        return aq_fail(ctx, AQ_E_INVALID_ARG, "%s: scale %g is not above 0 and below 1e38", name, static_cast<double>(scale));
    if (B < 0 || T < 0 || keys < 0 || S < 0 || keys > kMost || S > kMost || keys + S > kMost || heads < 1 || kv_heads < 1 || heads > kMost ||
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
    // Rows of q and out go by whole pieces too, where there is no key at all as well.
    a.direct = D * size % 16 == 0 && (S == 0 || (pieces(k, D, size) && pieces(v, D, size))) &&
               (P == 0 || (pieces(prefix_k, D, size) && pieces(prefix_v, D, size)));
    return attend(ctx, type, a);
}

}  // extern "C"
