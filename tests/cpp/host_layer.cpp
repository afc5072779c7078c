// The entry points of a layer that answers with codes against a HIP runtime of
// its own (below) that runs no kernel: what they refuse, what they launch and
// how much scratch they take.  No GPU.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "aq_mi355x.h"

namespace {

struct launch {
    dim3 grid, block;
    size_t lds;
};
std::vector<launch> launches;
size_t allocated = 0, limit = SIZE_MAX;
uintptr_t next_address = 1 << 20;
hipError_t last = hipSuccess;

}  // namespace

extern "C" {

hipError_t hipMalloc(void **p, size_t n) {
    if (n > limit) return last = hipErrorOutOfMemory;
    *p = reinterpret_cast<void *>(next_address);
    next_address += (n + 4095) / 4096 * 4096;
    allocated += n;
    return hipSuccess;
}
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
const char *hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceCount(int *n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) { return p->multiProcessorCount = 256, hipSuccess; }
hipError_t hipMemcpy(void *, const void *, size_t, hipMemcpyKind) { return hipSuccess; }
hipError_t hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipMemset(void *, int, size_t) { return hipSuccess; }
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) { return *s = hipStreamCaptureStatusNone, hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t *e) { return *e = nullptr, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { return *e = nullptr, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) { return *ms = 0, hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipFuncGetAttributes(hipFuncAttributes *a, const void *) { return *a = hipFuncAttributes{}, hipSuccess; }
hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void **, const void *) { return hipErrorInvalidSymbol; }
hipError_t hipLaunchKernel(const void *, dim3 grid, dim3 block, void **, size_t lds, hipStream_t) {
    launches.push_back({grid, block, lds});
    return hipSuccess;
}
hipError_t hipExtLaunchKernel(const void *, dim3 grid, dim3 block, void **, size_t lds, hipStream_t, hipEvent_t, hipEvent_t, int) {
    launches.push_back({grid, block, lds});
    return hipSuccess;
}
// What compiled HIP code calls around its kernels.
void **__hipRegisterFatBinary(const void *) {
    static void *module = nullptr;
    return &module;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, dim3 *, dim3 *, int *) {}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
static launch pushed;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t) {
    pushed = {grid, block, lds};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
    *grid = pushed.grid;
    *block = pushed.block;
    *lds = pushed.lds;
    *stream = nullptr;
    return hipSuccess;
}

}  // extern "C"

namespace {

int failures = 0;

void expect(bool ok, const char *what) {
    if (!ok) {
        std::printf("FAIL: %s\n", what);
        ++failures;
    }
}

aq_ctx *ctx = nullptr;
void *const kSome = reinterpret_cast<void *>(uintptr_t{1} << 40);   // device addresses are not looked into

bool said(const char *name) { return std::strstr(aq_last_error(ctx), name) != nullptr; }

// Launches that the card takes: at least one block, fewer than 2^32 threads, LDS of a compute unit.
bool fits() {
    for (const launch &l : launches) {
        const uint64_t threads = uint64_t{l.grid.x} * l.block.x;
        if (!l.grid.x || !l.grid.y || threads >= uint64_t{1} << 32 || l.grid.y > 65535 || l.block.x > 1024 ||
            l.lds > 160 * 1024 - 2048)
            return false;
    }
    return !launches.empty();
}

struct attention {
    int type = AQ_T_BF16;
    int64_t B = 2, T = 3, P = 0, S = 50, H = 4, Hkv = 2, D = 64;
    aq_heads q{}, pk{}, pv{}, k{}, v{}, out{};
    float scale = 0.125f;
    const uint8_t *mask = nullptr;
    int64_t mask_ld = 50;

    void lay_out() {
        q = out = {kSome, T * H * D, H * D, D};
        k = v = {kSome, S * Hkv * D, Hkv * D, D};
        pk = pv = {kSome, 0, Hkv * D, D};
    }
    aq_status cross() const {
        launches.clear();
        return aq_cross_attention(ctx, type, B, T, S, H, Hkv, D, q, k, v, nullptr, nullptr, mask, mask_ld, scale, out);
    }
    aq_status prefix() const {
        launches.clear();
        return aq_prefix_attention(ctx, type, B, T, P, S, H, Hkv, D, q, pk, pv, k, v, nullptr, nullptr, scale, out);
    }
};

void attention_refusals() {
    attention good;
    good.lay_out();
    expect(good.cross() == AQ_OK && good.prefix() == AQ_OK, "an ordinary call");
    struct {
        const char *what;
        void (*spoil)(attention &);
        aq_status status;
    } const bad[] = {
        {"type", [](attention &a) { a.type = AQ_T_I8; }, AQ_E_INVALID_ARG},
        {"scale 0", [](attention &a) { a.scale = 0; }, AQ_E_INVALID_ARG},
        {"scale below 0", [](attention &a) { a.scale = -1; }, AQ_E_INVALID_ARG},
        {"scale NaN", [](attention &a) { a.scale = NAN; }, AQ_E_INVALID_ARG},
        {"scale of 3e38", [](attention &a) { a.scale = 3e38f; }, AQ_E_INVALID_ARG},
        {"null q", [](attention &a) { a.q.data = nullptr; }, AQ_E_INVALID_ARG},
        {"null k", [](attention &a) { a.k.data = nullptr; }, AQ_E_INVALID_ARG},
        {"null v", [](attention &a) { a.v.data = nullptr; }, AQ_E_INVALID_ARG},
        {"null out", [](attention &a) { a.out.data = nullptr; }, AQ_E_INVALID_ARG},
        {"B below 0", [](attention &a) { a.B = -1; }, AQ_E_SHAPE},
        {"T below 0", [](attention &a) { a.T = -1; }, AQ_E_SHAPE},
        {"S below 0", [](attention &a) { a.S = -1; }, AQ_E_SHAPE},
        {"S above 2^30", [](attention &a) { a.S = (int64_t{1} << 30) + 1; }, AQ_E_SHAPE},
        {"no heads", [](attention &a) { a.H = 0; }, AQ_E_SHAPE},
        {"no key heads", [](attention &a) { a.Hkv = 0; }, AQ_E_SHAPE},
        {"heads no multiple", [](attention &a) { a.H = 5; }, AQ_E_SHAPE},
        {"D 0", [](attention &a) { a.D = 0; }, AQ_E_SHAPE},
        {"D 257", [](attention &a) { a.D = 257; }, AQ_E_SHAPE},
        {"too many rows", [](attention &a) { a.B = a.T = int64_t{1} << 20; }, AQ_E_SHAPE},
        {"a negative stride", [](attention &a) { a.k.row_ld = -1; }, AQ_E_SHAPE},
        {"rows of out that share", [](attention &a) { a.out.batch_ld = 0; }, AQ_E_SHAPE},
        {"rows of out too close", [](attention &a) { a.out.head_ld = 63; }, AQ_E_SHAPE},
    };
    for (const auto &b : bad) {
        attention a = good;
        b.spoil(a);
        expect(a.cross() == b.status && said("aq_cross_attention") && launches.empty(), b.what);
        expect(a.prefix() == b.status && said("aq_prefix_attention") && launches.empty(), b.what);
    }
    attention a = good;
    a.mask = static_cast<const uint8_t *>(kSome);
    expect(a.cross() == AQ_OK, "a mask");
    a.mask_ld = 0;
    expect(a.cross() == AQ_OK, "one mask for all streams");
    a.mask_ld = 49;
    expect(a.cross() == AQ_E_SHAPE && launches.empty(), "rows of a mask that overlap");
    a = good;
    a.P = 7;
    a.pv.data = nullptr;
    expect(a.prefix() == AQ_E_INVALID_ARG && launches.empty(), "null prefix_v");
    a = good;
    a.P = a.S = int64_t{1} << 29;
    a.P += 1;
    expect(a.prefix() == AQ_E_SHAPE && launches.empty(), "2^30 + 1 keys");
    for (int64_t zero : {0, 1}) {
        attention none;
        (zero ? none.B : none.T) = 0;
        expect(none.cross() == AQ_OK && none.prefix() == AQ_OK && launches.empty(), "an empty call looks at no pointer");
    }
    attention heads_only = good;   // a layout [B, heads, T, D]
    heads_only.out = {kSome, 4 * 3 * 64, 64, 3 * 64};
    expect(heads_only.cross() == AQ_OK, "heads before rows");
}

void attention_launches() {
    for (int type : {AQ_T_F32, AQ_T_F16, AQ_T_BF16})
        for (int64_t D : {1, 33, 64, 128, 130, 256})
            for (int64_t B : {1, 3, 128, 4000})
                for (int64_t T : {1, 7, 40, 2000})
                    for (int64_t S : {1, 100, 20000})
                        for (int64_t P : {0, 90, 70000}) {
                            attention a;
                            a.type = type;
                            a.D = D, a.B = B, a.T = T, a.S = S, a.P = P;
                            a.lay_out();
                            const size_t before = allocated;
                            expect(a.cross() == AQ_OK && fits() && launches.size() <= 2, "launches of cross attention");
                            expect(a.prefix() == AQ_OK && fits() && launches.size() <= 2, "launches of attention over a prefix");
                            expect(allocated - before <= size_t{1} << 30, "scratch");
                        }
    attention many;   // more blocks than a launch takes
    many.B = int64_t{1} << 25;
    many.T = 1;
    many.lay_out();
    expect(many.cross() == AQ_E_SHAPE && launches.empty(), "2^26 blocks");
}

void i8_launches() {
    std::vector<int8_t> w(300 * 1000);
    std::vector<float> scale(300);
    for (int64_t K : {1, 64, 100, 1000})
        for (int64_t N : {1, 17, 300}) {
            aq_i8 *h = nullptr;
            expect(aq_i8_upload(ctx, N, K, w.data(), scale.data(), nullptr, &h) == AQ_OK && h, "upload");
            for (int64_t M : {1, 16, 17, 64, 65, 500, 100000, 1 << 20})
                for (int type : {AQ_T_I8, AQ_T_F32, AQ_T_F16, AQ_T_BF16}) {
                    launches.clear();
                    const float *xs = type == AQ_T_I8 ? static_cast<const float *>(kSome) : nullptr;
                    expect(aq_i8_forward(ctx, h, type, kSome, K, xs, M, AQ_T_BF16, kSome, N) == AQ_OK && fits(), "launches of a product");
                    launches.clear();
                    expect(aq_i8_forward(ctx, h, type, kSome, K, xs ? nullptr : static_cast<const float *>(kSome), M, AQ_T_BF16, kSome, N) ==
                                   AQ_E_INVALID_ARG && launches.empty(),
                           "a scale that does not go with x");
                }
            launches.clear();
            expect(aq_i8_forward(ctx, h, AQ_T_F32, nullptr, K, nullptr, 0, AQ_T_F32, nullptr, N) == AQ_OK && launches.empty(), "no rows");
            expect(aq_i8_forward(ctx, h, AQ_T_E4M3, kSome, K, nullptr, 1, AQ_T_F32, kSome, N) == AQ_E_INVALID_ARG, "x_type");
            expect(aq_i8_forward(ctx, h, AQ_T_F32, kSome, K, nullptr, 1, AQ_T_I8, kSome, N) == AQ_E_INVALID_ARG, "y_type");
            expect(aq_i8_forward(ctx, h, AQ_T_F32, kSome, K - 1, nullptr, 1, AQ_T_F32, kSome, N) == AQ_E_SHAPE, "x_ld");
            expect(aq_i8_forward(ctx, h, AQ_T_F32, kSome, K, nullptr, 1, AQ_T_F32, kSome, N - 1) == AQ_E_SHAPE, "y_ld");
            expect(aq_i8_forward(ctx, h, AQ_T_F32, kSome, K, nullptr, (1 << 20) + 1, AQ_T_F32, kSome, N) == AQ_E_SHAPE, "M");
            expect(launches.empty(), "nothing is launched for a refused product");
            aq_i8_release(h);
        }
    aq_i8 *h = nullptr;
    expect(aq_i8_upload(ctx, 0, 5, w.data(), scale.data(), nullptr, &h) == AQ_E_SHAPE && !h, "no rows of W");
    expect(aq_i8_upload(ctx, 5, 1 << 17, w.data(), scale.data(), nullptr, &h) == AQ_E_SHAPE && !h, "2^17 columns");
    expect(aq_i8_upload(ctx, 5, 5, nullptr, scale.data(), nullptr, &h) == AQ_E_INVALID_ARG && !h, "null w");
    expect(aq_i8_upload(ctx, 5, 5, w.data(), nullptr, nullptr, &h) == AQ_E_INVALID_ARG && !h, "null scale");
    limit = 1000;
    expect(aq_i8_upload(ctx, 300, 1000, w.data(), scale.data(), nullptr, &h) == AQ_E_NOMEM && !h && last == hipSuccess,
           "an upload without memory leaves no error behind");
    limit = SIZE_MAX;
}

}  // namespace

int main() {
    if (aq_ctx_create(0, nullptr, &ctx) != AQ_OK) return 1;
    attention_refusals();
    attention_launches();
    i8_launches();
    aq_ctx_destroy(ctx);
    std::printf("%d failures\n", failures);
    return failures != 0;
}
