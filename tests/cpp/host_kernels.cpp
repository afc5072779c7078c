// Which kernels the calls of a layer that answers with codes launch, against a
// HIP runtime of its own (below) that runs none.  Attention kernels for whole
// pieces (their fifth template argument) read and write rows 16 bytes at a
// time, so they may only be taken where a row is a whole number of them.  And
// the kernels that sizes of the GPU tests are there for are those that such
// calls launch.  No GPU.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <string>
#include <vector>

#include <cxxabi.h>

#include "aq_mi355x.h"

namespace {

std::map<const void *, std::string> &names() {   // of the kernels, filled before main
    static std::map<const void *, std::string> all;
    return all;
}
std::vector<std::string> launched;
uintptr_t next_address = 1 << 20;

hipError_t launch(const void *kernel) {
    launched.push_back(names()[kernel]);
    return hipSuccess;
}

}  // namespace

extern "C" {

hipError_t hipMalloc(void **p, size_t n) {
    *p = reinterpret_cast<void *>(next_address);
    next_address += (n + 4095) / 4096 * 4096;
    return hipSuccess;
}
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
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
hipError_t hipLaunchKernel(const void *kernel, dim3, dim3, void **, size_t, hipStream_t) { return launch(kernel); }
hipError_t hipExtLaunchKernel(const void *kernel, dim3, dim3, void **, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) {
    return launch(kernel);
}
// What compiled HIP code calls around its kernels.
void **__hipRegisterFatBinary(const void *) {
    static void *module = nullptr;
    return &module;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *kernel, char *, const char *name, unsigned, void *, void *, dim3 *, dim3 *, int *) {
    int status = 0;
    char *plain = abi::__cxa_demangle(name, nullptr, nullptr, &status);
    names()[kernel] = plain ? plain : name;
    std::free(plain);
}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
    *grid = *block = dim3(1);
    *lds = 0;
    *stream = nullptr;
    return hipSuccess;
}

}  // extern "C"

namespace {

aq_ctx *ctx = nullptr;
void *const some = reinterpret_cast<void *>(uintptr_t{1} << 40);   // device addresses are not looked into
int failures = 0, whole = 0;

void by_whole_pieces() {
    for (int type : {AQ_T_F32, AQ_T_F16, AQ_T_BF16})
        for (int64_t D = 1; D <= 256; ++D)
            for (int64_t P : {0, 5, 300})
                for (int64_t S : {0, 7, 300})
                    for (int64_t T : {1, 50, 300})
                        for (int call = 0; call < 2; ++call) {
                            const aq_heads q{some, T * 2 * D, 2 * D, D}, k{some, S * D, D, D}, pk{some, 0, D, D};
                            launched.clear();
                            const aq_status st =
                                call == 0 ? aq_prefix_attention(ctx, type, 3, T, P, S, 2, 1, D, q, pk, pk, k, k, nullptr, nullptr, 1.0f, q)
                                          : aq_cross_attention(ctx, type, 3, T, S, 2, 1, D, q, k, k, nullptr, nullptr, nullptr, 0, 1.0f, q);
                            const std::string name = launched.empty() ? std::string() : launched[0];
                            const bool pieces = D * (type == AQ_T_F32 ? 4 : 2) % 16 == 0;
                            const bool direct = name.find(", true, ") != std::string::npos;
                            whole += direct;
                            if ((st != AQ_OK || name.find("attn_kernel<") == std::string::npos || direct != pieces) && ++failures <= 10)
                                std::printf("FAIL: type %d D %d P %d S %d T %d: %s\n", type, (int)D, (int)P, (int)S, (int)T, name.c_str());
                        }
}

void reached(bool ok, const char *kernel) {
    bool found = false;
    for (const std::string &name : launched) found = found || name.find(kernel) != std::string::npos;
    if (ok && found) return;
    ++failures;
    std::printf("FAIL: %s is not among", kernel);
    for (const std::string &name : launched) std::printf(" %s", name.c_str());
    std::printf("\n");
}

void products() {
    struct {
        int64_t N, K, M;
        int type;
        int64_t x_ld;
        const char *kernel;
    } const cases[] = {
        {3090, 336, 4100, AQ_T_I8, 336, "i8_gemm_kernel<false, 8, 4>"},
        {3090, 1001, 4100, AQ_T_I8, 1003, "i8_gemm_kernel<true, 8, 4>"},
        {3090, 336, 4100, AQ_T_F32, 336, "i8_gemm_kernel<true, 8, 4>"},
        {16397, 1100, 37, AQ_T_I8, 1100, "i8_product_kernel<true, 4, 4, 1>"},
        {16397, 1100, 70, AQ_T_BF16, 1100, "i8_product_kernel<true, 4, 4, 1>"},
        {300, 8100, 8265, AQ_T_BF16, 8100, "i8_gemm_kernel<true, 4, 2>"},
        {300, 8100, 8265, AQ_T_BF16, 8100, "i8_product_kernel<true, 1, 1, 4>"},   // of the second turn
        {20, 8100, 8300, AQ_T_BF16, 8100, "i8_product_kernel<true, 2, 2, 2>"},
    };
    for (const auto &c : cases) {
        std::vector<int8_t> w(static_cast<size_t>(c.N * c.K));
        std::vector<float> scale(static_cast<size_t>(c.N));
        aq_i8 *h = nullptr;
        if (aq_i8_upload(ctx, c.N, c.K, w.data(), scale.data(), nullptr, &h) != AQ_OK) {
            ++failures;
            continue;
        }
        launched.clear();
        reached(aq_i8_forward(ctx, h, c.type, some, c.x_ld, c.type == AQ_T_I8 ? static_cast<const float *>(some) : nullptr, c.M, AQ_T_F32,
                              some, c.N) == AQ_OK,
                c.kernel);
        aq_i8_release(h);
    }
}

void two_jobs() {
    struct {
        int64_t B, T, P, S, H, Hkv, D;
        int type;
        const char *kernel;
    } const cases[] = {
        {3, 17, 300, 90, 4, 2, 64, AQ_T_BF16, "attn_kernel<aq_types::bf16, 64, 2, 4, true, 1>"},
        {2, 32, 500, 70, 4, 2, 100, AQ_T_F16, "attn_kernel<aq_types::f16, 128, 2, 4, false, 1>"},
        {30, 2, 700, 90, 4, 2, 80, AQ_T_F32, "attn_kernel<aq_types::f32, 128, 1, 4, true, 3>"},
        {9, 16, 1000, 50, 2, 2, 128, AQ_T_F32, "attn_kernel<aq_types::f32, 128, 1, 4, true, 3>"},
    };
    for (const auto &c : cases) {
        const aq_heads q{some, c.T * c.H * c.D, c.H * c.D, c.D}, k{some, c.S * c.Hkv * c.D, c.Hkv * c.D, c.D}, pk{some, 0, c.Hkv * c.D, c.D};
        launched.clear();
        const bool ok = aq_prefix_attention(ctx, c.type, c.B, c.T, c.P, c.S, c.H, c.Hkv, c.D, q, pk, pk, k, k, nullptr, nullptr, 1.0f, q) == AQ_OK;
        reached(ok, c.kernel);
        reached(ok, "attn_join_kernel");   // (each of the two jobs is a part at least)
    }
}

}  // namespace

int main() {
    if (aq_ctx_create(0, nullptr, &ctx) != AQ_OK) return 1;
    by_whole_pieces();
    products();
    two_jobs();
    aq_ctx_destroy(ctx);
    std::printf("%d failures, %d calls by whole pieces\n", failures, whole);
    return failures != 0;
}
