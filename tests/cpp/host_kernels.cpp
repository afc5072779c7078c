// Which kernels an attention call launches, against a HIP runtime of its own
// (below) that runs none.  Kernels for whole pieces (their fifth template
// argument) read and write rows 16 bytes at a time, so they may only be taken
// where a row is a whole number of them.  No GPU.
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

int main() {
    aq_ctx *ctx = nullptr;
    if (aq_ctx_create(0, nullptr, &ctx) != AQ_OK) return 1;
    void *const some = reinterpret_cast<void *>(uintptr_t{1} << 40);   // device addresses are not looked into
    int failures = 0, whole = 0;
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
                            const std::string &name = launched.empty() ? std::string() : launched[0];
                            const bool pieces = D * (type == AQ_T_F32 ? 4 : 2) % 16 == 0;
                            const bool direct = name.find(", true, ") != std::string::npos;
                            whole += direct;
                            if (st != AQ_OK || name.find("attn_kernel<") == std::string::npos || direct != pieces) {
                                if (++failures <= 10)
                                    std::printf("FAIL: type %d D %d P %d S %d T %d: %s\n", type, (int)D, (int)P, (int)S, (int)T, name.c_str());
                            }
                        }
    aq_ctx_destroy(ctx);
    std::printf("%d failures, %d calls by whole pieces\n", failures, whole);
    return failures != 0;
}
