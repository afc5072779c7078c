// The library's host code against a HIP runtime of its own (below) that only
// keeps account of device memory: what calls ask for, what they do when it
// cannot be had, and what is freed.  No GPU; kernels are not run.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <map>

#include "aq_mi355x.h"

namespace {

std::map<uintptr_t, size_t> live;   // allocations
size_t used = 0, limit = SIZE_MAX, allocations = 0, bad_frees = 0, launches = 0;
uintptr_t next_address = 1 << 20;
hipError_t last = hipSuccess;

hipError_t done(hipError_t e) {
    if (e != hipSuccess) last = e;   // stays until it is read
    return e;
}

}  // namespace

extern "C" {

hipError_t hipMalloc(void **p, size_t n) {
    if (n > limit || used > limit - n) return done(hipErrorOutOfMemory);
    *p = reinterpret_cast<void *>(next_address);
    live[next_address] = n;
    next_address += (n + 4095) / 4096 * 4096;
    used += n;
    ++allocations;
    return hipSuccess;
}
hipError_t hipFree(void *p) {
    const auto it = live.find(reinterpret_cast<uintptr_t>(p));
    if (it == live.end()) {
        ++bad_frees;
        return done(hipErrorInvalidValue);
    }
    used -= it->second;
    live.erase(it);
    return hipSuccess;
}
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
const char *hipGetErrorString(hipError_t e) { return e == hipErrorOutOfMemory ? "out of memory" : "error"; }
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
hipError_t hipGetSymbolAddress(void **, const void *) { return done(hipErrorInvalidSymbol); }
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) { return ++launches, hipSuccess; }
hipError_t hipExtLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t, hipEvent_t, hipEvent_t, int) {
    return ++launches, hipSuccess;
}
// What compiled HIP code calls around its kernels.
void **__hipRegisterFatBinary(const void *) {
    static void *module = nullptr;
    return &module;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, dim3 *, dim3 *, int *) {}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
static dim3 pushed_grid, pushed_block;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) {
    pushed_grid = grid;
    pushed_block = block;
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
    *grid = pushed_grid;
    *block = pushed_block;
    *lds = 0;
    *stream = nullptr;
    return hipSuccess;
}

}  // extern "C"

namespace {

int failures = 0;

void expect(bool ok, const char *what) {
    std::printf("%s: %s\n", ok ? "ok" : "FAIL", what);
    if (!ok) ++failures;
}

// Sampling from `rows` rows of 20000 takes scratch that grows with them.
aq_status sampled(aq_ctx *ctx, int64_t rows) {
    float *f = reinterpret_cast<float *>(64);   // never read here
    return aq_sample(ctx, AQ_T_F32, f, 20000, rows, 20000, f, nullptr, nullptr, f, nullptr, reinterpret_cast<int32_t *>(64),
                     nullptr);
}

// An upload that runs out of memory at each of its allocations in turn.
void refused_uploads(aq_ctx *ctx) {
    const uint8_t codes[32 * 32] = {}, zero[32 * 2] = {};
    const uint16_t scale[32 * 2] = {};
    const float bias[32] = {};
    const size_t before = used;
    aq_q4 *w = nullptr;
    limit = SIZE_MAX;
    expect(aq_q4_upload(ctx, 32, 64, 32, codes, scale, zero, bias, &w) == AQ_OK, "an upload");
    const size_t held = used - before;
    expect(aq_q4_release(w) == AQ_OK && used == before, "and its release");
    bool refused = true, clean = true, freed = true;
    int refusals = 0;
    for (limit = before; limit < before + held; limit += 64) {
        const aq_status st = aq_q4_upload(ctx, 32, 64, 32, codes, scale, zero, bias, &w);
        refused &= st == AQ_E_NOMEM && !w;
        clean &= last == hipSuccess;
        freed &= used == before;
        last = hipSuccess;
        ++refusals;
    }
    expect(refusals > 5 && refused, "uploads without room are refused");
    expect(freed, "and hold nothing");
    expect(clean, "and leave no error behind");
    limit = SIZE_MAX;
}

}  // namespace

int main() {
    aq_ctx *ctx = nullptr;
    expect(aq_ctx_create(0, nullptr, &ctx) == AQ_OK, "context");
    refused_uploads(ctx);
    const size_t before = used;
    expect(sampled(ctx, 8) == AQ_OK, "first call");
    const size_t eight = used - before;
    expect(sampled(ctx, 9) == AQ_OK && used - before >= 3 * eight && used - before < 3 * eight + 4096,
           "a buffer that grows doubles, and the old one stays");
    const size_t had = allocations;
    expect(sampled(ctx, 16) == AQ_OK && allocations == had, "within it nothing is allocated");

    // Room for what is needed, not for twice what there is.
    limit = used + 2 * eight + eight / 2;
    const size_t ran = launches;
    expect(sampled(ctx, 18) == AQ_OK, "what is needed is taken where its double cannot be had");
    expect(launches == ran + 4 && last == hipSuccess, "the call runs and leaves no error behind");
    limit = used;
    expect(sampled(ctx, 19) == AQ_E_NOMEM, "no room");
    expect(last == hipSuccess, "a refusal leaves no error behind");
    expect(sampled(ctx, 18) == AQ_OK, "the buffer before a refusal is still used");

    // As often as it takes, a little more each time.
    bool all = true;
    for (int64_t rows = 19; rows <= 256; ++rows) {
        limit = used + eight * static_cast<size_t>(rows) / 8 + eight / 16;
        all &= sampled(ctx, rows) == AQ_OK;
    }
    expect(all, "238 buffers, each a little larger");
    expect(aq_ctx_destroy(ctx) == AQ_OK && used == 0 && live.empty() && bad_frees == 0, "all are freed with the context, once");
    return failures != 0;
}
