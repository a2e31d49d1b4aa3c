// A CUDA runtime made of notes: what the token operators' host code asks of it is written down, and any call can be made to fail. The
// operators' sources are linked against this instead of the runtime library; no kernel runs and no device is needed.
#pragma once

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <string>
#include <vector>

#include <cuda.h>
#include <cuda_runtime.h>

namespace fake {

enum Kind { LAUNCH, CLEAR, RECORD, WAIT };  // CLEAR: an asynchronous memset
struct Op {
    Kind kind;
    cudaStream_t stream;
    const void* what;  // the kernel, the memory or the event
    bool captured;     // into a graph: nothing runs
};

// One set for each thread: a lock here would order the threads, and hide what the library shares between them without one.
inline thread_local std::vector<Op> ops;                // what has been enqueued
inline thread_local int fail_at = -1, fail_for = 1;     // this many enqueueing calls from now, so many in a row fail
inline thread_local size_t memory = ~size_t(0);         // the largest allocation that succeeds
inline thread_local size_t allocated = 0;               // bytes asked for and got
inline thread_local std::set<cudaStream_t> capturing;
inline thread_local cudaError_t last = cudaSuccess;
inline thread_local std::string message;                // of the library's last error

inline cudaError_t result(cudaError_t e) {
    if (e != cudaSuccess) last = e;
    return e;
}
inline cudaError_t enqueue(Kind k, cudaStream_t s, const void* what) {
    if (fail_at == 0) {
        if (--fail_for == 0) fail_at = -1, fail_for = 1;
        return result(cudaErrorLaunchOutOfResources);
    }
    if (fail_at > 0) fail_at--;
    ops.push_back({k, s, what, capturing.count(s) != 0});
    return cudaSuccess;
}
inline CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                       CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}

}  // namespace fake

namespace oxz {
int32_t fail(int32_t status, const char* fmt, ...) {
    char text[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    fake::message = text;
    return status;
}
}  // namespace oxz

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetLastError(void) { const cudaError_t e = fake::last; fake::last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t) { return "fake error"; }
cudaError_t cudaMalloc(void** p, size_t n) {
    if (n > fake::memory || !(*p = aligned_alloc(256, (n + 255) / 256 * 256))) return fake::result(cudaErrorMemoryAllocation);
    fake::allocated += n;
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { *p = calloc(1, n); return cudaSuccess; }
cudaError_t cudaHostGetDevicePointer(void** d, void* p, unsigned) { *d = p; return cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaMemset(void*, int, size_t) { return cudaSuccess; }
cudaError_t cudaDeviceSynchronize(void) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t*) { *n = 4; return cudaSuccess; }
cudaError_t cudaGetDriverEntryPointByVersion(const char*, void** fn, unsigned, unsigned long long, cudaDriverEntryPointQueryResult* st) {
    *fn = (void*)&fake::encode;
    *st = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { *e = (cudaEvent_t)malloc(1); return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t e) { free((void*)e); return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t s, cudaStreamCaptureStatus* st) {
    *st = fake::capturing.count(s) ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { return fake::enqueue(fake::RECORD, s, e); }
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned) { return fake::enqueue(fake::WAIT, s, e); }
cudaError_t cudaMemsetAsync(void* p, int, size_t, cudaStream_t s) { return fake::enqueue(fake::CLEAR, s, p); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* cfg, const void* f, void**) { return fake::enqueue(fake::LAUNCH, cfg->stream, f); }
cudaError_t cudaLaunchKernel(const void* f, dim3, dim3, void**, size_t, cudaStream_t s) { return fake::enqueue(fake::LAUNCH, s, f); }
// what the compiler's own host code calls
static thread_local cudaStream_t pushed_stream;
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t s) { pushed_stream = s; return 0; }
cudaError_t __cudaPopCallConfiguration(dim3* g, dim3* b, size_t* n, void* s) {
    *g = *b = dim3(1);
    *n = 0;
    *static_cast<cudaStream_t*>(s) = pushed_stream;
    return cudaSuccess;
}
void** __cudaRegisterFatBinary(void*) { static void* handle; return &handle; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
char __cudaInitModule(void**) { return 1; }
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
}
