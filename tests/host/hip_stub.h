/* hip_stub.h - as much of the HIP runtime as k3g_host.h uses, for the host: two devices, calls
 * that fail on request, and a last error that stays until it is read, as the runtime's does (test
 * infrastructure; never linked into the library). The test copies this file as
 * hip/hip_runtime.h. */
#pragma once
#include <stddef.h>

typedef enum { hipSuccess = 0, hipErrorInvalidValue = 1, hipErrorInvalidConfiguration = 9 } hipError_t;
typedef struct StubStream { int device; } *hipStream_t;
typedef int hipDevice_t;
struct dim3 {
    unsigned x, y, z;
    dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};

struct Stub {
    hipError_t last, launch, set, stream;      /* the last error; what each call returns */
    int device, launches;
};
static Stub stub;

static hipError_t stub_end(hipError_t e)
{
    if (e != hipSuccess) stub.last = e;
    return e;
}
static inline hipError_t hipGetLastError(void)
{
    const hipError_t e = stub.last;
    stub.last = hipSuccess;
    return e;
}
static inline const char *hipGetErrorString(hipError_t) { return "on request"; }
static inline hipError_t hipGetDevice(int *d) { *d = stub.device; return hipSuccess; }
static inline hipError_t hipSetDevice(int d)
{
    if (stub.set == hipSuccess) stub.device = d;
    return stub_end(stub.set);
}
static inline hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t *d)
{
    *d = s->device;
    return stub_end(stub.stream);
}
static inline hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t)
{
    ++stub.launches;
    return stub_end(stub.launch);
}
