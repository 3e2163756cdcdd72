/* k3g_host.h - host-side helpers of the entry points that take a stream and no context. */
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

/* The stream's device is the current one while this lives (kernels are launched on the device
 * of their stream, whichever is current in the caller's thread); a null stream is the current
 * device's. */
struct K3hOn {
    hipStream_t st;
    bool ok;
    int back;
    explicit K3hOn(void *stream) : st((hipStream_t)stream), ok(true), back(-1)
    {
        if (!st) return;
        hipDevice_t on;
        int cur;
        if (hipStreamGetDevice(st, &on) != hipSuccess || hipGetDevice(&cur) != hipSuccess) {
            refuse("told");
        } else if (on != cur) {
            if (hipSetDevice(on) == hipSuccess) back = cur;
            else refuse("made the current one");
        }
    }
    ~K3hOn()
    {
        if (back >= 0) (void)hipSetDevice(back);
    }
    K3hOn(const K3hOn &) = delete;
    K3hOn &operator=(const K3hOn &) = delete;

private:
    void refuse(const char *what)
    {
        (void)hipGetLastError();
        fprintf(stderr, "k3moe: the stream's device cannot be %s\n", what);
        ok = false;
    }
};

static inline bool k3h_misaligned(const void *p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

/* One launch and its own status (not an earlier call's error, which hipGetLastError would
 * give): 0, or -1 with a message. The runtime keeps a failed launch as its last error, which a later
 * call that asks for it would take for its own: it is read here. */
template <typename... A>
static inline int k3h_launch(const char *who, void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t st,
                             A... a)
{
    void *args[] = {(void *)&a...};
    const hipError_t e = hipLaunchKernel((const void *)kernel, grid, block, args, 0, st);
    if (e == hipSuccess) return 0;
    (void)hipGetLastError();
    fprintf(stderr, "%s: launch failed: %s\n", who, hipGetErrorString(e));
    return -1;
}
