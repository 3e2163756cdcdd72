/* host_guard.cpp - k3g_host.h on the stub runtime: prints "ok <case>" for each case that holds. */
#include "k3g_host.h"

static void kernel(int, float) {}

static void said(const char *name, bool holds) { printf("%s %s\n", holds ? "ok" : "FAILS", name); }

int main()
{
    /* a failed launch is reported once, by its own call */
    stub = {};
    stub.launch = hipErrorInvalidConfiguration;
    said("failed launch is reported", k3h_launch("who", kernel, dim3(1), dim3(64), (hipStream_t)nullptr, 1, 2.0f) == -1);
    said("failed launch leaves no error behind", hipGetLastError() == hipSuccess);

    /* an earlier call's error is neither taken for a launch's own nor taken from its owner */
    stub = {};
    stub.last = hipErrorInvalidValue;
    said("launch after another's error", k3h_launch("who", kernel, dim3(1), dim3(64), (hipStream_t)nullptr, 1, 2.0f) == 0 &&
                                             stub.launches == 1);
    said("another's error stays", hipGetLastError() == hipErrorInvalidValue);

    /* the stream's device is current for as long as the guard lives */
    StubStream there = {1};
    stub = {};
    {
        K3hOn on(&there);
        said("the stream's device is current", on.ok && stub.device == 1);
    }
    said("the caller's device is current again", stub.device == 0 && stub.last == hipSuccess);

    /* a stream whose device cannot be told or made current */
    stub = {};
    stub.stream = hipErrorInvalidValue;
    {
        fprintf(stderr, "told:");
        K3hOn on(&there);
        said("a stream without a device is refused", !on.ok && stub.device == 0);
    }
    said("and leaves no error behind", hipGetLastError() == hipSuccess);
    stub = {};
    stub.set = hipErrorInvalidValue;
    {
        fprintf(stderr, "current:");
        K3hOn on(&there);
        said("a device that cannot be current is refused", !on.ok && stub.device == 0);
    }
    said("and leaves no error behind it", hipGetLastError() == hipSuccess);
    return 0;
}
