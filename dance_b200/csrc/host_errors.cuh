// host_errors.cuh -- status codes with a message and the launch counter: what
// every C entry point of the library reports through.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

namespace dance
{

// ---------------------------------------------------------------- errors
extern thread_local char g_err[512];
extern std::atomic<uint64_t> g_launches;

inline int fail(int code, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    fprintf(stderr, "[dance_b200] %s\n", g_err);
    return code;
}

#define DANCE_CUDA(call)                                                                                        \
    do                                                                                                          \
    {                                                                                                           \
        cudaError_t e__ = (call);                                                                               \
        if (e__ != cudaSuccess)                                                                                 \
            return fail(-2, "CUDA error %s at %s:%d (%s)", cudaGetErrorString(e__), __FILE__, __LINE__, #call); \
    } while (0)

#define DANCE_LAUNCHED()                                                                                        \
    do                                                                                                          \
    {                                                                                                           \
        g_launches.fetch_add(1, std::memory_order_relaxed);                                                    \
        cudaError_t e__ = cudaGetLastError();                                                                   \
        if (e__ != cudaSuccess)                                                                                 \
            return fail(-2, "kernel launch failed: %s at %s:%d", cudaGetErrorString(e__), __FILE__, __LINE__);  \
    } while (0)

inline cudaStream_t as_stream(void *s) { return reinterpret_cast<cudaStream_t>(s); }

} // namespace dance
