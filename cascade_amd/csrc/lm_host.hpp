// What the host sides of the language-model operators share: the calling thread's last error, rounding up, workspaces, limits of launches.
#pragma once
#include "../../include/cascade_lm.h"

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

namespace lm {

inline thread_local char g_err[512] = "";

inline int fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

inline int launched(const char* who)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? CSA_OK : fail(CSA_ERR_HIP, "%s: a launch failed: %s", who, hipGetErrorString(e));
}

inline uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }
inline uint64_t parts_of(uint64_t x, uint64_t size) { return (x + size - 1) / size; }
// HIP starts fewer than 2^32 threads along an axis. What would need more is refused before the call's first launch.
inline bool launchable(uint64_t groups, uint64_t threads) { return groups < (1ull << 32) / threads; }
inline bool aligned(const void* p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Hands out the pieces of a workspace, or only adds them up.
struct Carver {
    char* base;
    uint64_t used = 0;
    template <class T>
    T* take(uint64_t count)
    {
        T* at = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used = up(used + count * sizeof(T), 256);
        return at;
    }
};

inline int check_work(const char* who, const void* work, uint64_t have, uint64_t need)
{
    if (need && (!work || !aligned(work, 256)))
        return fail(CSA_ERR_ARG, "%s: the workspace is null or not aligned to 256 bytes", who);
    if (have < need)
        return fail(CSA_ERR_ARG, "%s: a workspace of %llu bytes where %llu are needed", who, (unsigned long long)have, (unsigned long long)need);
    return CSA_OK;
}

} // namespace lm
