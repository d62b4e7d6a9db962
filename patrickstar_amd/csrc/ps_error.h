// The text behind ps_last_error(), shared by the library's sources.
#ifndef PS_ERROR_H
#define PS_ERROR_H

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

namespace ps_detail {

inline thread_local char error_text[512] = "";

}  // namespace ps_detail

namespace {

int fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(ps_detail::error_text, sizeof(ps_detail::error_text), fmt, ap);
    va_end(ap);
    return code;
}

int hip_fail(hipError_t e, const char* what)
{
    return fail(-(int)e, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace

#define PS_HIP(call)                                      \
    do {                                                  \
        hipError_t e_ = (call);                           \
        if (e_ != hipSuccess) return hip_fail(e_, #call); \
    } while (0)

#endif  // PS_ERROR_H
