// rt_internal.hpp — what the translation units of librt_is.so share of a context.  Nothing here is exported.
#pragma once
#include <hip/hip_runtime.h>
#include "../../include/rt_is.h"

#define RT_HIDDEN __attribute__((visibility("hidden")))

// What a kernel launch needs to know of a context.
struct RtCtxView {
    int device;
    int cu_count;
    hipStream_t stream;
};
RT_HIDDEN void rt_ctx_view(const rt_ctx* ctx, RtCtxView* out);
RT_HIDDEN int rt_ctx_fail(rt_ctx* ctx, int code, const char* msg);   // sets rt_last_error's text, returns code
