// Stands in for the context of librt_is.so, so that the argument checks of the network-block entry points (rt_block.hip) can
// be tested where there is no GPU: linked with that translation unit into a library of its own, loaded only by tests.  Calls
// that pass every check end at the first HIP call, with an error.
#include <stdlib.h>
#include <string>
#include "../../roundtrip_amd/csrc/rt_internal.hpp"

struct rt_ctx {
    std::string err;
};

void rt_ctx_view(const rt_ctx*, RtCtxView* out) {
    out->device = 1 << 20;      // no such device: a call that passes its checks ends here, GPU or not
    out->cu_count = 256;
    out->stream = nullptr;
}

int rt_ctx_fail(rt_ctx* ctx, int code, const char* msg) {
    ctx->err = msg;
    return code;
}

extern "C" {
rt_ctx* double_ctx() { return new rt_ctx(); }
const char* double_error(rt_ctx* ctx) { return ctx->err.c_str(); }
}
