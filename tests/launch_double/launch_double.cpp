// Stands in for the context and for the HIP runtime's launches, so that tests without a GPU can see which kernels the
// network-block entry points (rt_block.hip) launch, with which grids and plans, and which device they make current.  Linked
// with -Bsymbolic into a library of its own, loaded only by tests; nothing in it reaches a GPU.
#include <cxxabi.h>
#include <stdio.h>
#include <stdlib.h>
#include <map>
#include <string>
#include "../../roundtrip_amd/csrc/rt_block.hpp"

struct rt_ctx {
    std::string err;
    int device, cus;
};

namespace {
struct State {
    std::map<const void*, std::string> kernels;      // by the handle that a launch names
    std::string calls;                               // one line a call
    int current = 0, launches = 0, fail_at = -1;     // fail_at: the launch that fails
    hipError_t last = hipSuccess;
    dim3 grid, block;
    size_t shmem = 0;
    hipStream_t stream = nullptr;
};
State& st() {                                        // made on first use: kernels are registered by static constructors
    static State s;
    return s;
}
}  // namespace

void rt_ctx_view(const rt_ctx* ctx, RtCtxView* out) {
    out->device = ctx->device;
    out->cu_count = ctx->cus;
    out->stream = nullptr;
}

int rt_ctx_fail(rt_ctx* ctx, int code, const char* msg) {
    ctx->err = msg;
    return code;
}

extern "C" {

hipError_t hipGetDevice(int* d) {
    *d = st().current;
    return hipSuccess;
}

hipError_t hipSetDevice(int d) {
    st().calls += "device " + std::to_string(d) + "\n";
    st().current = d;
    return hipSuccess;
}

hipError_t hipGetLastError() {
    const hipError_t e = st().last;
    st().last = hipSuccess;
    return e;
}

const char* hipGetErrorString(hipError_t) { return "an error of the double"; }

void** __hipRegisterFatBinary(const void*) {
    static void* handle = nullptr;
    return &handle;
}

void __hipUnregisterFatBinary(void**) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}

void __hipRegisterFunction(void**, const void* handle, char*, const char* name, unsigned, void*, void*, dim3*, dim3*, int*) {
    int rc = 0;
    char* plain = abi::__cxa_demangle(name, nullptr, nullptr, &rc);
    std::string s = rc == 0 ? plain : name;
    free(plain);
    for (const char* drop : {"rt_block::", "(anonymous namespace)::", "void "})
        for (size_t at; (at = s.find(drop)) != std::string::npos;) s.erase(at, std::string(drop).size());
    st().kernels[handle] = s.substr(0, s.rfind('('));
}

hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shmem, hipStream_t stream) {
    st().grid = grid;
    st().block = block;
    st().shmem = shmem;
    st().stream = stream;
    return hipSuccess;
}

hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shmem, hipStream_t* stream) {
    *grid = st().grid;
    *block = st().block;
    *shmem = st().shmem;
    *stream = st().stream;
    return hipSuccess;
}

// "launch <kernel> | grid x y z block n [| splits a each b steps c]": of a matrix product, K's steps and how they are split
hipError_t hipLaunchKernel(const void* handle, dim3 grid, dim3 block, void** args, size_t, hipStream_t) {
    State& s = st();
    const std::string& name = s.kernels[handle];
    char line[400];
    snprintf(line, sizeof line, "launch %s | grid %u %u %u block %u", name.c_str(), grid.x, grid.y, grid.z, block.x);
    s.calls += line;
    if (name.compare(0, 4, "gemm") == 0) {
        const rt_block::GemmArgs& a = *(const rt_block::GemmArgs*)args[0];
        snprintf(line, sizeof line, " | splits %d each %d steps %d", a.splits, a.per_split, a.nk * a.nseg);
        s.calls += line;
    }
    s.calls += " on device " + std::to_string(s.current) + "\n";
    if (s.launches++ == s.fail_at) s.last = hipErrorLaunchFailure;
    return s.last;
}

rt_ctx* double_ctx(int device, int cus) {
    rt_ctx* c = new rt_ctx();
    c->device = device;
    c->cus = cus;
    return c;
}
const char* double_error(rt_ctx* ctx) { return ctx->err.c_str(); }

// Forgets the calls, makes `current` the current device and lets launch number fail_at (from 0; -1: none) fail.
void double_reset(int current, int fail_at) {
    st().calls.clear();
    st().current = current;
    st().launches = 0;
    st().fail_at = fail_at;
    st().last = hipSuccess;
}
int double_current() { return st().current; }
const char* double_calls() { return st().calls.c_str(); }

// Every kernel there is, a line each.
const char* double_kernels() {
    static std::string all;
    all.clear();
    for (const auto& k : st().kernels) all += k.second + "\n";
    return all.c_str();
}
}
