// Stand-ins for what the C entries of attention over a 4-bit cache call, so
// that their checks run without a GPU: a context with the buffers that a test
// names, and launchers that count. Built with csrc/kv4.cpp.
#include <hip/hip_runtime.h>

#include "../stratacuda_amd/csrc/internal.h"

static int launches = 0, device = 0;

namespace smi {
int fail(sm_ctx *ctx, int code, const std::string &msg) {
    if (ctx) ctx->error = msg;
    return code;
}
int need(sm_ctx *ctx, uint64_t handle, uint64_t bytes, const char *what) {
    auto it = ctx->buffers.find(handle);
    if (it == ctx->buffers.end()) return fail(ctx, SM_E_HANDLE, std::string(what) + ": not a live buffer of this context");
    return it->second < bytes ? fail(ctx, SM_E_BOUNDS, what) : SM_OK;
}
// Every launch finds the context's device current.
static int launch(sm_ctx *ctx) { return device == ctx->device ? (launches++, SM_OK) : SM_E_HIP; }
int qk_norm_rope_launch(sm_ctx *ctx, const QkNormRope &, const void *, const void *, void *, void *, bool) { return launch(ctx); }
int kv4_write_launch(sm_ctx *ctx, const void *, const Kv4View &, const void *, const Kv4View &, bool, const Kv4Sequences &, int, int,
                     uint8_t *, int) {
    return launch(ctx);
}
int kv4_read_launch(sm_ctx *ctx, const uint8_t *, int, int, int, const Kv4Sequences &, void *, const Kv4View &, void *, const Kv4View &,
                    bool) {
    return launch(ctx);
}
int kv4_attention_launch(sm_ctx *ctx, const Kv4Attention &, const void *, const uint8_t *, const void *, void *, bool, void *) {
    return launch(ctx);
}
}  // namespace smi

// Two devices, of which one is current.
extern "C" hipError_t hipGetDevice(int *d) { return *d = device, hipSuccess; }
extern "C" hipError_t hipSetDevice(int d) { return device = d, hipSuccess; }

extern "C" {
sm_ctx *stub_context() {
    sm_ctx *ctx = new sm_ctx();
    ctx->device = 1;
    return ctx;
}
void stub_free(sm_ctx *ctx) { delete ctx; }
void stub_buffer(sm_ctx *ctx, uint64_t handle, uint64_t bytes) { ctx->buffers[handle] = bytes; }
const char *stub_error(sm_ctx *ctx) { return ctx->error.c_str(); }
int stub_launches() { return launches; }
int stub_device() { return device; }
}
