// Stand-ins for what the C entries of the 8-bit operators call, so that their
// checks run without a GPU: a context with the buffers that a test names, and
// launchers that count. Built with csrc/f8.cpp.
#include <hip/hip_runtime.h>

#include "../stratacuda_amd/csrc/internal.h"

static int launches = 0;

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
int f8_quantize_launch(sm_ctx *, const void *, bool, int, int, int, uint8_t *, uint8_t *) { return launches++, SM_OK; }
int f8_norm_launch(sm_ctx *, const void *, bool, const float *, const float *, float, int, int, float *, uint8_t *, uint8_t *) {
    return launches++, SM_OK;
}
int f8_project_launch(sm_ctx *, const F8Operand &, int, int, const F8Operand &, int, const float *, void *, bool, int64_t,
                      int64_t) {
    return launches++, SM_OK;
}
uint64_t f8_gate_up_workspace(int tokens, int ff) { return (uint64_t)tokens * ff * 4; }
int f8_gate_up_launch(sm_ctx *, const F8Operand &, int, int, const F8Operand &, const F8Operand &, int, uint8_t *, uint8_t *,
                      void *) {
    return launches++, SM_OK;
}
}  // namespace smi

// One device, current.
extern "C" hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }

extern "C" {
sm_ctx *stub_context() { return new sm_ctx(); }
void stub_free(sm_ctx *ctx) { delete ctx; }
void stub_buffer(sm_ctx *ctx, uint64_t handle, uint64_t bytes) { ctx->buffers[handle] = bytes; }
const char *stub_error(sm_ctx *ctx) { return ctx->error.c_str(); }
int stub_launches() { return launches; }
}
