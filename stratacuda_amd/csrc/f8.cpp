// C entries of the 8-bit floating-point operators: arguments and buffers are
// checked here, before anything runs.
#include <initializer_list>

#include "internal.h"

using namespace smi;

namespace {

constexpr int kMaxDim = 1 << 21;
constexpr int64_t kMaxValues = (int64_t)1 << 33;

int check_shape(sm_ctx *ctx, const char *what, int64_t rows, int64_t cols) {
    if (rows < 1 || cols < 1 || rows > kMaxDim || cols > kMaxDim || rows * cols > kMaxValues)
        return fail(ctx, SM_E_ARG, std::string(what) + ": dimensions must be 1 to 2^21 and their product at most 2^33");
    return SM_OK;
}
int check_type(sm_ctx *ctx, const char *what, int type) {
    if (type != SM_TYPE_F32 && type != SM_TYPE_BF16)
        return fail(ctx, SM_E_ARG, std::string(what) + ": type must be SM_TYPE_F32 or SM_TYPE_BF16");
    return SM_OK;
}
int need_f8(sm_ctx *ctx, const char *what, uint64_t codes, uint64_t scales, int rows, int cols, int block_rows) {
    const F8Layout L = f8_layout(rows, cols, block_rows);
    if (int rc = need(ctx, codes, L.codes, what)) return rc;
    return need(ctx, scales, L.scales, (std::string(what) + " scales").c_str());
}
// Distinct handles are distinct allocations.
int check_distinct(sm_ctx *ctx, const char *what, std::initializer_list<uint64_t> outputs,
                   std::initializer_list<uint64_t> inputs) {
    for (const uint64_t *o = outputs.begin(); o != outputs.end(); o++) {
        for (const uint64_t *p = outputs.begin(); p != o; p++)
            if (*o && *o == *p) return fail(ctx, SM_E_ARG, std::string(what) + ": two outputs are one buffer");
        for (uint64_t i : inputs)
            if (*o && *o == i) return fail(ctx, SM_E_ARG, std::string(what) + ": an output is a buffer that the call reads");
    }
    return SM_OK;
}

// The context's device for the launches of one call.
class Device {
  public:
    explicit Device(sm_ctx *ctx) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = ctx->device;
        if (before_ != ctx->device) (void)hipSetDevice(ctx->device);
        else before_ = -1;
    }
    ~Device() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }

  private:
    int before_ = -1;
};

}  // namespace

extern "C" {

int sm_f8_bytes(int rows, int cols, int block_rows, uint64_t *codes, uint64_t *scales) {
    if (!codes || !scales || (block_rows != 1 && block_rows != 128)) return SM_E_ARG;
    if (int rc = check_shape(nullptr, "f8 matrix", rows, cols)) return rc;
    const F8Layout L = f8_layout(rows, cols, block_rows);
    *codes = L.codes;
    *scales = L.scales;
    return SM_OK;
}

int sm_f8_quantize(sm_ctx *ctx, uint64_t X, int type, int rows, int cols, int block_rows, uint64_t codes,
                   uint64_t scales) {
    const char *what = "f8 quantize";
    if (!ctx) return SM_E_ARG;
    if (int rc = check_shape(ctx, what, rows, cols)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (block_rows != 1 && block_rows != 128) return fail(ctx, SM_E_ARG, "f8 quantize: block_rows must be 1 or 128");
    if (int rc = need(ctx, X, (uint64_t)rows * cols * (type == SM_TYPE_BF16 ? 2 : 4), "f8 quantize X")) return rc;
    if (int rc = need_f8(ctx, "f8 quantize codes", codes, scales, rows, cols, block_rows)) return rc;
    if (int rc = check_distinct(ctx, what, {codes, scales}, {X})) return rc;
    Device device(ctx);
    return f8_quantize_launch(ctx, (const void *)X, type == SM_TYPE_BF16, rows, cols, block_rows, (uint8_t *)codes,
                              (uint8_t *)scales);
}

int sm_f8_norm(sm_ctx *ctx, uint64_t X, int type, uint64_t R, uint64_t gamma, float eps, int rows, int cols, uint64_t H,
               uint64_t codes, uint64_t scales) {
    const char *what = "f8 norm";
    if (!ctx) return SM_E_ARG;
    if (int rc = check_shape(ctx, what, rows, cols)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (!(eps >= 0.0f)) return fail(ctx, SM_E_ARG, "epsilon must be >= 0");
    const uint64_t values = (uint64_t)rows * cols;
    if (int rc = need(ctx, X, values * (type == SM_TYPE_BF16 ? 2 : 4), "f8 norm X")) return rc;
    if (R)
        if (int rc = need(ctx, R, values * 4, "f8 norm R")) return rc;
    if (int rc = need(ctx, gamma, (uint64_t)cols * 4, "f8 norm gamma")) return rc;
    if (H)
        if (int rc = need(ctx, H, values * 4, "f8 norm H")) return rc;
    if (int rc = need_f8(ctx, "f8 norm codes", codes, scales, rows, cols, 1)) return rc;
    if (int rc = check_distinct(ctx, what, {codes, scales, H}, {gamma})) return rc;
    if (int rc = check_distinct(ctx, what, {codes, scales}, {X, R})) return rc;
    if (H && H == X && type == SM_TYPE_BF16) return fail(ctx, SM_E_ARG, "f8 norm: H may be X only where X is f32");
    Device device(ctx);
    return f8_norm_launch(ctx, (const void *)X, type == SM_TYPE_BF16, (const float *)R, (const float *)gamma, eps, rows,
                          cols, (float *)H, (uint8_t *)codes, (uint8_t *)scales);
}

int sm_f8_project(sm_ctx *ctx, uint64_t X, uint64_t x_scales, int tokens, int cols, uint64_t W, uint64_t w_scales,
                  int rows, uint64_t R, uint64_t Y, int type, int64_t stride, int64_t offset) {
    const char *what = "f8 project";
    if (!ctx) return SM_E_ARG;
    if (int rc = check_shape(ctx, what, tokens, cols)) return rc;
    if (int rc = check_shape(ctx, what, rows, cols)) return rc;
    if (int rc = check_shape(ctx, what, tokens, rows)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (offset < 0 || stride < rows || offset > kMaxValues || stride > kMaxValues / tokens)
        return fail(ctx, SM_E_ARG, "f8 project: offset must be >= 0, stride >= rows and tokens * stride at most 2^33");
    if (R && type == SM_TYPE_BF16) return fail(ctx, SM_E_ARG, "f8 project: a residual needs an f32 output");
    if (int rc = need_f8(ctx, "f8 project X", X, x_scales, tokens, cols, 1)) return rc;
    if (int rc = need_f8(ctx, "f8 project W", W, w_scales, rows, cols, 128)) return rc;
    const uint64_t end = (uint64_t)((tokens - 1) * stride + offset + rows) * (type == SM_TYPE_BF16 ? 2 : 4);
    if (int rc = need(ctx, Y, end, "f8 project Y")) return rc;
    if (R)
        if (int rc = need(ctx, R, end, "f8 project R")) return rc;
    if (int rc = check_distinct(ctx, what, {Y}, {X, x_scales, W, w_scales})) return rc;
    Device device(ctx);
    return f8_project_launch(ctx, {(const uint8_t *)X, (const uint8_t *)x_scales}, tokens, cols,
                             {(const uint8_t *)W, (const uint8_t *)w_scales}, rows, (const float *)R, (void *)Y,
                             type == SM_TYPE_BF16, stride, offset);
}

int sm_f8_gate_up_workspace(int tokens, int ff, uint64_t *bytes) {
    if (!bytes) return SM_E_ARG;
    if (int rc = check_shape(nullptr, "f8 gate_up", tokens, ff)) return rc;
    *bytes = f8_gate_up_workspace(tokens, ff);
    return SM_OK;
}

int sm_f8_gate_up(sm_ctx *ctx, uint64_t X, uint64_t x_scales, int tokens, int cols, uint64_t Wg, uint64_t wg_scales,
                  uint64_t Wu, uint64_t wu_scales, int ff, uint64_t codes, uint64_t scales, uint64_t workspace,
                  uint64_t workspace_bytes) {
    const char *what = "f8 gate_up";
    if (!ctx) return SM_E_ARG;
    if (int rc = check_shape(ctx, what, tokens, cols)) return rc;
    if (int rc = check_shape(ctx, what, ff, cols)) return rc;
    if (int rc = check_shape(ctx, what, tokens, ff)) return rc;
    if (int rc = need_f8(ctx, "f8 gate_up X", X, x_scales, tokens, cols, 1)) return rc;
    if (int rc = need_f8(ctx, "f8 gate_up Wg", Wg, wg_scales, ff, cols, 128)) return rc;
    if (int rc = need_f8(ctx, "f8 gate_up Wu", Wu, wu_scales, ff, cols, 128)) return rc;
    if (int rc = need_f8(ctx, "f8 gate_up codes", codes, scales, tokens, ff, 1)) return rc;
    const uint64_t ws = f8_gate_up_workspace(tokens, ff);
    if (workspace_bytes < ws) return fail(ctx, SM_E_ARG, "workspace too small");
    if (int rc = need(ctx, workspace, ws, "workspace")) return rc;
    if (int rc = check_distinct(ctx, what, {codes, scales, workspace}, {X, x_scales, Wg, wg_scales, Wu, wu_scales}))
        return rc;
    Device device(ctx);
    return f8_gate_up_launch(ctx, {(const uint8_t *)X, (const uint8_t *)x_scales}, tokens, cols,
                             {(const uint8_t *)Wg, (const uint8_t *)wg_scales},
                             {(const uint8_t *)Wu, (const uint8_t *)wu_scales}, ff, (uint8_t *)codes, (uint8_t *)scales,
                             (void *)workspace);
}

}  // extern "C"
