// C entries of attention over a 4-bit key-value cache: arguments and buffers
// are checked here, before anything runs.
#include <initializer_list>

#include "kv4_shapes.h"

using namespace smi;

namespace {

constexpr int kMaxRows = 1 << 24;
constexpr int64_t kMaxPlace = (int64_t)1 << 40;

int bad(sm_ctx *ctx, const char *what, const char *why) { return fail(ctx, SM_E_ARG, std::string(what) + ": " + why); }

int check_heads(sm_ctx *ctx, const char *what, int heads, int kv_heads, int dim) {
    if (kv_heads < 1 || heads < kv_heads || heads > 1024 || heads % kv_heads)
        return bad(ctx, what, "heads must be a multiple of kv_heads, 1 to 1024");
    if (dim < 8 || dim > 256 || dim % 8) return bad(ctx, what, "dim must be a multiple of 8, 8 to 256");
    return SM_OK;
}
int check_type(sm_ctx *ctx, const char *what, int type) {
    return type == SM_TYPE_F32 || type == SM_TYPE_BF16 ? SM_OK : bad(ctx, what, "type must be SM_TYPE_F32 or SM_TYPE_BF16");
}
int check_rows(sm_ctx *ctx, const char *what, int64_t tokens, int64_t heads) {
    return tokens >= 1 && tokens * heads <= kMaxRows ? SM_OK : bad(ctx, what, "tokens must be at least 1, tokens * heads at most 2^24");
}
// The view, or rows without gaps; the bytes that it reaches over. `apart`: rows and heads must not overlap.
int take_view(sm_ctx *ctx, const char *what, const int64_t *v, int tokens, int heads, int dim, int type, bool apart, Kv4View *view,
              uint64_t *bytes) {
    *view = {(int64_t)heads * dim, dim, 0};
    if (v) *view = {v[0], v[1], v[2]};
    for (int64_t n : {view->stride, view->head, view->offset})
        if (n < 0 || n > kMaxPlace) return bad(ctx, what, "a view's numbers must be 0 to 2^40");
    if (view->stride > kMaxPlace / tokens || view->head > kMaxPlace / heads) return bad(ctx, what, "a view reaches past 2^40 values");
    // one after another, rows with their heads or heads with their rows
    const bool rows = (heads == 1 || view->head >= dim) && (tokens == 1 || view->stride >= (heads - 1) * view->head + dim);
    const bool by_head = (tokens == 1 || view->stride >= dim) && (heads == 1 || view->head >= (tokens - 1) * view->stride + dim);
    if (apart && !rows && !by_head) return bad(ctx, what, "an output's rows overlap");
    *bytes = (uint64_t)((tokens - 1) * view->stride + (heads - 1) * view->head + view->offset + dim) * (type == SM_TYPE_BF16 ? 2 : 4);
    return SM_OK;
}
int check_sequences(sm_ctx *ctx, const char *what, int tokens, int count, int longest, int table_pages) {
    if (count < 1 || count > 32768) return bad(ctx, what, "count must be 1 to 32768");
    if (table_pages < 1 || (int64_t)count * table_pages > kMaxRows)
        return bad(ctx, what, "table_pages must be at least 1, count * table_pages at most 2^24");
    if (longest < 1 || longest > tokens) return bad(ctx, what, "longest must be 1 to tokens");
    return SM_OK;
}
int check_pool(sm_ctx *ctx, const char *what, int pages, int kv_heads, int dim, uint64_t *bytes) {
    if (pages < 1 || pages > kMaxRows) return bad(ctx, what, "pages must be 1 to 2^24");
    *bytes = pages * kv4_page_bytes(kv_heads, dim);
    return SM_OK;
}
// Distinct handles are distinct allocations.
int check_distinct(sm_ctx *ctx, const char *what, std::initializer_list<uint64_t> outputs,
                   std::initializer_list<uint64_t> inputs) {
    for (const uint64_t *o = outputs.begin(); o != outputs.end(); o++) {
        for (const uint64_t *p = outputs.begin(); p != o; p++)
            if (*o && *o == *p) return bad(ctx, what, "two outputs are one buffer");
        for (uint64_t i : inputs)
            if (*o && *o == i) return bad(ctx, what, "an output is a buffer that the call reads");
    }
    return SM_OK;
}
int need_sequences(sm_ctx *ctx, int count, int table_pages, uint64_t starts, uint64_t lengths, uint64_t table) {
    if (int rc = need(ctx, starts, ((uint64_t)count + 1) * 4, "starts")) return rc;
    if (int rc = need(ctx, lengths, (uint64_t)count * 4, "lengths")) return rc;
    return need(ctx, table, (uint64_t)count * table_pages * 4, "table");
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

int sm_qk_norm_rope(sm_ctx *ctx, uint64_t Q, const int64_t *q_view, uint64_t K, const int64_t *k_view, int type, int tokens,
                    int heads, int kv_heads, int dim, uint64_t q_gamma, uint64_t k_gamma, float eps, uint64_t Cos, uint64_t Sin,
                    int rotary, int context, uint64_t positions, uint64_t Yq, uint64_t Yk) {
    const char *what = "qk norm rope";
    if (!ctx) return SM_E_ARG;
    if (int rc = check_heads(ctx, what, heads, kv_heads, dim)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (int rc = check_rows(ctx, what, tokens, (int64_t)heads + kv_heads)) return rc;
    if (!(eps >= 0.0f)) return fail(ctx, SM_E_ARG, "epsilon must be >= 0");
    if (rotary < 2 || rotary > dim || rotary % 2) return bad(ctx, what, "rotary must be even, 2 to dim");
    if (context < 1) return bad(ctx, what, "context must be at least 1");
    QkNormRope a = {tokens, heads, kv_heads, dim, rotary, context, eps, (const float *)q_gamma, (const float *)k_gamma,
                    (const float *)Cos, (const float *)Sin, (const int *)positions, {}, {}};
    uint64_t q_bytes, k_bytes;
    if (int rc = take_view(ctx, what, q_view, tokens, heads, dim, type, false, &a.q_view, &q_bytes)) return rc;
    if (int rc = take_view(ctx, what, k_view, tokens, kv_heads, dim, type, false, &a.k_view, &k_bytes)) return rc;
    const uint64_t size = type == SM_TYPE_BF16 ? 2 : 4, table = (uint64_t)context * (rotary / 2) * 4;
    if (int rc = need(ctx, Q, q_bytes, "qk norm rope Q")) return rc;
    if (int rc = need(ctx, K, k_bytes, "qk norm rope K")) return rc;
    if (int rc = need(ctx, q_gamma, (uint64_t)dim * 4, "qk norm rope q_gamma")) return rc;
    if (int rc = need(ctx, k_gamma, (uint64_t)dim * 4, "qk norm rope k_gamma")) return rc;
    if (int rc = need(ctx, Cos, table, "qk norm rope Cos")) return rc;
    if (int rc = need(ctx, Sin, table, "qk norm rope Sin")) return rc;
    if (int rc = need(ctx, positions, (uint64_t)tokens * 4, "qk norm rope positions")) return rc;
    if (int rc = need(ctx, Yq, (uint64_t)tokens * heads * dim * size, "qk norm rope Yq")) return rc;
    if (int rc = need(ctx, Yk, (uint64_t)tokens * kv_heads * dim * size, "qk norm rope Yk")) return rc;
    if (int rc = check_distinct(ctx, what, {Yq, Yk}, {Q, K, q_gamma, k_gamma, Cos, Sin, positions})) return rc;
    Device device(ctx);
    return qk_norm_rope_launch(ctx, a, (const void *)Q, (const void *)K, (void *)Yq, (void *)Yk, type == SM_TYPE_BF16);
}

int sm_kv4_bytes(int pages, int kv_heads, int dim, uint64_t *bytes) {
    if (!bytes) return SM_E_ARG;
    if (int rc = check_heads(nullptr, "kv4 pool", kv_heads, kv_heads, dim)) return rc;
    return check_pool(nullptr, "kv4 pool", pages, kv_heads, dim, bytes);
}

int sm_kv4_write(sm_ctx *ctx, uint64_t K, const int64_t *k_view, uint64_t V, const int64_t *v_view, int type, int tokens,
                 int count, int longest, uint64_t starts, uint64_t lengths, uint64_t table, int table_pages, int kv_heads,
                 int dim, uint64_t pool, int pages) {
    const char *what = "kv4 write";
    if (!ctx) return SM_E_ARG;
    uint64_t pool_bytes, k_bytes, v_bytes;
    Kv4View kv, vv;
    if (int rc = check_heads(ctx, what, kv_heads, kv_heads, dim)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (int rc = check_rows(ctx, what, tokens, kv_heads)) return rc;
    if (int rc = check_sequences(ctx, what, tokens, count, longest, table_pages)) return rc;
    if (int rc = check_pool(ctx, what, pages, kv_heads, dim, &pool_bytes)) return rc;
    if (int rc = take_view(ctx, what, k_view, tokens, kv_heads, dim, type, false, &kv, &k_bytes)) return rc;
    if (int rc = take_view(ctx, what, v_view, tokens, kv_heads, dim, type, false, &vv, &v_bytes)) return rc;
    if (int rc = need(ctx, K, k_bytes, "kv4 write K")) return rc;
    if (int rc = need(ctx, V, v_bytes, "kv4 write V")) return rc;
    if (int rc = need_sequences(ctx, count, table_pages, starts, lengths, table)) return rc;
    if (int rc = need(ctx, pool, pool_bytes, "kv4 write pool")) return rc;
    if (int rc = check_distinct(ctx, what, {pool}, {K, V, starts, lengths, table})) return rc;
    Device device(ctx);
    return kv4_write_launch(ctx, (const void *)K, kv, (const void *)V, vv, type == SM_TYPE_BF16,
                            {count, tokens, longest, table_pages, (const int *)starts, (const int *)lengths, (const int *)table},
                            kv_heads, dim, (uint8_t *)pool, pages);
}

int sm_kv4_read(sm_ctx *ctx, uint64_t pool, int pages, int kv_heads, int dim, int tokens, int count, int longest, uint64_t starts,
                uint64_t lengths, uint64_t table, int table_pages, uint64_t K, const int64_t *k_view, uint64_t V,
                const int64_t *v_view, int type) {
    const char *what = "kv4 read";
    if (!ctx) return SM_E_ARG;
    uint64_t pool_bytes, k_bytes, v_bytes;
    Kv4View kv, vv;
    if (int rc = check_heads(ctx, what, kv_heads, kv_heads, dim)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (int rc = check_rows(ctx, what, tokens, kv_heads)) return rc;
    if (int rc = check_sequences(ctx, what, tokens, count, longest, table_pages)) return rc;
    if (int rc = check_pool(ctx, what, pages, kv_heads, dim, &pool_bytes)) return rc;
    if (int rc = take_view(ctx, what, k_view, tokens, kv_heads, dim, type, true, &kv, &k_bytes)) return rc;
    if (int rc = take_view(ctx, what, v_view, tokens, kv_heads, dim, type, true, &vv, &v_bytes)) return rc;
    if (int rc = need(ctx, pool, pool_bytes, "kv4 read pool")) return rc;
    if (int rc = need_sequences(ctx, count, table_pages, starts, lengths, table)) return rc;
    if (int rc = need(ctx, K, k_bytes, "kv4 read K")) return rc;
    if (int rc = need(ctx, V, v_bytes, "kv4 read V")) return rc;
    if (int rc = check_distinct(ctx, what, {K, V}, {pool, starts, lengths, table})) return rc;
    Device device(ctx);
    return kv4_read_launch(ctx, (const uint8_t *)pool, pages, kv_heads, dim,
                           {count, tokens, longest, table_pages, (const int *)starts, (const int *)lengths, (const int *)table},
                           (void *)K, kv, (void *)V, vv, type == SM_TYPE_BF16);
}

int sm_kv4_attention_workspace(int tokens, int count, int longest, int table_pages, int heads, int kv_heads, int dim,
                               uint64_t *bytes) {
    const char *what = "kv4 attention";
    if (!bytes) return SM_E_ARG;
    if (int rc = check_heads(nullptr, what, heads, kv_heads, dim)) return rc;
    if (int rc = check_rows(nullptr, what, tokens, heads)) return rc;
    if (int rc = check_sequences(nullptr, what, tokens, count, longest, table_pages)) return rc;
    *bytes = kv4_workspace({count, tokens, longest, table_pages, nullptr, nullptr, nullptr}, heads, kv_heads, dim);
    return SM_OK;
}

int sm_kv4_attention(sm_ctx *ctx, uint64_t Q, const int64_t *q_view, int type, int tokens, int count, int longest,
                     uint64_t starts, uint64_t lengths, uint64_t table, int table_pages, uint64_t pool, int pages, int heads,
                     int kv_heads, int dim, float scale, int window, uint64_t G, const int64_t *g_view, uint64_t Y,
                     uint64_t workspace, uint64_t workspace_bytes) {
    const char *what = "kv4 attention";
    if (!ctx) return SM_E_ARG;
    uint64_t pool_bytes, q_bytes, g_bytes;
    if (int rc = check_heads(ctx, what, heads, kv_heads, dim)) return rc;
    if (int rc = check_type(ctx, what, type)) return rc;
    if (int rc = check_rows(ctx, what, tokens, heads)) return rc;
    if (int rc = check_sequences(ctx, what, tokens, count, longest, table_pages)) return rc;
    if (int rc = check_pool(ctx, what, pages, kv_heads, dim, &pool_bytes)) return rc;
    if (!(scale > 0.0f && scale < 1e30f)) return bad(ctx, what, "scale must be > 0 and below 1e30");
    if (window < 0) return bad(ctx, what, "window must be >= 0");
    Kv4Attention a = {{count, tokens, longest, table_pages, (const int *)starts, (const int *)lengths, (const int *)table},
                      pages, heads, kv_heads, dim, kv4_window(window, table_pages), scale * 1.44269504088896340736f,
                      {}, {}, false, 0, 0, nullptr};
    if (int rc = take_view(ctx, what, q_view, tokens, heads, dim, type, false, &a.q_view, &q_bytes)) return rc;
    if (int rc = take_view(ctx, what, G ? g_view : nullptr, tokens, heads, dim, type, false, &a.g_view, &g_bytes)) return rc;
    a.vec = a.q_view.multiple_of(8);
    if (int rc = need(ctx, Q, q_bytes, "kv4 attention Q")) return rc;
    if (G)
        if (int rc = need(ctx, G, g_bytes, "kv4 attention G")) return rc;
    if (int rc = need_sequences(ctx, count, table_pages, starts, lengths, table)) return rc;
    if (int rc = need(ctx, pool, pool_bytes, "kv4 attention pool")) return rc;
    if (int rc = need(ctx, Y, (uint64_t)tokens * heads * dim * (type == SM_TYPE_BF16 ? 2 : 4), "kv4 attention Y")) return rc;
    const uint64_t ws = kv4_workspace(a.q, heads, kv_heads, dim);
    if (ws) {
        if (workspace_bytes < ws) return fail(ctx, SM_E_ARG, "workspace too small");
        if (int rc = need(ctx, workspace, ws, "workspace")) return rc;
        if (int rc = check_distinct(ctx, what, {workspace}, {Q, G, starts, lengths, table, pool, Y})) return rc;
    }
    if (int rc = check_distinct(ctx, what, {Y}, {Q, G, starts, lengths, table, pool})) return rc;
    Device device(ctx);
    return kv4_attention_launch(ctx, a, (const void *)Q, (const uint8_t *)pool, (const void *)G, (void *)Y, type == SM_TYPE_BF16,
                                (void *)workspace);
}

}  // extern "C"
