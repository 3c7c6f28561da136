// The stand-ins of kv4_entries_stub.cpp, with a launcher of the attention that
// keeps the window which it is given.
#include "../stratacuda_amd/csrc/internal.h"

#define kv4_attention_launch kv4_attention_launch_apart
#include "kv4_entries_stub.cpp"
#undef kv4_attention_launch

static int window = -1;

namespace smi {
int kv4_attention_launch(sm_ctx *ctx, const Kv4Attention &a, const void *, const uint8_t *, const void *, void *, bool, void *) {
    return window = a.window, launch(ctx);
}
}  // namespace smi

extern "C" int stub_window() { return window; }
