// An 8-bit cache's handle of any size without a device behind it.
#include "serving.cuh"

extern "C" {
void* t_context() { return new loom_b200_ctx(); }
void* t_kv8(void* ctx, int seqs, int max_len, int heads, int dim) {
    auto* c = new loom_b200_kv8();
    c->ctx = static_cast<loom_b200_ctx*>(ctx);
    c->seqs = seqs;
    c->max_len = max_len;
    c->heads = heads;
    c->dim = dim;
    c->blocks = max_len / kKvBlock > 0 ? max_len / kKvBlock : 1;
    c->dim_k = (dim + 31) / 32 * 32;
    return c;
}
}
