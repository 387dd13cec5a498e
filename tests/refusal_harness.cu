// A context and handles without a device behind them, for calls that are refused before they reach one.
#include "serving.cuh"

extern "C" {
void* t_context(int capturing) {
    auto* c = new loom_b200_ctx();
    c->capturing = capturing != 0;
    return c;
}
void t_context_free(void* c) { delete static_cast<loom_b200_ctx*>(c); }
void* t_adapters(void* ctx, int slots, int rows, int cols, int max_rank) {
    auto* a = new loom_b200_adapters();
    a->ctx = static_cast<loom_b200_ctx*>(ctx);
    a->slots = slots;
    a->rows = rows;
    a->cols = cols;
    a->max_rank = max_rank;
    return a;
}
void t_adapters_free(void* a) { delete static_cast<loom_b200_adapters*>(a); }
void* t_kv8(void* ctx, int seqs, int heads, int dim) {
    auto* c = new loom_b200_kv8();
    c->ctx = static_cast<loom_b200_ctx*>(ctx);
    c->seqs = seqs;
    c->heads = heads;
    c->dim = dim;
    return c;
}
void t_kv8_free(void* c) { delete static_cast<loom_b200_kv8*>(c); }
}
