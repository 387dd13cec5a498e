// serving.cuh -- what serving several requests on one decoder keeps: the 8-bit cache of keys and values, adapters.
#pragma once
#include "common.cuh"

constexpr int kKvBlock = 64;

struct loom_b200_kv8 {
    loom_b200_ctx* ctx = nullptr;
    int seqs = 0, max_len = 0, heads = 0, dim = 0;
    int blocks = 0;               // per sequence: whole ones that max_len positions can have
    int dim_k = 0, dim_v = 0;     // dimensions of the codes: multiples of 32 and of 8
    int dim_o = 0;                // of the open rows: a multiple of 4
    uint8_t *k = nullptr, *v = nullptr;      // [seqs][heads][blocks][64 * dim_k or dim_v]
    float *k_top = nullptr, *v_top = nullptr;  // [seqs][heads][blocks] largest |x|
    float *k_open = nullptr, *v_open = nullptr;  // [seqs][heads][2][64][dim_o]: rows of the open block and of the one in front, by the block's parity
    int* placed = nullptr;        // [seqs][heads][keys, values][2] which blocks those are
    void* work = nullptr;         // partial results of attention that several CTAs share, and arrival counters (zero between launches)
    size_t work_bytes = 0;
};

struct loom_b200_adapters {
    loom_b200_ctx* ctx = nullptr;
    int slots = 0, rows = 0, cols = 0, max_rank = 0, dtype = 0;
    int rank_pad = 0, cols_pad = 0, rows_pad = 0;  // multiples of 16, 32 and 16; what they add is zero
    void *down = nullptr, *up = nullptr;  // [slots][rank_pad][cols_pad], [slots][rows_pad][rank_pad]
    int* rank = nullptr;                  // [slots], 0: empty
    float* scale = nullptr;
};
