// adapters.cu -- low-rank adapters of several requests beside a projection that they share:  out[t] = base[t] + c up (down x[t]),
// with down [rank, cols], up [rows, rank] and the factor c of the adapter that token t's slot names.
//
// One launch.  A cluster of CTAs takes a tile of tokens that share an adapter; which tokens, every CTA works out from the slots (a histogram,
// then the tile's stretch of the adapter's tokens in their order).  The CTAs split the columns of down x, add up their parts through
// distributed shared memory -- always in the order of their ranks -- and then split the rows of up h.
//
// Both products run on bf16 matrix instructions with float32 sums.  A float32 operand is the sum of three bf16 numbers, cut off it from the
// top eight bits at a time, exactly; a product with a bf16 matrix is then three instructions, with a float32 one six (what is left out
// is 2^-24 of the product).  So x, h and float32 adapters enter with all their bits, whatever the matrices' type.  A row of x that
// is not finite makes its output not-a-numbers.
#include "serving.cuh"

#include <cuda_bf16.h>

namespace {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxRank = 256;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdPass = 64;  // ranks of one pass over x

struct AdapterParams {
    const void *down, *up;
    const int* rank;
    const float* scale;
    const int32_t* slot;
    const float *x, *base;
    float* out;
    long long ldx;
    int slots, rows, cols, rank_pad, cols_pad, rows_pad, tokens;
    int copy;  // tokens without an adapter have something to be written
};

// a float32 value's top sixteen bits, and what is left
__device__ __forceinline__ float cut(float& f) {
    const float top = __uint_as_float(__float_as_uint(f) & 0xffff0000u);
    f -= top;
    return top;
}
// two values' top halves as a bf16 pair
__device__ __forceinline__ uint32_t pair_of(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ void split2(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const float ta = cut(a), tb = cut(b);
        w[k] = pair_of(ta, tb);
    }
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// a[part][register] . b: the parts of both that reach 2^-24
template <bool F32>
__device__ __forceinline__ void products(float (&d)[4], const uint32_t (&a)[3][4], const uint32_t (&b0)[3], const uint32_t (&b1)[3]) {
    if (F32) {
        mma_bf16(d, a[1][0], a[1][1], a[1][2], a[1][3], b0[1], b1[1]);
        mma_bf16(d, a[0][0], a[0][1], a[0][2], a[0][3], b0[2], b1[2]);
    }
    mma_bf16(d, a[2][0], a[2][1], a[2][2], a[2][3], b0[0], b1[0]);
    if (F32) mma_bf16(d, a[0][0], a[0][1], a[0][2], a[0][3], b0[1], b1[1]);
    mma_bf16(d, a[1][0], a[1][1], a[1][2], a[1][3], b0[0], b1[0]);
    mma_bf16(d, a[0][0], a[0][1], a[0][2], a[0][3], b0[0], b1[0]);
}

// four consecutive values of a row of an adapter's matrix as B registers of both pairs
template <bool F32>
__device__ __forceinline__ void load4(const void* base, size_t at, uint32_t (&b0)[3], uint32_t (&b1)[3]) {
    if (F32) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at));
        split2(f.x, f.y, b0);
        split2(f.z, f.w, b1);
    } else {
        const uint2 f = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + at));
        b0[0] = f.x;
        b1[0] = f.y;
    }
}

// MT: tiles of 16 tokens in a cluster's tile
template <int MT, bool F32>
__global__ void __launch_bounds__(kAdThreads) lb_adapters_kernel(const AdapterParams p) {
    constexpr int M = 16 * MT, KS = kAdWarps / MT;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    float* part = reinterpret_cast<float*>(smem_raw);  // [KS][M][kAdPass] down x of this CTA's columns; the groups' histogram before that
    const int hs_ld = p.rank_pad + 4;
    __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(part + KS * M * kAdPass);  // [3][M][hs_ld] h in three parts
    __shared__ int s_tok[M];
    __shared__ int s_warp[kAdWarps];
    __shared__ int s_group, s_tile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const unsigned crank = lb_cluster_rank();
    int tile = blockIdx.x / size;

    // the tile's adapter and tokens
    const auto group_of = [&](int token) {
        const int s = __ldg(p.slot + token);
        return s >= 0 && s < p.slots && __ldg(p.rank + s) > 0 ? s : p.slots;
    };
    {
        int* count = reinterpret_cast<int*>(part);  // [slots + 1]
        for (int i = tid; i <= p.slots; i += kAdThreads) count[i] = 0;
        if (tid == 0) s_group = -1;
        __syncthreads();
        for (int i = tid; i < p.tokens; i += kAdThreads) atomicAdd(&count[group_of(i)], 1);
        __syncthreads();
        int before = 0;
        for (int g0 = 0; g0 <= p.slots; g0 += kAdThreads) {
            const int gi = g0 + tid;
            const int mine = gi < p.slots || (gi == p.slots && p.copy) ? (count[gi] + M - 1) / M : 0;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (lane == 31) s_warp[warp] = sum;
            __syncthreads();
            int all = 0;
            for (int w = 0; w < kAdWarps; ++w) {
                if (w < warp) sum += s_warp[w];
                all += s_warp[w];
            }
            if (tile >= before + sum - mine && tile < before + sum) {
                s_group = gi;
                s_tile = tile - (before + sum - mine);
            }
            before += all;
            __syncthreads();
        }
    }
    const int group = s_group;
    if (group < 0) return;  // (the whole cluster: fewer tiles than the grid has room for)
    tile = s_tile;
    if (tid < M) s_tok[tid] = -1;
    int seen = 0;
    for (int i0 = 0; i0 < p.tokens && seen < (tile + 1) * M; i0 += kAdThreads) {
        const int i = i0 + tid;
        const bool mine = i < p.tokens && group_of(i) == group;
        const unsigned hit = __ballot_sync(0xffffffffu, mine);
        __syncthreads();
        if (lane == 0) s_warp[warp] = __popc(hit);
        __syncthreads();
        int at = seen + __popc(hit & ((1u << lane) - 1u));
        for (int w = 0; w < kAdWarps; ++w) {
            if (w < warp) at += s_warp[w];
            seen += s_warp[w];
        }
        if (mine && at >= tile * M && at < (tile + 1) * M) s_tok[at - tile * M] = i;
    }
    __syncthreads();
    if (group == p.slots) {  // no adapter: the base as it is
        for (int r = 0; r < M && s_tok[r] >= 0; ++r) {
            const size_t at = (size_t)s_tok[r] * p.rows;
            for (int i = crank * kAdThreads + tid; i < p.rows; i += size * kAdThreads) p.out[at + i] = p.base ? p.base[at + i] : 0.f;
        }
        return;
    }
    const int rank = __ldg(p.rank + group);
    const float scale = __ldg(p.scale + group);
    const int mt = warp % MT, ks = warp / MT;
    const int tok0 = s_tok[16 * mt + g], tok1 = s_tok[16 * mt + g + 8];
    const size_t wsize = F32 ? 4 : 2;

    // h = c down x
    {
        const float* x0 = p.x + (size_t)(tok0 < 0 ? 0 : tok0) * p.ldx;
        const float* x1 = p.x + (size_t)(tok1 < 0 ? 0 : tok1) * p.ldx;
        const bool wide = ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)p.ldx * 4) & 15) == 0;
        const auto load_x = [&](const float* row, bool is, int k) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!is) return f;
            if (wide && k + 4 <= p.cols) return __ldg(reinterpret_cast<const float4*>(row + k));
            if (k < p.cols) f.x = __ldg(row + k);
            if (k + 1 < p.cols) f.y = __ldg(row + k + 1);
            if (k + 2 < p.cols) f.z = __ldg(row + k + 2);
            if (k + 3 < p.cols) f.w = __ldg(row + k + 3);
            return f;
        };
        const uint8_t* down = static_cast<const uint8_t*>(p.down) + (size_t)group * p.rank_pad * p.cols_pad * wsize;
        for (int n0 = 0; n0 < rank; n0 += kAdPass) {
            const int tiles = (min(rank - n0, kAdPass) + 7) / 8;
            float acc[kAdPass / 8][4] = {};
            for (int k0 = ((int)crank * KS + ks) * 16; k0 < p.cols_pad; k0 += (int)size * KS * 16) {
                const int k = k0 + 4 * t;
                const float4 f0 = load_x(x0, tok0 >= 0, k), f1 = load_x(x1, tok1 >= 0, k);
                uint32_t a[3][4], w[3];
                split2(f0.x, f0.y, w);
#pragma unroll
                for (int i = 0; i < 3; ++i) a[i][0] = w[i];
                split2(f1.x, f1.y, w);
#pragma unroll
                for (int i = 0; i < 3; ++i) a[i][1] = w[i];
                split2(f0.z, f0.w, w);
#pragma unroll
                for (int i = 0; i < 3; ++i) a[i][2] = w[i];
                split2(f1.z, f1.w, w);
#pragma unroll
                for (int i = 0; i < 3; ++i) a[i][3] = w[i];
#pragma unroll
                for (int n = 0; n < kAdPass / 8; ++n) {
                    if (n >= tiles) break;
                    uint32_t b0[3], b1[3];
                    load4<F32>(down, (size_t)(n0 + 8 * n + g) * p.cols_pad + k, b0, b1);
                    products<F32>(acc[n], a, b0, b1);
                }
            }
            __syncthreads();  // (the histogram, or the pass before, has been read)
#pragma unroll
            for (int n = 0; n < kAdPass / 8; ++n) {
                if (n >= tiles) break;
                float* to = part + ((size_t)ks * M + 16 * mt + g) * kAdPass + 8 * n + 2 * t;
                *reinterpret_cast<float2*>(to) = make_float2(acc[n][0], acc[n][1]);
                *reinterpret_cast<float2*>(to + 8 * kAdPass) = make_float2(acc[n][2], acc[n][3]);
            }
            __syncthreads();
            for (int i = tid; i < M * kAdPass; i += kAdThreads) {
                float sum = part[i];
                for (int j = 1; j < KS; ++j) sum += part[(size_t)j * M * kAdPass + i];
                part[i] = sum;
            }
            lb_cluster_sync();
            for (int i = tid; i < M * kAdPass; i += kAdThreads) {
                const int r = i / kAdPass, n = i % kAdPass;
                if (n0 + n >= p.rank_pad) continue;
                float sum = 0.f;
                if (n < 8 * tiles)
                    for (unsigned q = 0; q < size; ++q) sum += ld_cluster_f32(lb_cluster_addr(lb_smem_u32(part + i), q));
                sum *= scale;
#pragma unroll
                for (int k = 0; k < 3; ++k) hs[((size_t)k * M + r) * hs_ld + n0 + n] = __ushort_as_bfloat16((unsigned short)(__float_as_uint(cut(sum)) >> 16));
            }
            lb_cluster_sync();  // (the parts have been read)
        }
    }

    // out = base + up h
    const uint8_t* up = static_cast<const uint8_t*>(p.up) + (size_t)group * p.rows_pad * p.rank_pad * wsize;
    const bool wide = (p.rows & 3) == 0 && ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.base)) & 15) == 0;
    const int col_a = 4 * (g >> 1) + (g & 1);  // the rows of up whose sums lane t gets as four neighbours
    for (int c0 = ((int)crank * KS + ks) * 16; c0 < p.rows_pad; c0 += (int)size * KS * 16) {
        float acc[2][4] = {};
        for (int k0 = 0; k0 < rank; k0 += 16) {
            uint32_t a[3][4];
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const __nv_bfloat16* from = hs + ((size_t)i * M + 16 * mt + g) * hs_ld + k0 + 4 * t;
                const uint2 r0 = *reinterpret_cast<const uint2*>(from), r1 = *reinterpret_cast<const uint2*>(from + 8 * hs_ld);
                a[i][0] = r0.x;
                a[i][1] = r1.x;
                a[i][2] = r0.y;
                a[i][3] = r1.y;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                uint32_t b0[3], b1[3];
                load4<F32>(up, (size_t)(c0 + col_a + 2 * n) * p.rank_pad + k0 + 4 * t, b0, b1);
                products<F32>(acc[n], a, b0, b1);
            }
        }
        const int c = c0 + 4 * t;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int tok = z ? tok1 : tok0;
            if (tok < 0) continue;
            const size_t at = (size_t)tok * p.rows + c;
            float f[4] = {acc[0][2 * z], acc[0][2 * z + 1], acc[1][2 * z], acc[1][2 * z + 1]};
            if (wide && c < p.rows) {
                if (p.base) {
                    const float4 b = *reinterpret_cast<const float4*>(p.base + at);
                    f[0] += b.x;
                    f[1] += b.y;
                    f[2] += b.z;
                    f[3] += b.w;
                }
                *reinterpret_cast<float4*>(p.out + at) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < p.rows) p.out[at + e] = f[e] + (p.base ? p.base[at + e] : 0.f);
            }
        }
    }
}

// a slot's matrices into their padded places
template <typename WT>
__global__ void lb_adapters_put_kernel(const void* __restrict__ src, int src_dtype, int rows, int cols, int rows_pad, int cols_pad, WT* __restrict__ dst) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (size_t)rows_pad * cols_pad) return;
    const int r = (int)(i / cols_pad), c = (int)(i % cols_pad);
    float f = 0.f;
    if (r < rows && c < cols)
        f = src_dtype == LOOM_B200_DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(src)[(size_t)r * cols + c]) : static_cast<const float*>(src)[(size_t)r * cols + c];
    dst[i] = (WT)f;
}
__global__ void lb_adapters_meta_kernel(int* rank, float* scale, int r, float s) {
    *rank = r;
    *scale = s;
}

template <int MT, bool F32>
int launch_adapters(loom_b200_ctx* ctx, const AdapterParams& p, int tiles) {
    constexpr int M = 16 * MT, KS = kAdWarps / MT;
    const size_t front = (size_t)KS * M * kAdPass * 4;
    static_assert((size_t)KS * M * kAdPass >= kAdMaxSlots + 1, "room for the histogram");
    const size_t smem = front + (size_t)3 * M * (p.rank_pad + 4) * 2;
    LB_CUDA(ctx, cudaFuncSetAttribute(lb_adapters_kernel<MT, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(front + (size_t)3 * M * (kAdMaxRank + 4) * 2)));
    int size = 8;
    while (size > 1 && tiles * size > 4 * ctx->sm_count) size /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * size);
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LB_CUDA(ctx, cudaLaunchKernelEx(&cfg, lb_adapters_kernel<MT, F32>, p));
    ctx->launches++;
    return 0;
}

}  // namespace

extern "C" {

int loom_b200_adapters_create(loom_b200_ctx* ctx, int slots, int rows, int cols, int max_rank, int dtype, loom_b200_adapters** out) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "adapters_create: ctx is NULL");
    LB_REQUIRE(ctx, out != nullptr, "adapters_create: out is NULL");
    *out = nullptr;
    LB_REQUIRE(ctx, slots > 0 && rows > 0 && cols > 0 && max_rank > 0, "adapters_create: %d slots of rank %d for a matrix %dx%d", slots, max_rank, rows, cols);
    LB_REQUIRE(ctx, dtype == LOOM_B200_DTYPE_F32 || dtype == LOOM_B200_DTYPE_BF16, "adapters_create: dtype %d", dtype);
    if (slots > kAdMaxSlots || max_rank > kAdMaxRank || rows > (1 << 24) || cols > (1 << 24))
        return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "adapters_create: %d slots (%d at most) of rank %d (%d at most) for a matrix %dx%d", slots, kAdMaxSlots, max_rank, kAdMaxRank, rows, cols);
    if (ctx->capturing) return lb_fail(ctx, LOOM_B200_ERR_INVALID, "adapters_create cannot be recorded");
    if (int rc = lb_set_device(ctx)) return rc;
    auto* a = new loom_b200_adapters();
    a->ctx = ctx;
    a->slots = slots;
    a->rows = rows;
    a->cols = cols;
    a->max_rank = max_rank;
    a->dtype = dtype;
    a->rank_pad = (max_rank + 15) / 16 * 16;
    a->cols_pad = (cols + 31) / 32 * 32;
    a->rows_pad = (rows + 15) / 16 * 16;
    const size_t w = dtype == LOOM_B200_DTYPE_F32 ? 4 : 2;
    cudaError_t e = cudaMalloc(&a->down, (size_t)slots * a->rank_pad * a->cols_pad * w);
    if (e == cudaSuccess) e = cudaMalloc(&a->up, (size_t)slots * a->rows_pad * a->rank_pad * w);
    if (e == cudaSuccess) e = cudaMalloc((void**)&a->rank, (size_t)slots * 4);
    if (e == cudaSuccess) e = cudaMalloc((void**)&a->scale, (size_t)slots * 4);
    if (e == cudaSuccess) e = cudaMemsetAsync(a->rank, 0, (size_t)slots * 4, ctx->stream);
    if (e != cudaSuccess) {
        loom_b200_adapters_free(ctx, a);
        return lb_fail(ctx, LOOM_B200_ERR_CUDA, "adapters_create: %d slots of rank %d for a matrix %dx%d: %s", slots, max_rank, rows, cols, cudaGetErrorString(e));
    }
    *out = a;
    return 0;
}

int loom_b200_adapters_put(loom_b200_ctx* ctx, loom_b200_adapters* a, int slot, int rank, float scale, const void* down, const void* up, int src_dtype, int src_on_device) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "adapters_put: ctx is NULL");
    LB_REQUIRE(ctx, a != nullptr, "adapters_put: adapters is NULL");
    LB_REQUIRE(ctx, a->ctx == ctx, "adapters_put: the adapters belong to another context");
    LB_REQUIRE(ctx, slot >= 0 && slot < a->slots, "adapters_put: slot %d of %d", slot, a->slots);
    LB_REQUIRE(ctx, rank >= 0 && rank <= a->max_rank, "adapters_put: rank %d of at most %d", rank, a->max_rank);
    LB_REQUIRE(ctx, rank == 0 || (down && up), "adapters_put: NULL matrix");
    LB_REQUIRE(ctx, src_dtype == LOOM_B200_DTYPE_F32 || src_dtype == LOOM_B200_DTYPE_BF16, "adapters_put: dtype %d", src_dtype);
    if (ctx->capturing) return lb_fail(ctx, LOOM_B200_ERR_INVALID, "adapters_put cannot be recorded");
    if (int rc = lb_set_device(ctx)) return rc;
    const size_t w = a->dtype == LOOM_B200_DTYPE_F32 ? 4 : 2, sw = src_dtype == LOOM_B200_DTYPE_F32 ? 4 : 2;
    for (int m = 0; m < 2 && rank > 0; ++m) {
        const void* src = m ? up : down;
        const int rows = m ? a->rows : rank, cols = m ? rank : a->cols;
        const int rows_pad = m ? a->rows_pad : a->rank_pad, cols_pad = m ? a->rank_pad : a->cols_pad;
        if (!src_on_device) {
            const size_t bytes = (size_t)rows * cols * sw;
            if (int rc = lb_ensure_scratch(ctx, bytes)) return rc;
            LB_CUDA(ctx, cudaMemcpyAsync(ctx->scratch, src, bytes, cudaMemcpyHostToDevice, ctx->stream));
            src = ctx->scratch;
        }
        const size_t total = (size_t)rows_pad * cols_pad;
        uint8_t* dst = static_cast<uint8_t*>(m ? a->up : a->down) + (size_t)slot * total * w;
        const unsigned grid = (unsigned)((total + 255) / 256);
        if (a->dtype == LOOM_B200_DTYPE_F32) lb_adapters_put_kernel<float><<<grid, 256, 0, ctx->stream>>>(src, src_dtype, rows, cols, rows_pad, cols_pad, (float*)dst);
        else lb_adapters_put_kernel<__nv_bfloat16><<<grid, 256, 0, ctx->stream>>>(src, src_dtype, rows, cols, rows_pad, cols_pad, (__nv_bfloat16*)dst);
        LB_CHECK_LAUNCH(ctx, "lb_adapters_put_kernel");
    }
    lb_adapters_meta_kernel<<<1, 1, 0, ctx->stream>>>(a->rank + slot, a->scale + slot, rank, scale);
    LB_CHECK_LAUNCH(ctx, "lb_adapters_meta_kernel");
    LB_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
    return 0;
}

int loom_b200_adapters_info(const loom_b200_adapters* a, int* slots, int* rows, int* cols, int* max_rank, int* dtype) {
    if (!a) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "adapters_info: adapters is NULL");
    if (slots) *slots = a->slots;
    if (rows) *rows = a->rows;
    if (cols) *cols = a->cols;
    if (max_rank) *max_rank = a->max_rank;
    if (dtype) *dtype = a->dtype;
    return 0;
}

void loom_b200_adapters_free(loom_b200_ctx* ctx, loom_b200_adapters* a) {
    if (!a) return;
    if (ctx) {
        cudaSetDevice(ctx->device);
        cudaStreamSynchronize(ctx->stream);
    }
    void* ptrs[] = {a->down, a->up, a->rank, a->scale};
    for (void* p : ptrs)
        if (p) cudaFree(p);
    delete a;
}

int loom_b200_adapters_apply(loom_b200_ctx* ctx, const loom_b200_adapters* a, int tokens, const int32_t* slot, const float* x, long long ldx, const float* base, float* out) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "adapters_apply: ctx is NULL");
    LB_REQUIRE(ctx, a && slot && x && out, "adapters_apply: NULL argument");
    LB_REQUIRE(ctx, a->ctx == ctx, "adapters_apply: the adapters belong to another context");
    LB_REQUIRE(ctx, tokens > 0, "adapters_apply: %d tokens", tokens);
    LB_REQUIRE(ctx, ldx >= a->cols, "adapters_apply: %lld floats between rows of %d", ldx, a->cols);
    if (tokens > (1 << 22)) return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "adapters_apply: %d tokens, %d at most", tokens, 1 << 22);
    if (int rc = lb_set_device(ctx)) return rc;
    AdapterParams p;
    p.down = a->down;
    p.up = a->up;
    p.rank = a->rank;
    p.scale = a->scale;
    p.slot = slot;
    p.x = x;
    p.base = base;
    p.out = out;
    p.ldx = ldx;
    p.slots = a->slots;
    p.rows = a->rows;
    p.cols = a->cols;
    p.rank_pad = a->rank_pad;
    p.cols_pad = a->cols_pad;
    p.rows_pad = a->rows_pad;
    p.tokens = tokens;
    p.copy = base != out;
    const int groups = a->slots + 1, m = tokens >= 256 ? 64 : 16;
    const int tiles = tokens <= groups ? tokens : groups + (tokens - groups) / m;  // at most
    const bool f32 = a->dtype == LOOM_B200_DTYPE_F32;
    if (m == 64) return f32 ? launch_adapters<4, true>(ctx, p, tiles) : launch_adapters<4, false>(ctx, p, tiles);
    return f32 ? launch_adapters<1, true>(ctx, p, tiles) : launch_adapters<1, false>(ctx, p, tiles);
}

}  // extern "C"
