// adapters.cu -- low-rank adapters of several requests beside a projection that they share:  out[t] = base[t] + c up (down x[t]),
// with down [rank, cols], up [rows, rank] and the factor c of the adapter that token t's slot names.
//
// One launch.  A cluster of CTAs takes a tile of tokens that share an adapter; which tokens, every CTA works out from the slots (a histogram,
// then the tile's stretch of the adapter's tokens in their order; up to 16 tokens are a tile each, no histogram).  The CTAs split the
// columns of down x, add up their parts through distributed shared memory -- always in the order of their ranks -- and then split
// the rows of up h.
//
// Both products run on bf16 matrix instructions with float32 sums.  A float32 operand is the sum of three bf16 numbers, cut off it from the
// top eight bits at a time, exactly; a product with a bf16 matrix is then three instructions, with a float32 one six (what is left out
// is 2^-24 of the product).  So x, h and float32 adapters enter with all their bits, whatever the matrices' type.  A row of x that
// is not finite makes its output not-a-numbers.
//
// Bound: the rows of x, base and out; for few tokens the latencies of slot, row, sum and rows one behind the other.  2999 tokens, 2560 columns
// to 6912 rows of rank 16, five adapters: 62.8 us, 0.49 of what 197 MB take at the copy's rate -- 8 us to find the tiles, 10 for down x,
// 3 for its sums, 35 for up h and the rows of base and out at 5 TB/s.  (Asking L2 for rows of x and base some steps ahead: 64 to 69 us; tiles
// of 64 tokens, which read the adapter less often: 60.7 us, but 28 us instead of 20 for 512 tokens.)  One token 5.0 us, sixteen tokens of as
// many adapters, 4096 to 14336: 19.8 us.  4096 tokens of rank 64: 108 us, where the adapter's rows come from L2 for every sixteen of them.
#include "serving.cuh"

#include <cuda_bf16.h>

namespace {

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxRank = 256;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdMostCtas = 16;
constexpr int kAdGroups = 24 * 1024;  // where the tokens' groups stand while a tile is being found, behind histogram and flags
constexpr int kAdKept = 4096;         // tokens of a launch
constexpr int kAdTile = 16;  // tokens

struct AdapterParams {
    const void *down, *up;
    size_t down_plane, up_plane;  // bytes from one part of float32 values to the next
    const int* rank;
    const float* scale;
    const int32_t* slot;
    const float *x, *base;
    float* out;
    long long ldx;
    int slots, rows, cols, rank_pad, cols_pad, rows_pad, tokens;
    int copy;    // tokens without an adapter have something to be written
    int single;  // a tile is one token
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

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

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

// Consecutive values of a row of an adapter's matrix, four or eight, as they come: bf16, or the three parts of float32 values, which lie
// `plane` bytes apart.
template <bool F32, int N>
struct Raw {
    uint32_t w[F32 ? 3 : 1][N / 2];
};
template <bool F32, int N>
__device__ __forceinline__ void load_raw(const uint8_t* base, size_t plane, size_t at, Raw<F32, N>& r) {
#pragma unroll
    for (int k = 0; k < (F32 ? 3 : 1); ++k) {
        const uint8_t* p = base + k * plane + at * 2;
        if (N == 4) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            r.w[k][0] = v.x;
            r.w[k][1] = v.y;
        } else {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            r.w[k][0] = v.x;
            r.w[k][1] = v.y;
            r.w[k][N == 4 ? 0 : 2] = v.z;
            r.w[k][N == 4 ? 0 : 3] = v.w;
        }
    }
}
// the four values from 4 i on as B registers of both pairs
template <bool F32, int N>
__device__ __forceinline__ void parts_of(const Raw<F32, N>& r, int i, uint32_t (&b0)[3], uint32_t (&b1)[3]) {
#pragma unroll
    for (int k = 0; k < (F32 ? 3 : 1); ++k) {
        b0[k] = r.w[k][2 * i];
        b1[k] = r.w[k][2 * i + 1];
    }
}

constexpr int kAdPerSm = 2;  // CTAs (three or four with fewer registers each: 62 and 107 us for 2999 tokens, 62.8 with two, and more for all other sizes)

// TILES: ranks of one pass over x / 8.  Four at most for float32, whose 64 take so two passes: 4096 tokens 172 us, with eight and one CTA an SM 235.
template <int TILES, bool F32>
__global__ void __launch_bounds__(kAdThreads, kAdPerSm) lb_adapters_kernel(const AdapterParams p) {
    constexpr int M = kAdTile, KS = kAdWarps, kAdPass = 8 * TILES;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    float* part = reinterpret_cast<float*>(smem_raw);  // [KS][M][kAdPass] down x of this CTA's columns
    const int hs_ld = p.rank_pad + 4;
    __nv_bfloat16* hs = reinterpret_cast<__nv_bfloat16*>(part + KS * M * kAdPass);  // [3][M][hs_ld] h in three parts
    __shared__ int s_tok[M];
    __shared__ int s_warp[kAdWarps];
    __shared__ int s_group, s_tile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const unsigned crank = lb_cluster_rank();
    const int tile = blockIdx.x / size;
    lb_pdl_launch_dependents();
    lb_pdl_wait();

    // ---- the tile's adapter and tokens ----
    int group;
    if (p.single) {
        // (its x and base, which no slot has to be known for)
        for (int k = ((int)crank * KS + warp) * 32; k < p.cols; k += (int)size * KS * 32)
            if (lane == 0) prefetch_l2(p.x + (size_t)tile * p.ldx + k);
        const int c = ((int)crank * KS + warp) * 64 + lane * 32;
        if (p.base && lane < 2 && c < p.rows) prefetch_l2(p.base + (size_t)tile * p.rows + c);
        group = __ldg(p.slot + tile);
        if (group < 0 || group >= p.slots || __ldg(p.rank + group) <= 0) group = p.slots;
        if (group == p.slots && !p.copy) return;
        if (tid < M) s_tok[tid] = tid == 0 ? tile : -1;
        __syncthreads();
    } else {
        int* count = reinterpret_cast<int*>(smem_raw);                                          // [slots + 1]
        unsigned short* groups = reinterpret_cast<unsigned short*>(smem_raw + kAdGroups);       // [tokens]
        uint8_t* valid = smem_raw + kAdGroups - kAdMaxSlots;                                     // [slots]
        for (int i = tid; i <= p.slots; i += kAdThreads) {
            count[i] = 0;
            if (i < p.slots) valid[i] = __ldg(p.rank + i) > 0;
        }
        if (tid == 0) s_group = -1;
        __syncthreads();
        const auto group_at = [&](int token) {
            const int s = __ldg(p.slot + token);
            return s >= 0 && s < p.slots && valid[s] ? s : p.slots;
        };
#pragma unroll 8
        for (int i = tid; i < p.tokens; i += kAdThreads) {
            const int s = group_at(i);
            atomicAdd(&count[s], 1);
            groups[i] = (unsigned short)s;
        }
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
#pragma unroll
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
        group = s_group;
        if (group < 0) return;  // (the whole cluster: fewer tiles than the grid has room for)
        const int first = s_tile * M;
        if (tid < M) s_tok[tid] = -1;
        // the tokens in their order: a stretch of them to every warp, how many of each are the group's, then the tile's
        const int per = ((p.tokens + kAdWarps - 1) / kAdWarps + 31) / 32 * 32, from = warp * per, to = min(p.tokens, from + per);
        const auto is_mine = [&](int i) { return i < to && groups[i] == group; };
        int here = 0;
        for (int i0 = from; i0 < to; i0 += 32) here += __popc(__ballot_sync(0xffffffffu, is_mine(i0 + lane)));
        if (lane == 0) s_warp[warp] = here;
        __syncthreads();
        int at = 0;
        for (int w = 0; w < warp; ++w) at += s_warp[w];
        if (at < first + M && at + here > first)
            for (int i0 = from; i0 < to && at < first + M; i0 += 32) {
                const bool mine = is_mine(i0 + lane);
                const unsigned hit = __ballot_sync(0xffffffffu, mine);
                const int k = at + __popc(hit & ((1u << lane) - 1u));
                if (mine && k >= first && k < first + M) s_tok[k - first] = i0 + lane;
                at += __popc(hit);
            }
        __syncthreads();
    }
    if (group == p.slots) {  // no adapter: the base as it is
        for (int r = 0; r < M && s_tok[r] >= 0; ++r) {
            const size_t at = (size_t)s_tok[r] * p.rows;
#pragma unroll 4
            for (int i = crank * kAdThreads + tid; i < p.rows; i += size * kAdThreads) p.out[at + i] = p.base ? p.base[at + i] : 0.f;
        }
        return;
    }
    const int rank = __ldg(p.rank + group);
    const float scale = __ldg(p.scale + group);
    const int tok0 = s_tok[g], tok1 = s_tok[g + 8];
    constexpr int CH = TILES == 2 && !F32 ? 4 : 2;  // columns of out that a warp takes at a time, in sixteens
    const uint8_t* up = static_cast<const uint8_t*>(p.up) + (size_t)group * p.rows_pad * p.rank_pad * 2;
    {  // the first of them: the rows of up that they take
        const int c = ((int)crank * KS + warp) * 16 * CH, n = min(16 * CH, p.rows_pad - c);
        for (int k = 0; k < (F32 ? 3 : 1); ++k)
            for (int i = lane * 128; i < n * p.rank_pad * 2; i += 32 * 128) prefetch_l2(up + k * p.up_plane + (size_t)c * p.rank_pad * 2 + i);
    }

    // ---- h = c down x: 32 columns at a time, eight of them a lane ----
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
        const uint8_t* down = static_cast<const uint8_t*>(p.down) + (size_t)group * p.rank_pad * p.cols_pad * 2;
        for (int n0 = 0; n0 < rank; n0 += kAdPass) {
            const int tiles = (min(rank - n0, kAdPass) + 7) / 8, width = 8 * tiles;
            float acc[TILES][4] = {};
#pragma unroll 1
            for (int k0 = ((int)crank * KS + warp) * 32; k0 < p.cols_pad; k0 += (int)size * KS * 32) {
                const int k = k0 + 8 * t;
                float4 f[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    f[0][i] = load_x(x0, tok0 >= 0, k + 4 * i);
                    f[1][i] = load_x(x1, tok1 >= 0, k + 4 * i);
                }
                Raw<F32, 8> w[TILES];
#pragma unroll
                for (int n = 0; n < TILES; ++n)
                    if (n < tiles) load_raw<F32, 8>(down, p.down_plane, (size_t)(n0 + 8 * n + g) * p.cols_pad + k, w[n]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t a[3][4], v[3];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        split2(f[z][i].x, f[z][i].y, v);
#pragma unroll
                        for (int j = 0; j < 3; ++j) a[j][z] = v[j];
                        split2(f[z][i].z, f[z][i].w, v);
#pragma unroll
                        for (int j = 0; j < 3; ++j) a[j][2 + z] = v[j];
                    }
#pragma unroll
                    for (int n = 0; n < TILES; ++n)
                        if (n < tiles) {
                            uint32_t b0[3], b1[3];
                            parts_of<F32, 8>(w[n], i, b0, b1);
                            products<F32>(acc[n], a, b0, b1);
                        }
                }
            }
            __syncthreads();  // (what stood there has been read)
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                if (n >= tiles) break;
                float* to = part + ((size_t)warp * M + g) * kAdPass + 8 * n + 2 * t;
                *reinterpret_cast<float2*>(to) = make_float2(acc[n][0], acc[n][1]);
                *reinterpret_cast<float2*>(to + 8 * kAdPass) = make_float2(acc[n][2], acc[n][3]);
            }
            __syncthreads();
            for (int i = tid; i < M * width; i += kAdThreads) {
                float* at = part + i / width * kAdPass + i % width;
                float sum = *at;
#pragma unroll
                for (int j = 1; j < KS; ++j) sum += at[(size_t)j * M * kAdPass];
                *at = sum;
            }
            lb_cluster_sync();
            for (int i = tid; i < M * kAdPass; i += kAdThreads) {
                const int r = i / kAdPass, n = i % kAdPass;
                if (n0 + n >= p.rank_pad || s_tok[r] < 0) continue;  // (rows that are not there: whatever stands in hs)
                float sum = 0.f;
                if (n < width) {
#pragma unroll
                    for (unsigned q = 0; q < kAdMostCtas; ++q)
                        if (q < size) sum += ld_cluster_f32(lb_cluster_addr(lb_smem_u32(part + i), q));
                }
                sum *= scale;
#pragma unroll
                for (int k = 0; k < 3; ++k) hs[((size_t)k * M + r) * hs_ld + n0 + n] = __ushort_as_bfloat16((unsigned short)(__float_as_uint(cut(sum)) >> 16));
            }
            lb_cluster_sync();  // (the parts have been read)
        }
    }

    // ---- out = base + up h: 64 columns at a time ----
    const bool wide = (p.rows & 3) == 0 && ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.base)) & 15) == 0;
    const int col_a = 4 * (g >> 1) + (g & 1);  // the rows of up whose sums lane t gets as four neighbours
    for (int c0 = ((int)crank * KS + warp) * 16 * CH; c0 < p.rows_pad; c0 += (int)size * KS * 16 * CH) {
        float4 base[CH][2];
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int tok = z ? tok1 : tok0, c = c0 + 16 * j + 4 * t;
                base[j][z] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (wide && p.base && tok >= 0 && c < p.rows) base[j][z] = __ldcs(reinterpret_cast<const float4*>(p.base + (size_t)tok * p.rows + c));
            }
        float acc[CH][2][4] = {};
        // KU stretches of 4 KV ranks, lane t the KV from KV t on: every row of up that is there in flight at once
        constexpr int KV = TILES == 2 ? 4 : 8, KU = TILES == 8 ? 2 : 1;
        for (int k0 = 0; k0 < rank; k0 += 4 * KV * KU) {
            Raw<F32, KV> w[KU][CH][2];
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int j = 0; j < CH; ++j)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
                        if (c0 + 16 * j < p.rows_pad && (u == 0 || k0 + 4 * KV * u < rank))
                            load_raw<F32, KV>(up, p.up_plane, (size_t)(c0 + 16 * j + col_a + 2 * n) * p.rank_pad + k0 + 4 * KV * u + KV * t, w[u][j][n]);
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                if (u > 0 && k0 + 4 * KV * u >= rank) break;
#pragma unroll
                for (int e = 0; e < KV / 4; ++e) {
                    uint32_t a[3][4];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        const __nv_bfloat16* from = hs + ((size_t)i * M + g) * hs_ld + k0 + 4 * KV * u + KV * t + 4 * e;
                        const uint2 r0 = *reinterpret_cast<const uint2*>(from), r1 = *reinterpret_cast<const uint2*>(from + 8 * hs_ld);
                        a[i][0] = r0.x;
                        a[i][1] = r1.x;
                        a[i][2] = r0.y;
                        a[i][3] = r1.y;
                    }
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        if (c0 + 16 * j < p.rows_pad)
#pragma unroll
                            for (int n = 0; n < 2; ++n) {
                                uint32_t b0[3], b1[3];
                                parts_of<F32, KV>(w[u][j][n], e, b0, b1);
                                products<F32>(acc[j][n], a, b0, b1);
                            }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int tok = z ? tok1 : tok0, c = c0 + 16 * j + 4 * t;
                if (tok < 0 || c >= p.rows) continue;
                const size_t at = (size_t)tok * p.rows + c;
                float f[4] = {acc[j][0][2 * z], acc[j][0][2 * z + 1], acc[j][1][2 * z], acc[j][1][2 * z + 1]};
                if (wide) {
                    const float4 b = base[j][z];
                    __stcs(reinterpret_cast<float4*>(p.out + at), make_float4(f[0] + b.x, f[1] + b.y, f[2] + b.z, f[3] + b.w));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < p.rows) p.out[at + e] = f[e] + (p.base ? p.base[at + e] : 0.f);
                }
            }
    }
}

// a slot's matrix into its padded place: bf16, or float32 values in three parts
__global__ void lb_adapters_put_kernel(const void* __restrict__ src, int src_dtype, int rows, int cols, int rows_pad, int cols_pad, int parts, size_t plane, uint8_t* __restrict__ dst) {
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (size_t)rows_pad * cols_pad) return;
    const int r = (int)(i / cols_pad), c = (int)(i % cols_pad);
    float f = 0.f;
    if (r < rows && c < cols)
        f = src_dtype == LOOM_B200_DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(src)[(size_t)r * cols + c]) : static_cast<const float*>(src)[(size_t)r * cols + c];
    if (parts == 1) reinterpret_cast<__nv_bfloat16*>(dst)[i] = __float2bfloat16_rn(f);
    for (int k = 0; k < parts && parts > 1; ++k) *reinterpret_cast<unsigned short*>(dst + k * plane + i * 2) = (unsigned short)(__float_as_uint(cut(f)) >> 16);
}
__global__ void lb_adapters_meta_kernel(int* rank, float* scale, int r, float s) {
    *rank = r;
    *scale = s;
}

template <int TILES, bool F32>
int launch_adapters(loom_b200_ctx* ctx, const AdapterParams& p, int tiles) {
    constexpr int M = kAdTile;
    constexpr size_t find = (size_t)kAdGroups + kAdKept * 2, parts = (size_t)kAdWarps * M * 8 * TILES * 4, front = find > parts ? find : parts;
    static_assert((size_t)kAdGroups >= (kAdMaxSlots + 1) * 4 + kAdMaxSlots, "room for what finds a tile");
    const size_t smem = front + (size_t)3 * M * (p.rank_pad + 4) * 2;
    const auto kern = lb_adapters_kernel<TILES, F32>;
    LB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(front + (size_t)3 * M * (kAdMaxRank + 4) * 2)));
    LB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    // As many CTAs a tile as are there at once.  Clusters of more than eight find their places in a GPC less and less well (256 tokens of
    // two adapters: 12 CTAs a tile 13.9 us, 14 18.6 us), so those leave a quarter free; 14 clusters of 16 still fit (16 tokens of rank 16, 4096 to
    // 14336: 13.9 us by 16 CTAs each, 11.6 by 12, 12.0 by 8; 14 tokens 8.5, 10.8 and 11.8 us; with sixteen warps a CTA no better).  Both are measured on one
    // division of the SMs into GPCs; any size is right on any other.
    const int most = kAdPerSm * ctx->sm_count;
    int size = most * 7 / 8 / tiles;
    if (size >= kAdMostCtas) size = tiles <= 14 ? kAdMostCtas : 12;
    else if (size > 8) size = most * 3 / 4 / tiles > 8 ? most * 3 / 4 / tiles : 8;
    else if (size < 4) size = most / tiles > 4 ? 4 : most / tiles > 0 ? most / tiles : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * size);
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->opt_pdl ? 2 : 1;
    LB_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, p));
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
    a->rank_pad = max_rank <= 16 ? 16 : (max_rank + 31) / 32 * 32;  // (what lb_adapters_kernel takes at a time)
    a->cols_pad = (cols + 31) / 32 * 32;
    a->rows_pad = (rows + 15) / 16 * 16;
    const size_t w = dtype == LOOM_B200_DTYPE_F32 ? 6 : 2;  // (float32 values as three of 16 bits)
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
    const size_t sw = src_dtype == LOOM_B200_DTYPE_F32 ? 4 : 2;
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
        uint8_t* dst = static_cast<uint8_t*>(m ? a->up : a->down) + (size_t)slot * total * 2;
        const unsigned grid = (unsigned)((total + 255) / 256);
        lb_adapters_put_kernel<<<grid, 256, 0, ctx->stream>>>(src, src_dtype, rows, cols, rows_pad, cols_pad, a->dtype == LOOM_B200_DTYPE_F32 ? 3 : 1, (size_t)a->slots * total * 2, dst);
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
    p.down_plane = (size_t)a->slots * a->rank_pad * a->cols_pad * 2;
    p.up_plane = (size_t)a->slots * a->rows_pad * a->rank_pad * 2;
    p.rank = a->rank;
    p.scale = a->scale;
    p.ldx = ldx;
    p.slots = a->slots;
    p.rows = a->rows;
    p.cols = a->cols;
    p.rank_pad = a->rank_pad;
    p.cols_pad = a->cols_pad;
    p.rows_pad = a->rows_pad;
    p.copy = base != out;
    const auto launch = a->dtype == LOOM_B200_DTYPE_F32 ? a->max_rank <= 16 ? launch_adapters<2, true> : launch_adapters<4, true>
                                                        : a->max_rank <= 16 ? launch_adapters<2, false> : a->max_rank <= 32 ? launch_adapters<4, false> : launch_adapters<8, false>;
    // (every CTA reads all slots of its launch: 8192 tokens in one 151 us, in two 131)
    for (int at = 0; at < tokens; at += kAdKept) {
        p.tokens = tokens - at < kAdKept ? tokens - at : kAdKept;
        p.slot = slot + at;
        p.x = x + (size_t)at * ldx;
        p.base = base ? base + (size_t)at * a->rows : nullptr;
        p.out = out + (size_t)at * a->rows;
        p.single = p.tokens <= 16;
        const int groups = a->slots + 1;
        const int tiles = p.single || p.tokens <= groups ? p.tokens : groups + (p.tokens - groups) / kAdTile;  // at most
        if (int rc = launch(ctx, p, tiles)) return rc;
    }
    return 0;
}

}  // extern "C"
