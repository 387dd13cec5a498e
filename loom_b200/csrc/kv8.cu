// kv8.cu -- a cache of keys and values in 8 bits for several sequences, and attention over it.
//
// Positions of a sequence go by blocks of 64.  A whole block is held in 8 bits, with one scale for each KV head, keys and values apart:
// a = largest |x| of the block's 64 rows of that head, code = round(x * 127 / a) half away from zero (the arithmetic of the activation
// quantizer: float64 quotient and product), value = code * a / 127.  A block with a value that is not finite reads as not-a-numbers.
// The positions behind the last whole block are held in float32 as they came; of the block in front of them the float32 rows stay too, so
// a sequence may be cut back into it and go on from there.
//
// Codes lie as the tensor core's B operands want them, so that a warp's load of 16 bytes a lane is 512 consecutive bytes and needs no
// shared memory on its way (lane = 4 g + t):
//   keys    per block and KV head [position / 8][64 dimensions][position % 8 = g][64 bytes], the last 32 dimensions, if alone, 32 bytes
//           instead; lane (g, t) takes dimensions 16 t .. 16 t + 15 of a chunk: which of them an MMA sees as which k is the same for the
//           queries, so the order cancels
//   values  [dimension / 8][dimension % 8 = g][t][16 positions 8 j + 2 t + e, (j, e) in order]: the positions whose scores lane t holds
//           after the products with the keys
#include "serving.cuh"

#include <math_constants.h>

#include <cmath>

namespace {

struct Kv8 {
    int seqs, max_len, heads, dim, blocks, dim_k, dim_v;
    uint8_t *k, *v;
    float *k_top, *v_top, *k_open, *v_open;
    int* status;

    __host__ __device__ size_t head_of(int s, int h) const { return (size_t)s * heads + h; }
    __device__ __forceinline__ float* open_row(float* base, int s, int h, int pos) const {
        return base + ((head_of(s, h) * 2 + (pos / kKvBlock & 1)) * kKvBlock + pos % kKvBlock) * dim;
    }
};

// Rows of sequence s in this call: first row, and how many; the position of the first.  Starts that do not ascend, or lie outside of the
// rows, give the rows that there are.
struct Span {
    int row, count, pos;
};
__device__ __forceinline__ Span span_of(const int32_t* __restrict__ starts, const int32_t* __restrict__ lengths, int rows, int s) {
    Span a;
    a.pos = __ldg(lengths + s);
    if (!starts) {
        a.row = s;
        a.count = s < rows ? 1 : 0;
        return a;
    }
    a.row = min(max(__ldg(starts + s), 0), rows);
    a.count = max(min(__ldg(starts + s + 1), rows) - a.row, 0);
    return a;
}
// whether the sequence has room for them
__device__ __forceinline__ bool fits(const Kv8& c, const Span& a) { return a.pos >= 0 && a.pos <= c.max_len && a.count <= c.max_len - a.pos; }

// byte of a key's dimension d at place p of its block; of a value's
__device__ __forceinline__ int key_byte(int p, int d, int dim_k) {
    const int c = d >> 6, whole = dim_k >> 6;
    return (p >> 3) * 8 * dim_k + (c < whole ? c * 512 + (p & 7) * 64 + (d & 63) : whole * 512 + (p & 7) * 32 + (d & 31));
}
__device__ __forceinline__ int value_byte(int p, int d) { return (d >> 3) * 512 + (d & 7) * 64 + (p >> 1 & 3) * 16 + (p >> 3) * 2 + (p & 1); }

// ---- rows in ---------------------------------------------------------------------------------------------------------------------
//
// A CTA takes one block of one sequence and head that the call's rows touch.  It writes them to the open rows where the block is one of the
// last two, and where they complete it (the first of its rows may be there already) makes the codes.  Open rows go by the block's parity:
// the rows that the first block still reads there may be what a block two further on replaces, so the CTA of the first block
// writes for that one too, after its own reads.
constexpr int kApThreads = 256;

struct AppendParams {
    Kv8 c;
    int rows;
    const int32_t *starts, *lengths;
    const float *k, *v;
    long long ld;  // floats from one row of k (and of v) to the next
};

__global__ void __launch_bounds__(kApThreads) lb_kv8_append_kernel(const AppendParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    float* x = reinterpret_cast<float*>(smem_raw);  // [64][dim]
    __shared__ float s_top[kApThreads / 32];
    const Kv8& c = p.c;
    const int s = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const Span a = span_of(p.starts, p.lengths, p.rows, s);
    if (a.count == 0) return;
    if (!fits(c, a)) {
        if (blockIdx.x == 0 && h == 0 && tid == 0) atomicExch(c.status, 7);
        return;
    }
    const int end = a.pos + a.count;
    const int first = a.pos / kKvBlock, last = (end - 1) / kKvBlock;  // blocks
    for (int b = first + (int)blockIdx.x; b <= last; b += gridDim.x) {
        const int from = max(a.pos, b * kKvBlock), to = min(end, (b + 1) * kKvBlock);
        const bool whole = to == (b + 1) * kKvBlock;
        for (int kv = 0; kv < 2; ++kv) {
            const float* src = (kv ? p.v : p.k) + (size_t)h * c.dim;
            float* open = kv ? c.v_open : c.k_open;
            const auto row_of = [&](int pos) { return src + (size_t)(a.row + pos - a.pos) * p.ld; };
            if (whole) {
                float top = 0.f;
                bool odd = false;
                for (int i = tid; i < kKvBlock * c.dim; i += kApThreads) {
                    const int pos = b * kKvBlock + i / c.dim, d = i % c.dim;
                    const float f = pos >= from ? row_of(pos)[d] : c.open_row(open, s, h, pos)[d];
                    x[i] = f;
                    top = fmaxf(top, fabsf(f));
                    odd |= !(fabsf(f) <= CUDART_MAX_NORMAL_F);
                }
                top = lb_warp_max(odd ? CUDART_INF_F : top);
                if ((tid & 31) == 0) s_top[tid >> 5] = top;
                __syncthreads();
                for (int w = 0; w < kApThreads / 32; ++w) top = fmaxf(top, s_top[w]);
                const bool fine = top <= CUDART_MAX_NORMAL_F && top > 0.f;
                const double mul = fine ? __ddiv_rn(127.0, (double)top) : 0.0;
                const size_t at = c.head_of(s, h) * c.blocks + b;
                const int dims = kv ? c.dim_v : c.dim_k;
                uint8_t* codes = (kv ? c.v : c.k) + at * kKvBlock * dims;
                if (tid == 0) (kv ? c.v_top : c.k_top)[at] = fine || top == 0.f ? top : CUDART_NAN_F;
                for (int i = tid; i < kKvBlock * dims; i += kApThreads) {
                    const int pos = i / dims, d = i % dims;
                    const int code = fine && d < c.dim ? lb_quant_i8((double)x[pos * c.dim + d], mul) : 0;
                    codes[kv ? value_byte(pos, d) : key_byte(pos, d, c.dim_k)] = (uint8_t)code;
                }
                __syncthreads();
            }
            const auto keep = [&](int blk) {
                const int f0 = max(a.pos, blk * kKvBlock), f1 = min(end, (blk + 1) * kKvBlock);
                for (int i = tid; i < (f1 - f0) * c.dim; i += kApThreads) {
                    const int pos = f0 + i / c.dim, d = i % c.dim;
                    c.open_row(open, s, h, pos)[d] = row_of(pos)[d];
                }
            };
            if (b >= last - 1 && (b == first || ((b - first) & 1))) keep(b);
            if (b == first)
                for (int blk = max(first + 2, last - 1); blk <= last; ++blk)
                    if (!((blk - first) & 1)) keep(blk);
        }
    }
}

// ---- rows out, as the cache holds them --------------------------------------------------------------------------------------------

struct ReadParams {
    Kv8 c;
    int rows;
    const int32_t *starts, *lengths;
    float *k, *v;  // [rows][heads][dim]
};

__global__ void __launch_bounds__(kApThreads) lb_kv8_read_kernel(const ReadParams p) {
    const Kv8& c = p.c;
    const int s = blockIdx.z, h = blockIdx.y;
    const Span a = span_of(p.starts, p.lengths, p.rows, s);
    if (a.count == 0) return;
    if (!fits(c, a)) {
        if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) atomicExch(c.status, 7);
        return;
    }
    const int closed = (a.pos + a.count) / kKvBlock * kKvBlock;
    for (long long i = (long long)blockIdx.x * kApThreads + threadIdx.x; i < (long long)a.count * c.dim; i += (long long)gridDim.x * kApThreads) {
        const int j = (int)(i / c.dim), d = (int)(i % c.dim), pos = a.pos + j, at = pos % kKvBlock;
        const size_t out = ((size_t)(a.row + j) * c.heads + h) * c.dim + d;
        if (pos < closed) {
            const size_t blk = c.head_of(s, h) * c.blocks + pos / kKvBlock;
            p.k[out] = __fmul_rn((float)(int8_t)c.k[blk * kKvBlock * c.dim_k + key_byte(at, d, c.dim_k)], __fdiv_rn(c.k_top[blk], 127.f));
            p.v[out] = __fmul_rn((float)(int8_t)c.v[blk * kKvBlock * c.dim_v + value_byte(at, d)], __fdiv_rn(c.v_top[blk], 127.f));
        } else {
            p.k[out] = c.open_row(c.k_open, s, h, pos)[d];
            p.v[out] = c.open_row(c.v_open, s, h, pos)[d];
        }
    }
}

// ---- attention --------------------------------------------------------------------------------------------------------------------
//
// Row j of sequence s (head H of the KV head's group) sees positions 0 .. pos + j:  softmax(scale q k) v, the running maximum and
// sum in one pass, everything but the codes in 32 bits.
//
// The products run on the 8-bit integer matrix instruction, codes as they are, exactly: a query row becomes integers q' = round(q 8355711 /
// max |q|), written as q' = d0 + 256 d1 + 65536 d2 with digits in -128 .. 127, and a row of softmax weights, relative to the block's
// own largest score, p' = round(p 16777215) with digits in 0 .. 255.  Three products, one for each digit, make what float32 operands would have
// given (error 2^-24 of the row's largest), and nothing has to be converted on the side of the cache.
//
// Work is a list: sequences, their KV heads, tiles of up to 16 (token, head) rows, blocks.  Every CTA takes an equal stretch of it, so
// long and short sequences share the device evenly; its four warps take every fourth block.  A tile whose blocks lie in
// several CTAs' stretches is put together by the one that comes last, in the stretches' order, so results repeat bit for bit.
constexpr int kAtThreads = 128;
constexpr int kAtWarps = kAtThreads / 32;

struct AttendParams {
    Kv8 c;
    int rows, q_heads, group, ctas;
    const int32_t *starts, *lengths;
    const float* q;
    long long ldq;
    float* out;
    float scale;    // with log2(e)
    float* part;    // [ctas][2][tile rows][dim + 2]
    unsigned* cnt;  // [ctas]
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr float kQueryMax = 8355711.f;   // 127 (1 + 256 + 65536)
constexpr float kWeightMax = 16777215.f;

// bytes k of four integers as a word
__device__ __forceinline__ void digit_words(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t (&w)[3]) {
    const uint32_t a = __byte_perm(x0, x1, 0x5140), b = __byte_perm(x2, x3, 0x5140);
    w[0] = __byte_perm(a, b, 0x5410);
    w[1] = __byte_perm(a, b, 0x7632);
    w[2] = __byte_perm(__byte_perm(x0, x1, 0x0062), __byte_perm(x2, x3, 0x0062), 0x5410);
}

// HALF: tiles of eight rows (rows 8 .. 15 of the MMAs are zero); NK: 32 dimensions each
template <int NK, bool HALF>
struct Shape {
    static constexpr int kRows = HALF ? 8 : 16;
    static constexpr int kSets = HALF ? 1 : 2;  // rows g, and g + 8
    static constexpr int kDimTiles = 4 * NK;
};

template <int NK, bool HALF>
__global__ void __launch_bounds__(kAtThreads) lb_kv8_attend_kernel(const AttendParams p) {
    using S = Shape<NK, HALF>;
    constexpr int R = S::kRows, SETS = S::kSets, NT = S::kDimTiles;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const Kv8& c = p.c;
    const int hd = c.dim;
    float* qs = reinterpret_cast<float*>(smem_raw);       // [R][32 NK] the tile's query rows, zeros behind the dimension
    float* acc = qs + R * 32 * NK;                        // [R][32 NK] the tile's result as it is put together
    float* tail = acc + R * 32 * NK;                      // [R][64] weights of the open block
    float* st_m = tail + R * 64;                          // [warps + 1][R] largest score (log2) and sum
    float* st_l = st_m + (kAtWarps + 1) * R;
    float* qmax = st_l + (kAtWarps + 1) * R;              // [R]
    long long* work = reinterpret_cast<long long*>(qmax + R);  // [seqs + 1] work in front of every sequence
    __shared__ long long s_scan[kAtWarps];
    __shared__ int s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

    // blocks (the open one included) that the last row of sequence s sees, and its tiles
    const auto blocks_of = [&](const Span& a) { return (a.pos + a.count - 1) / kKvBlock + 1; };
    const auto tiles_of = [&](const Span& a) { return (int)(((long long)a.count * p.group + R - 1) / R); };
    {
        long long before = 0;
        for (int s0 = 0; s0 < c.seqs; s0 += kAtThreads) {
            const int s = s0 + tid;
            long long w = 0;
            if (s < c.seqs) {
                const Span a = span_of(p.starts, p.lengths, p.rows, s);
                if (a.count > 0) {
                    if (fits(c, a)) {
                        w = (long long)c.heads * tiles_of(a) * blocks_of(a);
                    } else if (blockIdx.x == 0) {
                        atomicExch(c.status, 7);
                        for (long long i = 0; i < (long long)a.count * p.q_heads * hd; ++i) p.out[(size_t)a.row * p.q_heads * hd + i] = 0.f;
                    }
                }
            }
            long long sum = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (lane == 31) s_scan[warp] = sum;
            __syncthreads();
            for (int w2 = 0; w2 < kAtWarps; ++w2) {
                if (w2 < warp) sum += s_scan[w2];
            }
            if (s < c.seqs) work[s + 1] = before + sum;
            for (int w2 = 0; w2 < kAtWarps; ++w2) before += s_scan[w2];
            __syncthreads();
        }
        if (tid == 0) work[0] = 0;
        __syncthreads();
    }
    const long long total = work[c.seqs];
    const auto begin_of = [&](int cta) { return total * cta / p.ctas; };
    const int me = blockIdx.x;
    long long at = begin_of(me);
    const long long stop = begin_of(me + 1);
    int s = 0;
    {
        int hi = c.seqs;  // the last sequence whose work begins at or in front of `at`
        while (hi - s > 1) {
            const int mid = (s + hi) / 2;
            if (work[mid] <= at) s = mid;
            else hi = mid;
        }
    }
    while (at < stop) {
        while (work[s + 1] <= at) ++s;
        const Span a = span_of(p.starts, p.lengths, p.rows, s);
        const int blocks = blocks_of(a), tiles = tiles_of(a);
        const long long unit = (at - work[s]) / blocks, unit0 = work[s] + unit * blocks;
        const int b0 = (int)(at - unit0), b1 = (int)min((long long)blocks, stop - unit0);
        const int h = (int)(unit / tiles), tile = (int)(unit % tiles);
        const int r0 = tile * R, nr = min(R, a.count * p.group - r0);  // rows i = token * group + head
        const int closed = (a.pos + a.count) / kKvBlock;               // whole blocks
        const auto pos_of = [&](int r) { return a.pos + (r0 + r) / p.group; };

        // query rows
        __syncthreads();
        for (int i = tid; i < R * 32 * NK; i += kAtThreads) {
            const int r = i / (32 * NK), d = i % (32 * NK);
            float f = 0.f;
            if (r < nr && d < hd) f = p.q[(size_t)(a.row + (r0 + r) / p.group) * p.ldq + (size_t)(h * p.group + (r0 + r) % p.group) * hd + d];
            qs[i] = f;
            acc[i] = 0.f;
        }
        __syncthreads();
        for (int r = warp; r < R; r += kAtWarps) {
            float m = 0.f, odd = 0.f;
            for (int d = lane; d < 32 * NK; d += 32) {
                m = fmaxf(m, fabsf(qs[r * 32 * NK + d]));
                odd += qs[r * 32 * NK + d] * 0.f;  // (not a number, from one or an infinity)
            }
            m = lb_warp_max(m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) odd += __shfl_xor_sync(0xffffffffu, odd, o);
            if (lane == 0) qmax[r] = m + odd;
        }
        __syncthreads();
        uint32_t qd[3][NK][2 * SETS];
        float cr[SETS];
        int see[SETS];  // the row's last position, -1: no row
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            const int r = g + 8 * z;
            const float top = qmax[r], div = top > 0.f ? top : 1.f;
            cr[z] = p.scale * top / (kQueryMax * 127.f);
            see[z] = r < nr ? pos_of(r) : -1;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                const int d0 = (kk >> 1) * 64 + ((NK & 1) && kk == NK - 1 ? 8 * t : 16 * t + 8 * (kk & 1));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t digits[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        int v = __float2int_rn(__fdiv_rn(qs[r * 32 * NK + d0 + 4 * half + e], div) * kQueryMax);
                        const int l0 = ((v + 128) & 255) - 128;
                        v = (v - l0) >> 8;
                        const int l1 = ((v + 128) & 255) - 128;
                        v = (v - l1) >> 8;
                        digits[e] = (l0 & 255) | (l1 & 255) << 8 | (v & 255) << 16;
                    }
                    uint32_t w[3];
                    digit_words(digits[0], digits[1], digits[2], digits[3], w);
#pragma unroll
                    for (int k = 0; k < 3; ++k) qd[k][kk][2 * z + half] = w[k];
                }
            }
        }

        float o[SETS][NT][2], m[SETS], l[SETS];
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            m[z] = -CUDART_INF_F;
            l[z] = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) o[z][n][0] = o[z][n][1] = 0.f;
        }
        const size_t head = c.head_of(s, h) * c.blocks;
        const int last_seen = pos_of(nr - 1);
        const int bend = min(min(b1, closed), last_seen / kKvBlock + 1);
        for (int b = b0 + warp; b < bend; b += kAtWarps) {
            const uint8_t* kb = c.k + (head + b) * kKvBlock * c.dim_k;
            const uint8_t* vb = c.v + (head + b) * kKvBlock * c.dim_v;
            const float kt = c.k_top[head + b], vt = c.v_top[head + b];
            float sc[SETS][8][2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                int d[3][4] = {};
                const uint8_t* kj = kb + j * 8 * c.dim_k;
#pragma unroll
                for (int ch = 0; ch < NK / 2; ++ch) {
                    const uint4 f = __ldg(reinterpret_cast<const uint4*>(kj + ch * 512 + lane * 16));
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        mma_s8(d[k], qd[k][2 * ch][0], SETS == 2 ? qd[k][2 * ch][SETS == 2 ? 2 : 0] : 0u, qd[k][2 * ch][1], SETS == 2 ? qd[k][2 * ch][SETS == 2 ? 3 : 0] : 0u, f.x, f.y);
                        mma_s8(d[k], qd[k][2 * ch + 1][0], SETS == 2 ? qd[k][2 * ch + 1][SETS == 2 ? 2 : 0] : 0u, qd[k][2 * ch + 1][1],
                               SETS == 2 ? qd[k][2 * ch + 1][SETS == 2 ? 3 : 0] : 0u, f.z, f.w);
                    }
                }
                if (NK & 1) {
                    const uint2 f = __ldg(reinterpret_cast<const uint2*>(kj + (NK / 2) * 512 + lane * 8));
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        mma_s8(d[k], qd[k][NK - 1][0], SETS == 2 ? qd[k][NK - 1][SETS == 2 ? 2 : 0] : 0u, qd[k][NK - 1][1], SETS == 2 ? qd[k][NK - 1][SETS == 2 ? 3 : 0] : 0u, f.x, f.y);
                }
#pragma unroll
                for (int z = 0; z < SETS; ++z)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int i = 2 * z + e;
                        const float dot = fmaf((float)d[2][i], 65536.f, (float)(d[1][i] * 256 + d[0][i]));
                        sc[z][j][e] = dot * (cr[z] * kt);
                    }
            }
            float mul[SETS];
            uint32_t pd[3][2][2 * SETS];  // [digit][k step][a0, a2 of rows g, then of rows g + 8]
            const bool edge = (b + 1) * kKvBlock - 1 > pos_of(0);
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                float mb = -CUDART_INF_F;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (edge && b * kKvBlock + 8 * j + 2 * t + e > see[z]) sc[z][j][e] = -CUDART_INF_F;
                        mb = fmaxf(mb, sc[z][j][e]);
                    }
                mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
                mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
                const bool any = see[z] >= b * kKvBlock;  // the row sees a part of the block
                uint32_t sum = 0;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t q4[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float w = exp2f(sc[z][4 * ks + 2 * half + (e >> 1)][e & 1] - mb);
                            q4[e] = any ? __float2uint_rn(w * kWeightMax) : 0u;
                            sum += q4[e];
                        }
                        uint32_t w[3];
                        digit_words(q4[0], q4[1], q4[2], q4[3], w);
#pragma unroll
                        for (int k = 0; k < 3; ++k) pd[k][ks][2 * z + half] = w[k];
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                mul[z] = 0.f;
                if (any) {
                    const float mn = fmaxf(m[z], mb);
                    const float old = exp2f(m[z] - mn);
                    mul[z] = exp2f(mb - mn) / kWeightMax;
                    l[z] = fmaf(l[z], old, (float)sum * mul[z]);
                    if (!(fabsf(kt) <= CUDART_MAX_NORMAL_F)) l[z] = CUDART_NAN_F;
                    m[z] = mn;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[z][n][0] *= old;
                        o[z][n][1] *= old;
                    }
                    mul[z] *= __fdiv_rn(vt, 127.f);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (8 * n >= hd) break;
                const uint4 f = __ldg(reinterpret_cast<const uint4*>(vb + n * 512 + lane * 16));
                int d[3][4] = {};
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    mma_u8s8(d[k], pd[k][0][0], SETS == 2 ? pd[k][0][SETS == 2 ? 2 : 0] : 0u, pd[k][0][1], SETS == 2 ? pd[k][0][SETS == 2 ? 3 : 0] : 0u, f.x, f.y);
                    mma_u8s8(d[k], pd[k][1][0], SETS == 2 ? pd[k][1][SETS == 2 ? 2 : 0] : 0u, pd[k][1][1], SETS == 2 ? pd[k][1][SETS == 2 ? 3 : 0] : 0u, f.z, f.w);
                }
#pragma unroll
                for (int z = 0; z < SETS; ++z)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int i = 2 * z + e;
                        const float sum = fmaf((float)d[2][i], 65536.f, (float)(d[1][i] * 256 + d[0][i]));
                        if (see[z] >= b * kKvBlock) o[z][n][e] = fmaf(sum, mul[z], o[z][n][e]);
                    }
            }
        }
        if (t == 0)
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                st_m[warp * R + g + 8 * z] = m[z];
                st_l[warp * R + g + 8 * z] = l[z];
            }

        // the open block: float32 rows, plain multiply-adds
        const bool open = b1 == blocks && closed < blocks;
        const int n_open = open ? a.pos + a.count - closed * kKvBlock : 0;
        float* om = st_m + kAtWarps * R;
        float* ol = st_l + kAtWarps * R;
        if (open) {
            for (int i = warp; i < n_open; i += kAtWarps) {
                const float* kr = c.open_row(c.k_open, s, h, closed * kKvBlock + i);
                for (int r = 0; r < nr; ++r) {
                    float dot = 0.f;
                    for (int d = lane; d < hd; d += 32) dot = fmaf(qs[r * 32 * NK + d], kr[d], dot);
#pragma unroll
                    for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
                    if (lane == 0) tail[r * 64 + i] = dot * p.scale;
                }
            }
            __syncthreads();
            for (int r = warp; r < nr; r += kAtWarps) {
                const int vis = min(n_open, pos_of(r) - closed * kKvBlock + 1);  // (0 or less: none)
                const float s0 = lane < vis ? tail[r * 64 + lane] : -CUDART_INF_F, s1 = lane + 32 < vis ? tail[r * 64 + lane + 32] : -CUDART_INF_F;
                const float top = lb_warp_max(fmaxf(s0, s1));
                const float w0 = lane < vis ? exp2f(s0 - top) : 0.f, w1 = lane + 32 < vis ? exp2f(s1 - top) : 0.f;
                float sum = w0 + w1;
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                tail[r * 64 + lane] = w0;
                tail[r * 64 + lane + 32] = w1;
                if (lane == 0) {
                    om[r] = vis > 0 ? top : -CUDART_INF_F;
                    ol[r] = sum;
                }
            }
            __syncthreads();
            for (int i = tid; i < nr * hd; i += kAtThreads) {
                const int r = i / hd, d = i % hd;
                const int vis = min(n_open, pos_of(r) - closed * kKvBlock + 1);
                float sum = 0.f;
                for (int j = 0; j < vis; ++j) sum = fmaf(tail[r * 64 + j], c.open_row(c.v_open, s, h, closed * kKvBlock + j)[d], sum);
                acc[r * 32 * NK + d] = sum;
            }
        } else if (tid < R) {
            om[tid] = -CUDART_INF_F;
            ol[tid] = 0.f;
        }
        __syncthreads();

        // five partial results of a row into one: acc = sum of o 2^(m - largest m)
        const auto largest = [&](int r) {
            float top = om[r];
            for (int w = 0; w < kAtWarps; ++w) top = fmaxf(top, st_m[w * R + r]);
            return top;
        };
        const auto factor = [](float mine, float top) { return mine == -CUDART_INF_F ? 0.f : exp2f(mine - top); };
        if (open)
            for (int i = tid; i < nr * hd; i += kAtThreads) {
                const int r = i / hd, d = i % hd;
                const float f = factor(om[r], largest(r));
                if (om[r] != -CUDART_INF_F) acc[r * 32 * NK + d] *= f;
            }
        __syncthreads();
        for (int w = 0; w < kAtWarps; ++w) {
            if (w == warp) {
#pragma unroll
                for (int z = 0; z < SETS; ++z) {
                    const int r = g + 8 * z;
                    if (r < nr && m[z] != -CUDART_INF_F) {
                        const float f = factor(m[z], largest(r));
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float& x = acc[r * 32 * NK + 8 * n + 2 * t + e];
                                x = fmaf(o[z][n][e], f, x);
                            }
                    }
                }
            }
            __syncthreads();
        }
        const auto sum_of = [&](int r) {
            const float top = largest(r);
            float sum = om[r] == -CUDART_INF_F && ol[r] == 0.f ? 0.f : ol[r] * factor(om[r], top);
            for (int w = 0; w < kAtWarps; ++w)
                if (st_m[w * R + r] != -CUDART_INF_F || st_l[w * R + r] != 0.f) sum = fmaf(st_l[w * R + r], factor(st_m[w * R + r], top), sum);
            return sum;
        };
        const auto odd_row = [&](int r) { return qmax[r] != qmax[r]; };
        const auto out_of = [&](int r) { return p.out + ((size_t)(a.row + (r0 + r) / p.group) * p.q_heads + (size_t)h * p.group + (r0 + r) % p.group) * hd; };
        if (b0 == 0 && b1 == blocks) {
            for (int i = tid; i < nr * hd; i += kAtThreads) {
                const int r = i / hd, d = i % hd;
                out_of(r)[d] = odd_row(r) ? CUDART_NAN_F : __fdiv_rn(acc[r * 32 * NK + d], sum_of(r));
            }
        } else {
            const size_t row_floats = (size_t)hd + 2;
            const auto slot = [&](int cta, int k) { return p.part + ((size_t)cta * 2 + k) * R * row_floats; };
            float* mine = slot(me, b0 == 0 ? 1 : 0);  // a stretch begins with a tile's end or middle, and ends with a beginning
            for (int i = tid; i < nr * (hd + 2); i += kAtThreads) {
                const int r = i / (hd + 2), d = i % (hd + 2);
                const float f = d == hd ? largest(r) : d == hd + 1 ? sum_of(r) : acc[r * 32 * NK + d];
                __stcg(mine + i, f);
            }
            __threadfence();
            __syncthreads();
            // the CTAs whose stretches this tile lies in
            int lo = (int)(unit0 * p.ctas / total);
            while (begin_of(lo + 1) <= unit0) ++lo;
            while (begin_of(lo) > unit0) --lo;
            const long long end = unit0 + blocks;
            int hi = (int)((end - 1) * p.ctas / total);
            while (begin_of(hi + 1) <= end - 1) ++hi;
            while (begin_of(hi) > end - 1) --hi;
            int parts = 0;  // (stretches may be empty)
            for (int q = lo; q <= hi; ++q) parts += begin_of(q + 1) > begin_of(q);
            if (tid == 0) {
                const unsigned old = atomicAdd(p.cnt + lo, 1u);
                s_last = old + 1 == (unsigned)parts;
                if (s_last) p.cnt[lo] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (int i = tid; i < nr * hd; i += kAtThreads) {
                    const int r = i / hd, d = i % hd;
                    float top = -CUDART_INF_F;
                    for (int q = lo; q <= hi; ++q)
                        if (begin_of(q + 1) > begin_of(q)) top = fmaxf(top, __ldcg(slot(q, begin_of(q) <= unit0 ? 1 : 0) + r * row_floats + hd));
                    float x = 0.f, sum = 0.f;
                    for (int q = lo; q <= hi; ++q) {
                        if (begin_of(q + 1) <= begin_of(q)) continue;
                        const float* from = slot(q, begin_of(q) <= unit0 ? 1 : 0) + r * row_floats;
                        const float mm = __ldcg(from + hd);
                        if (mm == -CUDART_INF_F && __ldcg(from + hd + 1) == 0.f) continue;
                        const float f = factor(mm, top);
                        x = fmaf(__ldcg(from + d), f, x);
                        sum = fmaf(__ldcg(from + hd + 1), f, sum);
                    }
                    out_of(r)[d] = odd_row(r) ? CUDART_NAN_F : __fdiv_rn(x, sum);
                }
            }
        }
        at = unit0 + b1;
    }
}

Kv8 view(const loom_b200_kv8* c) {
    return {c->seqs, c->max_len, c->heads, c->dim, c->blocks, c->dim_k, c->dim_v, c->k, c->v, c->k_top, c->v_top, c->k_open, c->v_open, c->ctx->status_dev};
}

}  // namespace

template <int NK, bool HALF>
static int launch_attend(loom_b200_ctx* ctx, const AttendParams& p) {
    using S = Shape<NK, HALF>;
    const size_t smem = (size_t)S::kRows * (2 * 32 * NK + 64 + 2 * (kAtWarps + 1) + 1) * 4 + (size_t)(p.c.seqs + 1) * 8;
    LB_CUDA(ctx, cudaFuncSetAttribute(lb_kv8_attend_kernel<NK, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    lb_kv8_attend_kernel<NK, HALF><<<p.ctas, kAtThreads, smem, ctx->stream>>>(p);
    LB_CHECK_LAUNCH(ctx, "lb_kv8_attend_kernel");
    return 0;
}

constexpr int kAtCtasPerSm = 2;
constexpr int kKvMaxSeqs = 4096;

extern "C" {

int loom_b200_kv8_create(loom_b200_ctx* ctx, int sequences, int max_len, int kv_heads, int head_dim, loom_b200_kv8** out) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "kv8_create: ctx is NULL");
    LB_REQUIRE(ctx, out != nullptr, "kv8_create: out is NULL");
    *out = nullptr;
    LB_REQUIRE(ctx, sequences > 0 && max_len > 0 && kv_heads > 0 && head_dim > 0, "kv8_create: %d sequences of %d positions, %d KV heads of %d", sequences, max_len, kv_heads, head_dim);
    if (sequences > kKvMaxSeqs || kv_heads > 65535 || head_dim > 256 || max_len > (1 << 30))
        return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "kv8_create: %d sequences (%d at most), %d positions, %d KV heads of %d (256 at most)", sequences, kKvMaxSeqs, max_len, kv_heads, head_dim);
    if (ctx->capturing) return lb_fail(ctx, LOOM_B200_ERR_INVALID, "kv8_create cannot be recorded");
    if (int rc = lb_set_device(ctx)) return rc;
    auto* c = new loom_b200_kv8();
    c->ctx = ctx;
    c->seqs = sequences;
    c->max_len = max_len;
    c->heads = kv_heads;
    c->dim = head_dim;
    c->blocks = max_len / kKvBlock > 0 ? max_len / kKvBlock : 1;
    c->dim_k = (head_dim + 31) / 32 * 32;
    c->dim_v = (head_dim + 7) / 8 * 8;
    const size_t blocks = (size_t)sequences * kv_heads * c->blocks, open = (size_t)sequences * kv_heads * 2 * kKvBlock * head_dim * 4;
    const size_t ctas = (size_t)ctx->sm_count * kAtCtasPerSm;
    c->work_bytes = ctas * 2 * 16 * (head_dim + 2) * 4 + ctas * 4;
    cudaError_t e = cudaSuccess;
    const auto get = [&](void** p, size_t bytes) {
        if (e == cudaSuccess) e = cudaMalloc(p, bytes);
    };
    get((void**)&c->k, blocks * kKvBlock * c->dim_k);
    get((void**)&c->v, blocks * kKvBlock * c->dim_v);
    get((void**)&c->k_top, blocks * 4);
    get((void**)&c->v_top, blocks * 4);
    get((void**)&c->k_open, open);
    get((void**)&c->v_open, open);
    get(&c->work, c->work_bytes);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->work, 0, c->work_bytes, ctx->stream);
    if (e != cudaSuccess) {
        loom_b200_kv8_free(ctx, c);
        return lb_fail(ctx, LOOM_B200_ERR_CUDA, "kv8_create: %d sequences of %d positions: %s", sequences, max_len, cudaGetErrorString(e));
    }
    *out = c;
    return 0;
}

void loom_b200_kv8_free(loom_b200_ctx* ctx, loom_b200_kv8* c) {
    if (!c) return;
    if (ctx) {
        cudaSetDevice(ctx->device);
        cudaStreamSynchronize(ctx->stream);
    }
    void* ptrs[] = {c->k, c->v, c->k_top, c->v_top, c->k_open, c->v_open, c->work};
    for (void* p : ptrs)
        if (p) cudaFree(p);
    delete c;
}

// what the three calls on rows check
static int kv8_ready(loom_b200_ctx* ctx, const loom_b200_kv8* c, int rows, const int32_t* starts, const int32_t* lengths, const void* a, const void* b, const char* who) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "%s: ctx is NULL", who);
    LB_REQUIRE(ctx, c && lengths && a && b, "%s: NULL argument", who);
    LB_REQUIRE(ctx, c->ctx == ctx, "%s: the cache belongs to another context", who);
    LB_REQUIRE(ctx, rows > 0, "%s: %d rows", who, rows);
    LB_REQUIRE(ctx, starts || rows <= c->seqs, "%s: %d rows without starts, one each of %d sequences", who, rows, c->seqs);
    return 0;
}

int loom_b200_kv8_append(loom_b200_ctx* ctx, loom_b200_kv8* c, int rows, const int32_t* starts, const int32_t* lengths, const float* k, const float* v, long long ld) {
    if (int rc = kv8_ready(ctx, c, rows, starts, lengths, k, v, "kv8_append")) return rc;
    LB_REQUIRE(ctx, ld >= (long long)c->heads * c->dim, "kv8_append: %lld floats between rows of %d", ld, c->heads * c->dim);
    if (int rc = lb_set_device(ctx)) return rc;
    AppendParams p{view(c), rows, starts, lengths, k, v, ld};
    const size_t smem = (size_t)kKvBlock * c->dim * 4;
    LB_CUDA(ctx, cudaFuncSetAttribute(lb_kv8_append_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvBlock * 256 * 4));
    const int blocks = starts ? (rows + kKvBlock - 2) / kKvBlock + 1 : 1;
    lb_kv8_append_kernel<<<dim3(blocks < 256 ? blocks : 256, c->heads, c->seqs), kApThreads, smem, ctx->stream>>>(p);
    LB_CHECK_LAUNCH(ctx, "lb_kv8_append_kernel");
    return 0;
}

int loom_b200_kv8_read(loom_b200_ctx* ctx, loom_b200_kv8* c, int rows, const int32_t* starts, const int32_t* lengths, float* k, float* v) {
    if (int rc = kv8_ready(ctx, c, rows, starts, lengths, k, v, "kv8_read")) return rc;
    if (int rc = lb_set_device(ctx)) return rc;
    ReadParams p{view(c), rows, starts, lengths, k, v};
    const long long per = starts ? ((long long)rows * c->dim + kApThreads - 1) / kApThreads : 1;
    lb_kv8_read_kernel<<<dim3((unsigned)(per < 256 ? per : 256), c->heads, c->seqs), kApThreads, 0, ctx->stream>>>(p);
    LB_CHECK_LAUNCH(ctx, "lb_kv8_read_kernel");
    return 0;
}

int loom_b200_kv8_attend(loom_b200_ctx* ctx, loom_b200_kv8* c, int rows, int heads, const int32_t* starts, const int32_t* lengths, const float* q, long long ldq, double scale, float* out) {
    if (int rc = kv8_ready(ctx, c, rows, starts, lengths, q, out, "kv8_attend")) return rc;
    LB_REQUIRE(ctx, heads > 0 && heads % c->heads == 0, "kv8_attend: %d query heads over %d KV heads", heads, c->heads);
    LB_REQUIRE(ctx, ldq >= (long long)heads * c->dim, "kv8_attend: %lld floats between rows of %lld", ldq, (long long)heads * c->dim);
    LB_REQUIRE(ctx, scale == scale, "kv8_attend: scale is not a number");
    AttendParams p;
    p.c = view(c);
    p.rows = rows;
    p.q_heads = heads;
    p.group = heads / c->heads;
    LB_REQUIRE(ctx, (long long)rows * p.group < (1 << 30), "kv8_attend: %d rows of %d heads", rows, heads);
    if (int rc = lb_set_device(ctx)) return rc;
    p.ctas = ctx->sm_count * kAtCtasPerSm;
    p.starts = starts;
    p.lengths = lengths;
    p.q = q;
    p.ldq = ldq;
    p.out = out;
    p.scale = (float)((scale > 0 ? scale : 1.0 / sqrt((double)c->dim)) * 1.4426950408889634);
    p.part = (float*)c->work;
    p.cnt = (unsigned*)(p.part + (size_t)p.ctas * 2 * 16 * (c->dim + 2));
    const bool half = !starts && p.group <= 8;
    switch (c->dim_k / 32) {
        case 1: return half ? launch_attend<1, true>(ctx, p) : launch_attend<1, false>(ctx, p);
        case 2: return half ? launch_attend<2, true>(ctx, p) : launch_attend<2, false>(ctx, p);
        case 3: return half ? launch_attend<3, true>(ctx, p) : launch_attend<3, false>(ctx, p);
        case 4: return half ? launch_attend<4, true>(ctx, p) : launch_attend<4, false>(ctx, p);
        case 5: return launch_attend<5, true>(ctx, p);
        case 6: return launch_attend<6, true>(ctx, p);
        case 7: return launch_attend<7, true>(ctx, p);
        default: return launch_attend<8, true>(ctx, p);
    }
}

}  // extern "C"
