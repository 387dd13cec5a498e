// kv8.cu -- a cache of keys and values in 8 bits for several sequences, and attention over it.
//
// Positions of a sequence go by blocks of 64.  A whole block is held in 8 bits, with one scale for each KV head, keys and values apart:
// a = largest |x| of the block's 64 rows of that head, code = round(x * 127 / a) half away from zero (the arithmetic of the activation
// quantizer: float64 quotient and product), value = code * a / 127.  A block with a value that is not finite reads as not-a-numbers.
// The positions behind the last whole block are held in float32 as they came; of the block in front of them the float32 rows stay too, so
// a sequence may be cut back into it and go on from there.  There are two places for such rows, for blocks of even and of odd numbers, and a
// note of which blocks' they are: cut back further, or into a block whose place another one has taken since, a sequence goes on from that
// block's rows as the codes have them (it was whole before another one could take its place).
//
// Codes lie as the tensor core's B operands want them, so that a warp's load of 16 bytes a lane is 512 consecutive bytes and needs no
// shared memory on its way (lane = 4 g + t):
//   keys    per block and KV head [position / 8][64 dimensions][position % 8 = g][64 bytes], the last 32 dimensions, if alone, 32 bytes
//           instead; lane (g, t) takes dimensions 16 t .. 16 t + 15 of a chunk: which of them an MMA sees as which k is the same for the
//           queries, so the order cancels
//   values  [dimension / 8][dimension % 8 = g][t][16 positions 8 j + 2 t + e, (j, e) in order]: the positions whose scores lane t holds
//           after the products with the keys
#include "serving.cuh"
#include "umma.cuh"

#include <cuda_fp16.h>
#include <math_constants.h>

#include <cmath>

namespace {

struct Kv8 {
    int seqs, max_len, heads, dim, blocks, dim_k, dim_v, dim_o;
    uint8_t *k, *v;
    float *k_top, *v_top, *k_open, *v_open;
    int* placed;  // [seqs][heads][keys, values][2] the even and the odd block whose rows are in the open places, -1: none
    int* status;

    __host__ __device__ size_t head_of(int s, int h) const { return (size_t)s * heads + h; }
    __device__ __forceinline__ float* open_row(float* base, int s, int h, int pos) const {
        return base + ((head_of(s, h) * 2 + (pos / kKvBlock & 1)) * kKvBlock + pos % kKvBlock) * dim_o;
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

// Rows that are not taken are said in the status word, unless a wait that ran out stands there: that one spoils other results too.
__device__ __forceinline__ void say_not_taken(int* status, int code) { atomicCAS(status, 0, code); }

// byte of a key's dimension d at place p of its block; of a value's
__device__ __forceinline__ int key_byte(int p, int d, int dim_k) {
    const int c = d >> 6, whole = dim_k >> 6;
    return (p >> 3) * 8 * dim_k + (c < whole ? c * 512 + (p & 7) * 64 + (d & 63) : whole * 512 + (p & 7) * 32 + (d & 31));
}
__device__ __forceinline__ int value_byte(int p, int d) { return (d >> 3) * 512 + (d & 7) * 64 + (p >> 1 & 3) * 16 + (p >> 3) * 2 + (p & 1); }

// ---- rows in, and rows out as the cache holds them ---------------------------------------------------------------------------------
//
// An item is a block that the call's rows touch, of one KV head, keys or values; a CTA finds its block in the list of them by itself.  A
// thread has eight positions of four dimensions at a time, so that its codes are words of what the cache holds and every access
// fills whole sectors: keys, positions j, 8 + j, 16 + j and so on; values, the pairs 2 t, 2 t + 1 of four groups of eight.
//
// Append writes the rows to the open rows where the block is one of the last two, and where they complete it (the first of its rows may
// be there already) makes the codes.  Open rows go by the block's parity: the rows that the first block still reads there may be what
// a block two further on replaces, so the CTA of the first block writes for that one too, after its own reads.
//
// A code is the float32 product where that is further than 2^-10 from a half (its error is below 2^-16) and the float64 arithmetic
// elsewhere, one value in five hundred: conversions and float64 take sixteen values a clock of an SM.
//
// Bound: memory; for few rows, latencies.  4944 rows of eight heads of 128 in 8 sequences: append 18.7 us, read 10.8 us (52 MB
// each way, 2.8 and 4.8 TB/s: waves of CTAs, each its loads, its largest value and its stores one behind the other); one row of each of 64 sequences: 7.4 and 6.1 us.  A CTA for each head: with two, four and all eight heads
// a CTA the append takes 28, 38 and 66 us; runs of two to eight blocks a CTA 21 to 40 us.
constexpr int kRowThreads = 256;

struct RowParams {
    Kv8 c;
    int rows;
    const int32_t *starts, *lengths;
    const float *k, *v;  // append's
    long long ld;        // floats from one row of k (and of v) to the next
    float *k_out, *v_out;  // read's: [rows][heads][dim]
    int wide;            // rows begin on 16 bytes
};

struct Unit {
    int col, oct;  // dimensions 4 col .. 4 col + 3; which positions
};
// unit u of a block: warps take 32 bytes of four key positions, or the values of four columns whole
template <bool V>
__device__ __forceinline__ Unit unit_of(int u) {
    const int l = u & 31, w = u >> 5;
    if (V) return {4 * w + (l & 3), l >> 2};
    return {8 * (w >> 1) + (l & 7), 4 * (w & 1) + (l >> 3)};
}
template <bool V>
__device__ __forceinline__ int place_of(int oct, int i) {
    return V ? 8 * (4 * (oct & 1) + (i >> 1)) + 2 * (oct >> 1) + (i & 1) : 8 * i + oct;
}

__device__ __forceinline__ int blocks_of(const Kv8& c, const Span& a) {
    if (a.count == 0) return 0;
    return fits(c, a) ? (a.pos + a.count - 1) / kKvBlock - a.pos / kKvBlock + 1 : 1;
}

// Block n of the list, in the sequences' order: its sequence, or -1, and which of the sequence's it is.  For the whole CTA.
struct Item {
    Span a;
    int seq, block;
    bool more;  // the list goes on behind this round of the grid
};
__device__ __forceinline__ Item item_of(const RowParams& p, int n) {
    __shared__ int s_sum[kRowThreads / 32], s_seq, s_block, s_span[3];
    Item r;
    if (!p.starts) {
        r.seq = n < min(p.rows, p.c.seqs) ? n : -1;
        r.block = 0;
        r.more = false;
        if (r.seq >= 0) r.a = span_of(p.starts, p.lengths, p.rows, r.seq);
    } else {
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
        __syncthreads();  // (the item before has been read)
        if (tid == 0) s_seq = -1;
        for (int s0 = 0; s0 < p.c.seqs; s0 += kRowThreads) {
            const int s = s0 + tid;
            Span a = {0, 0, 0};
            if (s < p.c.seqs) a = span_of(p.starts, p.lengths, p.rows, s);
            const int mine = blocks_of(p.c, a);
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (lane == 31) s_sum[warp] = sum;
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int w = 0; w < kRowThreads / 32; ++w) {
                const int u = s_sum[w];
                sum += w < warp ? u : 0;
                all += u;
            }
            if (n < sum && n >= sum - mine) {
                s_seq = s;
                s_block = n - (sum - mine);
                s_span[0] = a.row;
                s_span[1] = a.count;
                s_span[2] = a.pos;
            }
            n -= all;
            __syncthreads();
        }
        r.more = n + (int)gridDim.y < 0;  // (n: less all there are)
        r.seq = s_seq;
        r.block = s_block;
        r.a = {s_span[0], s_span[1], s_span[2]};
    }
    return r;
}

__device__ __forceinline__ float4 load_four(const float* row, int d, int dim, bool wide) {
    if (wide) return __ldcs(reinterpret_cast<const float4*>(row + d));
    return make_float4(__ldcs(row + d), d + 1 < dim ? __ldcs(row + d + 1) : 0.f, d + 2 < dim ? __ldcs(row + d + 2) : 0.f, d + 3 < dim ? __ldcs(row + d + 3) : 0.f);
}

__device__ __forceinline__ void store_four(float* row, int d, int dim, bool wide, const float4& f) {
    if (wide) {
        __stcs(reinterpret_cast<float4*>(row + d), f);
    } else {
        row[d] = f.x;
        if (d + 1 < dim) row[d + 1] = f.y;
        if (d + 2 < dim) row[d + 2] = f.z;
        if (d + 3 < dim) row[d + 3] = f.w;
    }
}

// codes of four values, a byte each
__device__ __noinline__ uint32_t codes_exactly(float4 x, double mul) {
    const uint32_t n0 = lb_quant_i8((double)x.x, mul), n1 = lb_quant_i8((double)x.y, mul), n2 = lb_quant_i8((double)x.z, mul), n3 = lb_quant_i8((double)x.w, mul);
    return __byte_perm(__byte_perm(n0, n1, 0x0040), __byte_perm(n2, n3, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t codes_of(const float4& x, float mulf, double mul) {
    constexpr float kRound = 12582912.f;  // 1.5 2^23: a sum's low bits are the nearest integer
    const float f[4] = {x.x, x.y, x.z, x.w};
    uint32_t n[4];
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float r = fmaf(f[e], mulf, kRound);
        n[e] = __float_as_uint(r);
        off = fmaxf(off, fabsf(fmaf(f[e], mulf, kRound - r)));
    }
    if (off > 0.5f - 1.f / 1024.f) return codes_exactly(x, mul);
    return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
}

template <int NU, bool V>
__device__ __forceinline__ void append_block(const RowParams& p, const Item& it, int b, int h, bool keep, uint32_t* s_top) {
    const Kv8& c = p.c;
    const Span a = it.a;
    const int tid = threadIdx.x, s = it.seq;
    const int dims = V ? c.dim_v : c.dim_k;
    const int units = V ? (dims + 15) / 16 * 32 : dims * 2;
    const float* src = (V ? p.v : p.k) + (size_t)h * c.dim;
    float* open = V ? c.v_open : c.k_open;
    const auto row_of = [&](int pos) { return src + (size_t)(a.row + pos - a.pos) * p.ld; };
    const auto open_of = [&](int pos) { return c.open_row(open, s, h, pos); };
    float4 x[NU][8];
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        const Unit w = unit_of<V>(tid + j * kRowThreads);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pos = b * kKvBlock + place_of<V>(w.oct, i);
            x[j][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (4 * w.col >= c.dim) continue;
            if (pos >= a.pos) x[j][i] = load_four(row_of(pos), 4 * w.col, c.dim, p.wide);
            else x[j][i] = *reinterpret_cast<const float4*>(open_of(pos) + 4 * w.col);
        }
    }
    uint32_t bits = 0;  // the largest magnitude's, or those of what is no finite value, which are above all
#pragma unroll
    for (int j = 0; j < NU; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 f = x[j][i];
            bits = max(max(bits, __float_as_uint(f.x) & 0x7fffffffu), __float_as_uint(f.y) & 0x7fffffffu);
            bits = max(max(bits, __float_as_uint(f.z) & 0x7fffffffu), __float_as_uint(f.w) & 0x7fffffffu);
        }
    bits = __reduce_max_sync(0xffffffffu, bits);
    if ((tid & 31) == 0) s_top[tid >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) bits = max(bits, s_top[w]);
    const float top = __uint_as_float(bits);
    const bool fine = top <= CUDART_MAX_NORMAL_F && top > 0.f;
    const double mul = fine ? __ddiv_rn(127.0, (double)top) : 0.0;
    const bool fast = top > 1e-30f && top < 1e30f;  // (the float32 factor is a normal number)
    const float mulf = (float)mul;
    const size_t at = c.head_of(s, h) * c.blocks + b;
    uint8_t* codes = (V ? c.v : c.k) + at * kKvBlock * dims;
    if (tid == 0) (V ? c.v_top : c.k_top)[at] = fine || top == 0.f ? top : CUDART_NAN_F;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        const int u = tid + j * kRowThreads;
        const Unit w = unit_of<V>(u);
        if (u >= units || 4 * w.col >= dims) continue;
        uint32_t n[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = fast ? codes_of(x[j][i], mulf, mul) : fine ? codes_exactly(x[j][i], mul) : 0u;
        if (V) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t sel = e | (e + 4) << 4;
                const uint32_t lo = __byte_perm(__byte_perm(n[0], n[1], sel), __byte_perm(n[2], n[3], sel), 0x5410);
                const uint32_t hi = __byte_perm(__byte_perm(n[4], n[5], sel), __byte_perm(n[6], n[7], sel), 0x5410);
                *reinterpret_cast<uint2*>(codes + value_byte(place_of<V>(w.oct, 0), 4 * w.col + e)) = make_uint2(lo, hi);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(codes + key_byte(place_of<V>(w.oct, i), 4 * w.col, dims)) = n[i];
        }
    }
    if (keep)
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            const Unit w = unit_of<V>(tid + j * kRowThreads);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pos = b * kKvBlock + place_of<V>(w.oct, i);
                if (4 * w.col < c.dim && pos >= a.pos) *reinterpret_cast<float4*>(open_of(pos) + 4 * w.col) = x[j][i];
            }
        }
    __syncthreads();  // (s_top)
}

// rows of block b into the open rows, or out of them
template <bool IN>
__device__ __forceinline__ void copy_rows(const RowParams& p, const Item& it, int b, int kv, int h) {
    const Kv8& c = p.c;
    const Span a = it.a;
    const int from = max(a.pos, b * kKvBlock), n = min(a.pos + a.count, (b + 1) * kKvBlock) - from;
    const int d4 = c.dim_o / 4;
    float* open = kv ? c.v_open : c.k_open;
    const float* src = kv ? p.v : p.k;
    float* out = kv ? p.v_out : p.k_out;
    const long long ld = IN ? p.ld : (long long)c.heads * c.dim;
    for (int i = threadIdx.x; i < n * d4; i += kRowThreads) {
        const int d = 4 * (i % d4), r = i / d4;
        const size_t at = (size_t)(a.row + from - a.pos + r) * ld + (size_t)h * c.dim;
        float4* in = reinterpret_cast<float4*>(c.open_row(open, it.seq, h, from + r) + d);
        if (IN) *in = load_four(src + at, d, c.dim, p.wide);
        else store_four(out + at, d, c.dim, p.wide, *in);
    }
}

// Rows of block b in front of position `end` from its codes into its open place, which holds another block's: the sequence was cut back to there.
template <bool V>
__device__ __forceinline__ void restore_rows(const Kv8& c, int s, int h, int b, int end) {
    const int dims = V ? c.dim_v : c.dim_k, n = end - b * kKvBlock;
    const size_t at = c.head_of(s, h) * c.blocks + b;
    const uint8_t* codes = (V ? c.v : c.k) + at * kKvBlock * dims;
    const float scale = __fdiv_rn((V ? c.v_top : c.k_top)[at], 127.f);
    float* open = c.open_row(V ? c.v_open : c.k_open, s, h, b * kKvBlock);
#pragma unroll 1
    for (int i = threadIdx.x; i < n * c.dim; i += kRowThreads) {
        const int r = i / c.dim, d = i - r * c.dim;
        open[(size_t)r * c.dim_o + d] = __fmul_rn((float)(int8_t)codes[V ? value_byte(r, d) : key_byte(r, d, dims)], scale);
    }
    __syncthreads();
}

template <int NU>
__global__ void __launch_bounds__(kRowThreads, NU == 1 ? 4 : 2) lb_kv8_append_kernel(const RowParams p) {
    __shared__ uint32_t s_top[kRowThreads / 32];
    lb_pdl_launch_dependents();
    lb_pdl_wait();
    const int kv = blockIdx.x & 1, h = blockIdx.x >> 1;
    bool more = true;
    for (int n = blockIdx.y; more; n += gridDim.y) {
        const Item it = item_of(p, n);
        if (it.seq < 0) return;
        more = it.more;
        // The first block's CTA alone reads and writes the note of its head's places.  (Read ahead of what the sequence's length decides.)
        const auto placed = [&](int i) -> int* { return p.c.placed + (p.c.head_of(it.seq, h) * 2 + kv) * 2 + i; };
        const int2 were = *reinterpret_cast<const int2*>(placed(0));
        if (!fits(p.c, it.a)) {
            if (blockIdx.x == 0 && threadIdx.x == 0) say_not_taken(p.c.status, 7);
            continue;
        }
        if (it.a.count == 0) continue;
        const int end = it.a.pos + it.a.count, first = it.a.pos / kKvBlock, last = (end - 1) / kKvBlock, b = first + it.block;
        const bool keep = b >= last - 1 && (b == first || ((b - first) & 1));
        const int there = it.a.pos % kKvBlock == 0 ? first : first & 1 ? were.y : were.x;
        const bool whole = (b + 1) * kKvBlock <= end;
        if (!whole && keep) copy_rows<true>(p, it, b, kv, h);
        if (b == first && there >= 0 && there != first && first < p.c.blocks) {  // (a last block that is no whole one has no codes)
            if (kv) restore_rows<true>(p.c, it.seq, h, first, it.a.pos);
            else restore_rows<false>(p.c, it.seq, h, first, it.a.pos);
        }
        if (whole) {
            if (kv) append_block<NU, true>(p, it, b, h, keep, s_top);
            else append_block<NU, false>(p, it, b, h, keep, s_top);
        }
        if (b == first && last - first >= 2) copy_rows<true>(p, it, last - ((last - first) & 1), kv, h);  // (behind the barrier that append_block ends with)
        if (b == first) {
            if (last == first) __syncthreads();  // (everyone has read it; one of several blocks is whole and has ended with a barrier)
            if (threadIdx.x < 2 && (threadIdx.x == 0 || last > first)) *placed(last - threadIdx.x & 1) = last - threadIdx.x;
        }
    }
}

// four codes times the block's scale
__device__ __forceinline__ float4 values_of(uint32_t w, float a) {
    w ^= 0x80808080u;
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + e)) - 8388736.f, a);  // 2^23 + 128
    return make_float4(f[0], f[1], f[2], f[3]);
}

template <bool V>
__device__ __forceinline__ void read_block(const RowParams& p, const Item& it, int b, int h) {
    const Kv8& c = p.c;
    const Span a = it.a;
    const int s = it.seq;
    const int dims = V ? c.dim_v : c.dim_k;
    const size_t at = c.head_of(s, h) * c.blocks + b;
    const uint8_t* codes = (V ? c.v : c.k) + at * kKvBlock * dims;
    const float scale = __fdiv_rn(__ldg((V ? c.v_top : c.k_top) + at), 127.f);
    const int units = V ? (dims + 15) / 16 * 32 : dims * 2;
    for (int u = threadIdx.x; u < units; u += kRowThreads) {
        const Unit w = unit_of<V>(u);
        if (4 * w.col >= c.dim) continue;
        uint32_t n[8];
        if (V) {
            uint2 e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = *reinterpret_cast<const uint2*>(codes + value_byte(place_of<V>(w.oct, 0), 4 * w.col + i));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t sel = i | (i + 4) << 4;
                n[i] = __byte_perm(__byte_perm(e[0].x, e[1].x, sel), __byte_perm(e[2].x, e[3].x, sel), 0x5410);
                n[4 + i] = __byte_perm(__byte_perm(e[0].y, e[1].y, sel), __byte_perm(e[2].y, e[3].y, sel), 0x5410);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = *reinterpret_cast<const uint32_t*>(codes + key_byte(place_of<V>(w.oct, i), 4 * w.col, dims));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pos = b * kKvBlock + place_of<V>(w.oct, i);
            if (pos < a.pos) continue;
            float* out = (V ? p.v_out : p.k_out) + ((size_t)(a.row + pos - a.pos) * c.heads + h) * c.dim;
            store_four(out, 4 * w.col, c.dim, p.wide, values_of(n[i], scale));
        }
    }
}

__global__ void __launch_bounds__(kRowThreads, 3) lb_kv8_read_kernel(const RowParams p) {
    lb_pdl_launch_dependents();
    lb_pdl_wait();
    const int kv = blockIdx.x & 1, h = blockIdx.x >> 1;
    bool more = true;
    for (int n = blockIdx.y; more; n += gridDim.y) {
        const Item it = item_of(p, n);
        if (it.seq < 0) return;
        more = it.more;
        if (!fits(p.c, it.a)) {
            if (blockIdx.x == 0 && threadIdx.x == 0) say_not_taken(p.c.status, 7);
            continue;
        }
        if (it.a.count == 0) continue;
        const int b = it.a.pos / kKvBlock + it.block;
        if ((b + 1) * kKvBlock > it.a.pos + it.a.count) {
            copy_rows<false>(p, it, b, kv, h);
        } else {
            if (kv) read_block<true>(p, it, b, h);
            else read_block<false>(p, it, b, h);
        }
    }
}

// ---- attention --------------------------------------------------------------------------------------------------------------------
//
// Row j of sequence s (head H of the KV head's group) sees positions 0 .. pos + j:  softmax(scale q k) v, the running maximum and
// sum in one pass, everything but the codes in 32 bits.
//
// The products run on the 8-bit integer matrix instruction, codes as they are, exactly: a query row becomes integers q' = round(q 8355584 /
// max |q|), written as q' = d0 + 256 d1 + 65536 d2 with digits in -128 .. 127, and a row of softmax weights, relative to the block's
// own largest score, p' = round(p 16777215) with digits in 0 .. 255.  Three products, one for each digit, make what float32 operands would have
// given (error 2^-24 of the row's largest), and nothing has to be converted on the side of the cache.  Put together in float32 they lose what
// the lowest digit's sum has below 256, 2^-25 of the largest possible sum.
//
// Work is a list: sequences, their KV heads, tiles of (token, head) rows, blocks.  A tile is either the rows of one warp's MMAs, and the four
// warps take every fourth block, each through a ring of its own (one token and a few: the cache is read once); or four times that,
// and the warps share the blocks (sequences of many rows where the kernel for portions does not have them, kv8_rows.cuh).  Every CTA
// finds its place in the list by itself: tiles are cut into parts of nearly equal work, the smallest size with no more parts than CTAs
// (a part's fixed cost is that of six blocks, so no CTA should have two); where there are more tiles than CTAs, each takes those that
// begin in its stretch of the work.  The parts of a tile are put together by the CTA that comes last, in their order, so results repeat bit
// for bit.
//
// Bound: the codes' way from memory, 5.4 TB/s while it lasts, behind the list and the queries (4 us) and in front of open blocks and joining.  One
// row of 32 heads over 8 of 128 dimensions at position 131,071: 67.5 us, 49 of them the blocks; 16 sequences of 2554 positions on the average: 36.9 us; 20
// heads over 5 at 1040: 14.1 us.
constexpr int kAtThreads = 128;
constexpr int kAtWarps = kAtThreads / 32;
constexpr int kAtRowsNk = 4;      // the kernel for portions has up to 128 dimensions: a row's results stay in a thread's registers
constexpr int kAtWideRows = 48;   // rows of a sequence beyond which its tiles are wide
constexpr int kAtPortionRows = 256;  // rows of a KV head's group, in a call, beyond which the kernel for portions looks for some
constexpr int kAtSizes = 8;       // sizes of parts that are tried: 1, 1 + 1/8, 1 + 2/8 and so on of an equal share
constexpr int kAtOpenFew = 6;     // what an open block costs, in blocks: beside one token's rows (5.8 us, four blocks 3.4 us)
constexpr int kAtOpenWide = 3;    // and beside a wide tile's
constexpr int kAtOpenRows = 16;   // rows that go through the open block together

// Work is counted in 31 bits; a call with more than they hold (sequences that share rows, as no others can) is not done at all.
constexpr double kAtMostWork = 2147483648.0 - 1024;
constexpr int kAtTooMuch = 8;  // the status then
__device__ __forceinline__ unsigned add_work(unsigned a, unsigned b) { return a + min(b, ~a); }

struct AttendParams {
    Kv8 c;
    int rows, q_heads, group, ctas;
    unsigned group_inv;  // 2^32 / group, rounded up, for quotients of numbers below 2^16; 0: one head a group
    const int32_t *starts, *lengths;
    const float* q;
    long long ldq;
    float* out;
    float scale;    // with log2(e)
    float* part;    // [2 ctas + 1][largest tile][part_ld]
    int part_ld;    // dimensions, rounded up to four, largest score, sum, two more
    unsigned* cnt;  // [2 ctas + 1]
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
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void copy16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(lb_smem_u32(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr float kQueryMax = 8355584.f;  // (three digits reach 127 (1 + 256 + 65536) = 8355711; a product with the row's scale may round up)
constexpr float kWeightMax = 16777215.f;

// bytes k of four integers as a word
__device__ __forceinline__ void digit_words(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t (&w)[3]) {
    const uint32_t a = __byte_perm(x0, x1, 0x5140), b = __byte_perm(x2, x3, 0x5140);
    w[0] = __byte_perm(a, b, 0x5410);
    w[1] = __byte_perm(a, b, 0x7632);
    w[2] = __byte_perm(__byte_perm(x0, x1, 0x0062), __byte_perm(x2, x3, 0x0062), 0x5410);
}
// Accumulators start at the bit pattern of 1.5 2^23, so that a sum of up to 2^22 comes out as the float32 that is larger by as much (the
// largest here is 256 dimensions x 128 x 127): no conversion, whose pipe takes sixteen values a clock and SM.
constexpr int kSumBits = 0x4b400000;
constexpr float kSumFrom = 12582912.f;
// d0 + 256 d1 + 65536 d2, over 256, of three such sums
__device__ __forceinline__ float digits_sum(int d0, int d1, int d2) {
    const float low = fmaf(__int_as_float(d0), 1.f / 256.f, __int_as_float(d1));
    return fmaf(__int_as_float(d2) - kSumFrom, 256.f, low) - (kSumFrom + kSumFrom / 256.f);
}

__device__ __forceinline__ void add_scaled(float4& x, const float4& v, float f) { x = make_float4(fmaf(v.x, f, x.x), fmaf(v.y, f, x.y), fmaf(v.z, f, x.z), fmaf(v.w, f, x.w)); }
__device__ __forceinline__ void sums_begin(int (&d)[3][4]) {
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[k][i] = kSumBits;
}

// SETS: rows of a warp's tile / 8 (with one, rows 8 .. 15 of the MMAs are zero); NK: 32 dimensions each
template <int NK, int SETS>
struct AttendShape {
    static constexpr int kRows = 8 * SETS;              // of a warp
    static constexpr int kTile = kAtWarps * kRows;      // of a wide tile
    static constexpr int kSlot = kKvBlock * 32 * NK;    // bytes of 64 keys or values
    // CTAs of an SM, and slots of a warp.  Two CTAs with three slots stream the cache at 5.4 TB/s; three CTAs with two slots each at 4.1 (a
    // warp then has one copy under way while it computes, and 168 registers).
    static constexpr int kPerSm = NK > 4 ? 1 : 2;
    static constexpr int kRing = 3;
    static constexpr int kSlots = kAtWarps * kRing;             // or pairs of them that all share
    static constexpr int kLd = 32 * NK + 8;             // floats of a row of partial results (the eight spread rows over banks)
    static constexpr int kLdOpen = 32 * NK + 16;        // of a key of the open block (two rows of a quarter warp in different banks)
    static constexpr size_t kMerge = ((size_t)(kTile + kAtOpenRows) * kLd + kKvBlock * kAtOpenRows + kKvBlock / 2 * (kLdOpen + 32 * NK)) * 4;
    static constexpr size_t kSmem = kMerge > (size_t)kSlots * kSlot ? kMerge : (size_t)kSlots * kSlot;
};

// WIDE: with wide tiles, for sequences that may have many rows
template <int NK, int SETS, bool WIDE>
__global__ void __launch_bounds__(kAtThreads, AttendShape<NK, SETS>::kPerSm) lb_kv8_attend_kernel(const AttendParams p) {
    using S = AttendShape<NK, SETS>;
    constexpr int RW = S::kRows, NT = 4 * NK, LD = S::kLd, D4 = 8 * NK, RING = S::kRing, STAGES = S::kSlots / 2;
    extern __shared__ __align__(16) uint8_t ring[];
    // over the ring, once a tile's blocks are through
    float* pieces = reinterpret_cast<float*>(ring);  // [4 warps][RW][LD], or [4 RW][LD] of a wide tile
    float* open_q = pieces + S::kTile * LD;          // [16][LD]
    float* open_w = open_q + kAtOpenRows * LD;       // [64][16] scores, then weights
    float* open_k = open_w + kKvBlock * kAtOpenRows; // [32][kLdOpen] half of its keys, then of the values, [32][dim_o]
    float* open_v = open_k + kKvBlock / 2 * S::kLdOpen;  // [32][dim_o] the other half of the values
    __shared__ float s_m[kAtWarps][S::kTile], s_l[kAtWarps][S::kTile];
    __shared__ float s_f[2][kAtOpenRows];            // factors of a row's piece and of its open block
    __shared__ int s_span[kAtThreads][3];            // the first sequences' rows
    __shared__ unsigned s_scan[kAtWarps][kAtSizes], s_at;
    __shared__ int s_seq, s_last, s_misfit;
    __shared__ __align__(8) uint64_t s_bar;  // copies of parts
    uint32_t bar_phase = 0;
    const Kv8& c = p.c;
    const int hd = c.dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    lb_pdl_launch_dependents();
    lb_pdl_wait();

    // ---- the list of work ----
    struct Seq {
        Span a;
        int blocks, tiles;  // blocks (the open one included) that its last row sees
        int load;           // the same, with what the open one costs
        int cost;           // of a block of a tile: 2^cost
        unsigned work;
    };
    if (tid == 0) {
        lb_mbar_init(&s_bar, 1);
        lb_fence_mbar_init();
        s_misfit = 0;
    }
    for (int i = tid; i < min(c.seqs, kAtThreads); i += kAtThreads) {
        const Span a = span_of(p.starts, p.lengths, p.rows, i);
        s_span[i][0] = a.row;
        s_span[i][1] = a.count;
        s_span[i][2] = a.pos;
    }
    __syncthreads();
    const auto seq_of = [&](int s) {
        Seq q;
        if (s < kAtThreads) q.a = {s_span[s][0], s_span[s][1], s_span[s][2]};
        else q.a = span_of(p.starts, p.lengths, p.rows, s);
        q.work = 0;
        if (q.a.count > 0 && fits(c, q.a)) {
            const int rows = q.a.count * p.group;
            if (!WIDE && rows > kAtWideRows) return q;  // (the kernel for portions')
            q.cost = WIDE && rows > kAtWideRows ? 2 : 0;  // (all four warps work on it)
            const int per = q.cost ? S::kTile : RW;
            q.blocks = (q.a.pos + q.a.count - 1) / kKvBlock + 1;
            q.tiles = (rows + per - 1) / per;
            q.load = q.blocks + ((q.a.pos + q.a.count) % kKvBlock ? (q.cost ? kAtOpenWide : kAtOpenFew) : 0);
            q.work = (unsigned)(c.heads * q.tiles * q.load) << q.cost;
        }
        return q;
    };
    const int me = blockIdx.x, chunks = (c.seqs + kAtThreads - 1) / kAtThreads;
    // all the work, then the number of parts for every size: a lane takes one size and every fourth of its warp's sequences
    const int my_size = lane % kAtSizes;
    unsigned total = 0, share = 0, size = 0;
    bool each = false;  // a part for every CTA, at most
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        unsigned v = 0;
#pragma unroll 1
        for (int i = warp * (32 / kAtSizes) + lane / kAtSizes; i < c.seqs; i += kAtThreads / kAtSizes) {
            const Seq q = seq_of(i);
            if (pass == 1) {
                if (q.work) v += c.heads * q.tiles * ((((unsigned)q.load << q.cost) + size - 1) / size);
                continue;
            }
            v = add_work(v, q.work);
            if (q.work == 0 && q.a.count > 0 && !fits(c, q.a)) s_misfit = 1;
        }
#pragma unroll
        for (int o = kAtSizes; o < 32; o <<= 1) v = add_work(v, __shfl_xor_sync(0xffffffffu, v, o));
        __syncthreads();
        if (lane < kAtSizes) s_scan[warp][lane] = v;
        __syncthreads();
        v = add_work(add_work(s_scan[0][my_size], s_scan[1][my_size]), add_work(s_scan[2][my_size], s_scan[3][my_size]));
        if (pass == 0) {
            total = v;
            if (total >> 31) {
                if (me == 0 && tid == 0) say_not_taken(c.status, kAtTooMuch);
                return;
            }
            share = total / p.ctas + 1;
            size = max((unsigned)kAtWarps, share + (unsigned)((unsigned long long)share * my_size / kAtSizes));
        } else {
            const unsigned fits_in = __ballot_sync(0xffffffffu, v <= (unsigned)p.ctas);
            each = fits_in != 0;
            size = __shfl_sync(0xffffffffu, size, each ? __ffs(fits_in) - 1 : 0);
            if (!each) size = (share + 7) / 8 * 8;  // (parts of a cut tile are half of it at least, which their places in p.part go by)
        }
    }
    if (s_misfit) {  // rows that have no room: zeros, by all CTAs
        if (me == 0 && tid == 0) say_not_taken(c.status, 7);
#pragma unroll 1
        for (int i = 0; i < c.seqs; ++i) {
            const Span a = span_of(p.starts, p.lengths, p.rows, i);
            if (fits(c, a)) continue;
            const size_t n = (size_t)a.count * p.q_heads * hd;
            float* to = p.out + (size_t)a.row * p.q_heads * hd;
#pragma unroll 1
            for (size_t j = (size_t)me * kAtThreads + tid; j < n; j += (size_t)p.ctas * kAtThreads) to[j] = 0.f;
        }
    }
    const auto parts_of = [&](const Seq& q) { return (int)((((unsigned)q.load << q.cost) + size - 1) / size); };  // of a tile
    // the sequence in which this CTA's first part lies, counted in parts (each) or in work
    const unsigned at = each ? me : (unsigned)((unsigned long long)total * me / p.ctas);
    const unsigned stop = each ? me + 1 : (unsigned)((unsigned long long)total * (me + 1) / p.ctas);
    if (tid == 0) s_seq = -1;
    unsigned before = 0;
#pragma unroll 1
    for (int k = 0; k < chunks; ++k) {
        const int i = k * kAtThreads + tid;
        unsigned mine = 0;
        if (i < c.seqs) {
            const Seq q = seq_of(i);
            if (q.work) mine = each ? c.heads * q.tiles * parts_of(q) : q.work;
        }
        unsigned sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp][0] = sum;
        __syncthreads();
        unsigned all = 0;
#pragma unroll
        for (int w = 0; w < kAtWarps; ++w) {
            if (w < warp) sum += s_scan[w][0];
            all += s_scan[w][0];
        }
        sum += before;
        before += all;
        if (mine > 0 && at >= sum - mine && at < sum) {
            s_seq = i;
            s_at = sum - mine;
        }
    }
    __syncthreads();
    int s = s_seq;
    if (s < 0 || at >= stop) return;
    unsigned first = s_at;  // parts or work in front of sequence s
    int part_at = -1;       // the part of that sequence, once it is known

#pragma unroll 1
    while (s < c.seqs) {
        const Seq sq = seq_of(s);
        const int blocks = sq.blocks, cuts = sq.work ? parts_of(sq) : 1;
        const unsigned unit_work = (unsigned)sq.load << sq.cost;
        // the load from which on it is a part's, and its block: the last part has the open block, whatever its load
        const auto load_at = [&](int cut) { return (int)((unsigned)sq.load * cut / cuts); };
        const auto block_at = [&](int cut) { return cut == cuts ? blocks : min(load_at(cut), blocks - 1); };
        const auto work_at = [&](int part) { return (unsigned)(part / cuts) * unit_work + ((unsigned)load_at(part % cuts) << sq.cost); };
        if (sq.work && part_at < 0) {
            part_at = each ? at - first : max(0, (int)((at - first) / unit_work) * cuts);
#pragma unroll 1
            while (!each && first + work_at(part_at) < at) ++part_at;
        }
        if (sq.work == 0 || part_at >= c.heads * sq.tiles * cuts) {
            if (each) break;
            first += sq.work;
            ++s;
            part_at = 0;
            continue;
        }
        if (!each && first + work_at(part_at) >= stop) break;
        const Span& a = sq.a;
        const bool wide = WIDE && sq.cost != 0;
        const int unit = part_at / cuts, cut = part_at - unit * cuts;
        const int b0 = block_at(cut), b1 = block_at(cut + 1);
        // this part's place among the partial results, and the first one's of its tile
        const auto place_of = [&](int k) { return each ? me - cut + k : (int)(2ull * (first + work_at(unit * cuts + k)) / size); };
        ++part_at;
        const int h = unit / sq.tiles, r0 = (unit - h * sq.tiles) * (wide ? S::kTile : RW);
        const int nr = min(wide ? S::kTile : RW, a.count * p.group - r0);  // rows i = token * group + head
        const int closed = (a.pos + a.count) / kKvBlock;                   // whole blocks
        const int token0 = r0 / p.group, head0 = r0 - token0 * p.group;
        const auto token_of = [&](int r) { return token0 + (p.group_inv ? (int)__umulhi((unsigned)(head0 + r), p.group_inv) : r); };
        const auto pos_of = [&](int r) { return a.pos + token_of(r); };
        // a row of queries or of the result: its first value, rows `ld` apart
        const auto row_at = [&](int r, long long ld) {
            const int token = token_of(r);
            return (size_t)(a.row + token) * ld + (size_t)(h * p.group + r0 + r - token * p.group) * hd;
        };
        const bool q_wide = ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)p.ldq * 4 | (uintptr_t)hd * 4) & 15) == 0;
        // `n` rows of queries from the tile's row r on, zeros behind their ends, by threads from, from + step, ...: a group of copies
        const auto stage_queries = [&](float* to, int ld, int r, int n, int from, int step) {
#pragma unroll 1
            for (int i = from; i < n * D4; i += step) {
                const int k = i / D4, d = (i - k * D4) * 4;
                float* dst = to + k * ld + d;
                const float* src = p.q + row_at(r + k, p.ldq) + d;
                if (q_wide && d < hd) {
                    copy16(dst, src);
                } else {
#pragma unroll 1
                    for (int e = 0; e < 4; ++e) dst[e] = d + e < hd ? __ldg(src + e) : 0.f;
                }
            }
            copies_commit();
        };
        const size_t head = c.head_of(s, h) * c.blocks;
        const int bend = min(min(b1, closed), pos_of(nr - 1) / kKvBlock + 1);
        const bool open = b1 == blocks && closed < blocks && pos_of(nr - 1) >= closed * kKvBlock;
        const int n_open = open ? a.pos + a.count - closed * kKvBlock : 0;

        {
            // ---- copies on their way ----
            const int vbytes = kKvBlock * c.dim_v;
            const auto copy_block = [&](uint8_t* to, bool values, int b, int from, int step) {
                const int bytes = values ? vbytes : S::kSlot;
                const uint8_t* src = (values ? c.v : c.k) + (head + b) * bytes;
#pragma unroll 4
                for (int i = from * 16; i < bytes; i += step * 16) copy16(to + i, src + i);
            };
            uint8_t* mine_ring = ring + warp * RING * S::kSlot;
            const int bstep = wide ? 1 : kAtWarps, bfirst = wide ? b0 : b0 + warp;
            // split: keys, values, keys, ... of this warp's blocks into its slots; wide: a block into the next two of all
            int ask_b = bfirst, ask_slot = 0;
            bool ask_v = false;
            const auto ask = [&]() {
                if (ask_b < bend) {
                    if (wide) copy_block(ring + ask_slot * S::kSlot, false, ask_b, tid, kAtThreads);
                    copy_block(wide ? ring + (ask_slot + 1) * S::kSlot : mine_ring + ask_slot * S::kSlot, wide || ask_v, ask_b, wide ? tid : lane, wide ? kAtThreads : 32);
                }
                copies_commit();
                if (wide || ask_v) ask_b += bstep;
                ask_v = !ask_v;
                ask_slot += wide ? 2 : 1;
                if (ask_slot == (wide ? S::kSlots : RING)) ask_slot = 0;
            };
            const int row0 = wide ? warp * RW : 0;  // this warp's rows in the tile
            // ---- query rows as digits ----
            uint32_t qd[3][NK][2 * SETS];
            float cr[SETS];
            int see[SETS];  // the row's last position, -1: no row
            float o[SETS][NT][2], m[SETS], l[SETS];
            float4 f[SETS][2 * NK];  // (asked for in front of the ring's copies, which keep the memory busy for microseconds)
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                const int r = g + 8 * z;
                const bool is = row0 + r < nr;
                see[z] = is ? pos_of(row0 + r) : -1;
                const float* src = p.q + row_at(is ? row0 + r : 0, p.ldq);
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) {
                    const int d = (i >> 2) * 64 + ((NK & 1) && i >= 2 * NK - 2 ? 8 * t + 4 * (i & 1) : 16 * t + 4 * (i & 3));
                    f[z][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (is && d < hd) {
                        if (q_wide) {
                            f[z][i] = __ldg(reinterpret_cast<const float4*>(src + d));
                        } else {
                            f[z][i].x = __ldg(src + d);
                            if (d + 1 < hd) f[z][i].y = __ldg(src + d + 1);
                            if (d + 2 < hd) f[z][i].z = __ldg(src + d + 2);
                            if (d + 3 < hd) f[z][i].w = __ldg(src + d + 3);
                        }
                    }
                }
            }
            __syncthreads();                        // (the ring is free)
#pragma unroll 1
            for (int i = 0; i < (wide ? STAGES - 1 : RING); ++i) ask();
            if (open)
#pragma unroll 1
                for (int i = tid; i * 32 < n_open * c.dim_o; i += kAtThreads) {
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(c.open_row(c.k_open, s, h, closed * kKvBlock) + i * 32));
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(c.open_row(c.v_open, s, h, closed * kKvBlock) + i * 32));
                }

#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                float top = 0.f, odd = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) {
                    top = fmaxf(fmaxf(fmaxf(top, fabsf(f[z][i].x)), fmaxf(fabsf(f[z][i].y), fabsf(f[z][i].z))), fabsf(f[z][i].w));
                    odd += (f[z][i].x + f[z][i].y) * 0.f + (f[z][i].z + f[z][i].w) * 0.f;  // (not a number, from one or an infinity)
                }
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    odd += __shfl_xor_sync(0xffffffffu, odd, x);
                }
                // two factors: one alone would overflow for the smallest rows
                const float half_mul = top > 0.f ? exp2f(-floorf(log2f(top))) : 1.f, mul = __fdiv_rn(kQueryMax, top > 0.f ? top * half_mul : 1.f);
                cr[z] = p.scale * top * 256.f / (kQueryMax * 127.f);
                m[z] = -CUDART_INF_F;
                l[z] = odd;  // 0, or not a number
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) {
                    const float e4[4] = {f[z][i].x, f[z][i].y, f[z][i].z, f[z][i].w};
                    uint32_t digits[4], w[3];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // v = d0 + 256 d1 + 65536 d2 with bytes of either sign: each but the last takes what it is over 127 into the next
                        const int v = __float2int_rn(e4[e] * half_mul * mul);
                        digits[e] = (uint32_t)(v + 0x8080) ^ 0x8080u;
                    }
                    digit_words(digits[0], digits[1], digits[2], digits[3], w);
#pragma unroll
                    for (int k = 0; k < 3; ++k) qd[k][i >> 1][2 * z + (i & 1)] = w[k];
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) o[z][n][0] = o[z][n][1] = 0.f;
            }
            const int first_seen = pos_of(min(row0, nr - 1));
            const int warp_last = row0 < nr ? pos_of(min(row0 + RW, nr) - 1) : -1;

            // ---- block by block: scores and their weights, then the weighted values ----
            const auto hi = [](const auto& x, int i) -> uint32_t { return SETS == 2 ? x[SETS == 2 ? i : 0] : 0u; };
            float kt = 0.f, vt = 0.f;
            if (bfirst < bend) {
                kt = __ldg(c.k_top + head + bfirst);
                vt = __ldg(c.v_top + head + bfirst);
            }
            int slot_at = 0;
#pragma unroll 1
            for (int b = bfirst; b < bend; b += bstep) {
                float kt1 = 0.f, vt1 = 0.f;
                if (b + bstep < bend) {
                    kt1 = __ldg(c.k_top + head + b + bstep);
                    vt1 = __ldg(c.v_top + head + b + bstep);
                }
                const uint8_t *kb, *vb;
                if (wide) {
                    copies_wait<STAGES - 2>();
                    __syncthreads();  // block b is there, and nobody reads block b - 1 any more
                    ask();
                    kb = ring + slot_at * S::kSlot;
                    vb = kb + S::kSlot;
                    slot_at = slot_at == S::kSlots - 2 ? 0 : slot_at + 2;
                } else {
                    copies_wait<RING - 1>();
                    __syncwarp();
                    kb = mine_ring + slot_at * S::kSlot;
                    slot_at = slot_at == RING - 1 ? 0 : slot_at + 1;
                    vb = mine_ring + slot_at * S::kSlot;
                    slot_at = slot_at == RING - 1 ? 0 : slot_at + 1;
                }
                const bool works = warp_last >= b * kKvBlock;
                uint32_t pd[3][2][2 * SETS];  // [digit][k step][a0, a2 of rows g, then of rows g + 8]
                float mul[SETS];
                if (works) {
                    float sc[SETS][8][2];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        int d[3][4];
                        sums_begin(d);
                        const uint8_t* kj = kb + j * (256 * NK);
#pragma unroll
                        for (int ch = 0; ch < NK / 2; ++ch) {
                            const uint4 f = *reinterpret_cast<const uint4*>(kj + ch * 512 + lane * 16);
#pragma unroll
                            for (int k = 0; k < 3; ++k) {
                                mma_s8(d[k], qd[k][2 * ch][0], hi(qd[k][2 * ch], 2), qd[k][2 * ch][1], hi(qd[k][2 * ch], 3), f.x, f.y);
                                mma_s8(d[k], qd[k][2 * ch + 1][0], hi(qd[k][2 * ch + 1], 2), qd[k][2 * ch + 1][1], hi(qd[k][2 * ch + 1], 3), f.z, f.w);
                            }
                        }
                        if (NK & 1) {
                            const uint2 f = *reinterpret_cast<const uint2*>(kj + (NK / 2) * 512 + lane * 8);
#pragma unroll
                            for (int k = 0; k < 3; ++k) mma_s8(d[k], qd[k][NK - 1][0], hi(qd[k][NK - 1], 2), qd[k][NK - 1][1], hi(qd[k][NK - 1], 3), f.x, f.y);
                        }
#pragma unroll
                        for (int z = 0; z < SETS; ++z)
#pragma unroll
                            for (int e = 0; e < 2; ++e) sc[z][j][e] = digits_sum(d[0][2 * z + e], d[1][2 * z + e], d[2][2 * z + e]);
                    }
                    const bool edge = (b + 1) * kKvBlock - 1 > first_seen;
                    bool same = true;
                    float old[SETS];
#pragma unroll
                    for (int z = 0; z < SETS; ++z) {
                        const float cs = cr[z] * kt;
                        float mb = -CUDART_INF_F;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                sc[z][j][e] *= cs;
                                if (edge && b * kKvBlock + 8 * j + 2 * t + e > see[z]) sc[z][j][e] = -CUDART_INF_F;
                                mb = fmaxf(mb, sc[z][j][e]);
                            }
                        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
                        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
                        const bool any = see[z] >= b * kKvBlock;  // the row sees a part of the block
                        const float wm = any ? kWeightMax : 0.f;
                        uint32_t sum = 0;
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                uint32_t q4[4], w[3];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    q4[e] = __float2uint_rn(exp2_of(sc[z][4 * ks + 2 * half + (e >> 1)][e & 1] - mb) * wm);
                                    sum += q4[e];
                                }
                                digit_words(q4[0], q4[1], q4[2], q4[3], w);
#pragma unroll
                                for (int k = 0; k < 3; ++k) pd[k][ks][2 * z + half] = w[k];
                            }
                        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                        mul[z] = 0.f;
                        old[z] = 1.f;
                        if (any) {
                            const float mn = fmaxf(m[z], mb);
                            old[z] = m[z] == mn ? 1.f : exp2_of(m[z] - mn);
                            const float now = exp2_of(mb - mn) * (1.f / kWeightMax);
                            l[z] = fmaf(l[z], old[z], (float)sum * now);
                            if (!(fabsf(kt) <= CUDART_MAX_NORMAL_F)) l[z] = CUDART_NAN_F;
                            m[z] = mn;
                            mul[z] = now * (256.f / 127.f) * vt;
                            same = same && old[z] == 1.f;
                        }
                    }
                    if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                        for (int z = 0; z < SETS; ++z)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                o[z][n][0] *= old[z];
                                o[z][n][1] *= old[z];
                            }
                    }
                }
                if (!wide) {
                    __syncwarp();
                    ask();
                    copies_wait<RING - 1>();
                    __syncwarp();
                }
                if (works) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (8 * n >= hd) break;
                        const uint4 f = *reinterpret_cast<const uint4*>(vb + n * 512 + lane * 16);
                        int d[3][4];
                        sums_begin(d);
#pragma unroll
                        for (int k = 0; k < 3; ++k) {
                            mma_u8s8(d[k], pd[k][0][0], hi(pd[k][0], 2), pd[k][0][1], hi(pd[k][0], 3), f.x, f.y);
                            mma_u8s8(d[k], pd[k][1][0], hi(pd[k][1], 2), pd[k][1][1], hi(pd[k][1], 3), f.z, f.w);
                        }
#pragma unroll
                        for (int z = 0; z < SETS; ++z)
                            if (see[z] >= b * kKvBlock) {  // (a scale that is not a number must not meet rows that do not see the block)
#pragma unroll
                                for (int e = 0; e < 2; ++e) o[z][n][e] = fmaf(digits_sum(d[0][2 * z + e], d[1][2 * z + e], d[2][2 * z + e]), mul[z], o[z][n][e]);
                            }
                    }
                }
                if (!wide) {
                    __syncwarp();
                    ask();
                }
                kt = kt1;
                vt = vt1;
            }
            copies_wait<0>();
            __syncthreads();  // the ring is free: partial results take its place

#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                const int r = g + 8 * z;
                float* to = pieces + (size_t)(warp * RW + r) * LD + 2 * t;
#pragma unroll
                for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(to + 8 * n) = make_float2(o[z][n][0], o[z][n][1]);
                if (t == 0) {
                    s_m[wide ? 0 : warp][row0 + r] = m[z];
                    s_l[wide ? 0 : warp][row0 + r] = l[z];
                }
            }

            // ---- the open block: float32 rows, plain multiply-adds, 16 rows at a time, into the first piece ----
            if (open) {
                const float* ko = c.open_row(c.k_open, s, h, closed * kKvBlock);
                const float* vo = c.open_row(c.v_open, s, h, closed * kKvBlock);
                const int o4 = c.dim_o / 4, half = kKvBlock / 2;
                const auto bring = [&](float* to, int ld, const float* from, int n) {  // rows, by warps
#pragma unroll 1
                    for (int j = warp; j < n; j += kAtWarps)
#pragma unroll 1
                        for (int d = lane; d < o4; d += 32) copy16(to + j * ld + d * 4, from + (size_t)j * c.dim_o + d * 4);
                    copies_commit();
                };
#pragma unroll 1
                for (int g0 = 0; g0 < nr; g0 += kAtOpenRows) {
                    const int gn = min(kAtOpenRows, nr - g0);
                    __syncthreads();
                    stage_queries(open_q, LD, g0, gn, tid, kAtThreads);
                    bring(open_k, S::kLdOpen, ko, min(n_open, half));
                    bring(open_v, c.dim_o, vo, min(n_open, half));
#pragma unroll 1
                    for (int j0 = warp * 8; j0 - warp * 8 < n_open; j0 += half) {  // a lane: a position (g) and every fourth four dimensions
                        if (j0 >= half) {
                            __syncthreads();
                            bring(open_k, S::kLdOpen, ko + (size_t)half * c.dim_o, n_open - half);
                            copies_wait<0>();
                        } else {
                            copies_wait<1>();
                        }
                        __syncthreads();
                        const float* row = open_k + (j0 % half + g) * S::kLdOpen + 4 * t;  // (rows past the last: whatever is there)
#pragma unroll 1
                        for (int r = 0; r < gn; r += 4) {
                            float dot[4] = {};
#pragma unroll
                            for (int i = 0; i < 2 * NK; ++i) {
                                if (16 * i + 4 * t >= c.dim_o) break;
                                const float4 f = *reinterpret_cast<const float4*>(row + 16 * i);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {  // (rows past gn: whatever is there)
                                    const float4 q = *reinterpret_cast<const float4*>(open_q + (r + e) * LD + 16 * i + 4 * t);
                                    dot[e] = fmaf(q.x, f.x, fmaf(q.y, f.y, fmaf(q.z, f.z, fmaf(q.w, f.w, dot[e]))));
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                dot[e] += __shfl_xor_sync(0xffffffffu, dot[e], 1);
                                dot[e] += __shfl_xor_sync(0xffffffffu, dot[e], 2);
                            }
                            const float mine = t == 0 ? dot[0] : t == 1 ? dot[1] : t == 2 ? dot[2] : dot[3];
                            if (j0 + g < n_open) open_w[(j0 + g) * kAtOpenRows + r + t] = mine * p.scale;
                        }
                    }
                    __syncthreads();
                    if (n_open > half) bring(open_k, c.dim_o, vo + (size_t)half * c.dim_o, n_open - half);
                    float* sm = s_m[0];
#pragma unroll 1
                    for (int r = warp; r < gn; r += kAtWarps) {
                        const int vis = min(n_open, pos_of(g0 + r) - closed * kKvBlock + 1);  // (0 or less: none)
                        const float s0 = lane < vis ? open_w[lane * kAtOpenRows + r] : -CUDART_INF_F;
                        const float s1 = lane + 32 < vis ? open_w[(lane + 32) * kAtOpenRows + r] : -CUDART_INF_F;
                        const float top = lb_warp_max(fmaxf(s0, s1));
                        const float w0 = lane < vis ? exp2_of(s0 - top) : 0.f, w1 = lane + 32 < vis ? exp2_of(s1 - top) : 0.f;
                        float sum = w0 + w1;
#pragma unroll
                        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                        open_w[lane * kAtOpenRows + r] = w0;
                        open_w[(lane + 32) * kAtOpenRows + r] = w1;
                        if (lane == 0) {  // the first piece's row and this one's on one scale
                            const float was = sm[g0 + r], both = fmaxf(was, top);
                            const float fp = was == -CUDART_INF_F ? 0.f : exp2_of(was - both), fo = vis > 0 ? exp2_of(top - both) : 0.f;
                            s_f[0][r] = fp;
                            s_f[1][r] = fo;
                            sm[g0 + r] = both;
                            s_l[0][g0 + r] = fmaf(s_l[0][g0 + r], fp, vis > 0 ? sum * fo : 0.f);
                        }
                    }
                    copies_wait<0>();
                    __syncthreads();
                    const int seen = min(n_open, pos_of(g0 + gn - 1) - closed * kKvBlock + 1);
                    const bool alike = pos_of(g0) == pos_of(g0 + gn - 1);
#pragma unroll 1
                    for (int d = tid; d < hd; d += kAtThreads) {
#pragma unroll 1
                        for (int r = 0; r < gn; r += 4) {
                            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                            for (int k = 0; k < 2; ++k) {
                                const float* from = (k ? open_k : open_v) + d;
                                const float* ws = open_w + k * half * kAtOpenRows + r;
                                const int n = min(seen - k * half, half);
                                if (alike) {
#pragma unroll 8
                                    for (int j = 0; j < n; ++j) {
                                        const float v = from[j * c.dim_o];
                                        const float4 w = *reinterpret_cast<const float4*>(ws + j * kAtOpenRows);
                                        sum = make_float4(fmaf(w.x, v, sum.x), fmaf(w.y, v, sum.y), fmaf(w.z, v, sum.z), fmaf(w.w, v, sum.w));
                                    }
                                } else {  // a row that does not see position j must not meet what is there
#pragma unroll 2
                                    for (int j = 0; j < n; ++j) {
                                        const float v = from[j * c.dim_o];
                                        const float4 w = *reinterpret_cast<const float4*>(ws + j * kAtOpenRows);
                                        sum.x = w.x != 0.f ? fmaf(w.x, v, sum.x) : sum.x;
                                        sum.y = w.y != 0.f ? fmaf(w.y, v, sum.y) : sum.y;
                                        sum.z = w.z != 0.f ? fmaf(w.z, v, sum.z) : sum.z;
                                        sum.w = w.w != 0.f ? fmaf(w.w, v, sum.w) : sum.w;
                                    }
                                }
                            }
                            const float e4[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (r + e < gn) {
                                    float& x = pieces[(g0 + r + e) * LD + d];
                                    const float fp = s_f[0][r + e], fo = s_f[1][r + e];
                                    x = fmaf(fp, x, fo != 0.f ? fo * e4[e] : 0.f);
                                }
                        }
                    }
                }
            }
            __syncthreads();

            // ---- the pieces into one, and out ----
            const bool o_wide = (hd & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
            const auto put = [&](int r, int d, float4 x, float sum) {
                const float inv = __fdiv_rn(1.f, sum);
                x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                float* to = p.out + row_at(r, (long long)p.q_heads * hd) + d;
                if (o_wide) {
                    *reinterpret_cast<float4*>(to) = x;
                } else {
                    to[0] = x.x;
                    if (d + 1 < hd) to[1] = x.y;
                    if (d + 2 < hd) to[2] = x.z;
                    if (d + 3 < hd) to[3] = x.w;
                }
            };
            const auto factor = [](float one, float top) { return one == -CUDART_INF_F ? 0.f : exp2_of(one - top); };
            const bool done = cuts == 1;
            const int d4s = (hd + 3) / 4, pieces_n = wide ? 1 : kAtWarps;
            const auto slot = [&](int k) { return p.part + (size_t)place_of(k) * S::kTile * p.part_ld; };
            float* part = slot(cut);
            if (tid < nr) {  // a row's largest score and sum, and factors in the place of the pieces' own
                float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll 1
                for (int w = 0; w < pieces_n; ++w) top = fmaxf(top, s_m[w][tid]);
#pragma unroll 1
                for (int w = 0; w < pieces_n; ++w) {
                    const float f = factor(s_m[w][tid], top);
                    sum = fmaf(s_l[w][tid], f, sum);
                    s_m[w][tid] = f;
                }
                s_l[0][tid] = sum;
                if (!done) __stcg(reinterpret_cast<float2*>(part + (size_t)tid * p.part_ld + 4 * d4s), make_float2(top, sum));
            }
            __syncthreads();
#pragma unroll 1
            for (int r = warp; r < nr; r += kAtWarps)
#pragma unroll 1
                for (int d = lane * 4; d < hd; d += 128) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                    for (int w = 0; w < pieces_n; ++w) {
                        const float f = s_m[w][r];
                        // (0 for a piece that has none of the row's positions: what stands there does not count)
                        if (f != 0.f) add_scaled(x, *reinterpret_cast<const float4*>(pieces + (w * RW + r) * LD + d), f);
                    }
                    if (done) put(r, d, x, s_l[0][r]);
                    else __stcg(reinterpret_cast<float4*>(part + (size_t)r * p.part_ld + d), x);
                }
            if (!done) {
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    unsigned* cnt = p.cnt + place_of(0);
                    s_last = atomicAdd(cnt, 1u) + 1 == (unsigned)cuts;
                    if (s_last) *cnt = 0;
                }
                __syncthreads();
                if (s_last) {
                    __threadfence();
                    lb_fence_proxy_async();  // (the other CTAs' ordinary stores, before copies that go another way)
                    // rows of the parts, some at a time, through shared memory, every copy in flight at once
                    const int ld = 4 * d4s + 4, room = (int)(S::kSmem / 4) - kAtWarps * 4;
                    const int per = min(nr, max(1, room / (cuts * (ld + 1))));           // rows of a round
                    const int fit = min(cuts, room / (per * (ld + 1)));                  // parts of a round: all of them, if one row's fit
                    float* got = pieces;                  // [fit][per][ld]
                    float* fs = got + fit * per * ld;     // [fit][per] factors
#pragma unroll 1
                    for (int g0 = 0; g0 < nr; g0 += per) {
                        const int gn = min(per, nr - g0), row4 = gn * (ld / 4);
                        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);  // (of the one row of a round, where the parts come in several)
                        float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll 1
                        for (int q0 = 0; q0 < cuts; q0 += fit) {
                            const int qn = min(fit, cuts - q0);
                            lb_fence_proxy_async();  // (what stood there was read and written by ordinary accesses)
                            __syncthreads();
                            if (warp == 0) {
                                if (lane == 0) lb_mbar_expect_tx(&s_bar, (uint32_t)qn * row4 * 16);
                                __syncwarp();
                                for (int q = lane; q < qn; q += 32) lb_bulk_g2s(got + q * row4 * 4, slot(q0 + q) + (size_t)g0 * ld, row4 * 16, &s_bar);
                            }
                            if (!lb_mbar_wait_bounded(&s_bar, bar_phase)) atomicExch(c.status, 1);
                            bar_phase ^= 1;
                            __syncthreads();
                            const float was = top;
#pragma unroll 1
                            for (int r = fit < cuts ? 0 : warp; r < gn; r += kAtWarps) {  // (the one row of several rounds: every warp)
                                const auto stat = [&](int q, int k) { return got[(q * gn + r) * ld + 4 * d4s + k]; };
                                float now = was, more = 0.f;
#pragma unroll 1
                                for (int q = lane; q < qn; q += 32) now = fmaxf(now, stat(q, 0));
                                now = lb_warp_max(now);
#pragma unroll 1
                                for (int q = lane; q < qn; q += 32) {
                                    const float f = factor(stat(q, 0), now);
                                    more = fmaf(stat(q, 1), f, more);
                                    fs[q * gn + r] = f;
                                }
#pragma unroll
                                for (int x = 16; x > 0; x >>= 1) more += __shfl_xor_sync(0xffffffffu, more, x);
                                if (fit < cuts) {
                                    const float f0 = factor(was, now);
                                    sum = fmaf(sum, f0, more);
                                    y = make_float4(y.x * f0, y.y * f0, y.z * f0, y.w * f0);
                                    top = now;
                                } else if (lane == 0) {
                                    s_l[0][r] = more;
                                }
                            }
                            __syncthreads();
                            if (fit < cuts) {  // (a row has 64 groups of four dimensions at most: every thread has one, or none)
                                if (tid < d4s)
#pragma unroll 4
                                    for (int q = 0; q < qn; ++q)
                                        if (const float f = fs[q]) add_scaled(y, *reinterpret_cast<const float4*>(got + q * ld + tid * 4), f);
                            } else {
#pragma unroll 1
                                for (int r = warp; r < gn; r += kAtWarps)
#pragma unroll 1
                                    for (int d = lane * 4; d < hd; d += 128) {
                                        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                                        for (int q = 0; q < qn; ++q)
                                            if (const float f = fs[q * gn + r]) add_scaled(x, *reinterpret_cast<const float4*>(got + (q * gn + r) * ld + d), f);
                                        put(g0 + r, d, x, s_l[0][r]);
                                    }
                            }
                        }
                        if (fit < cuts && tid < d4s) put(g0, tid * 4, y, sum);
                    }
                }
                __syncthreads();
            }
        }
        if (each) break;
    }
}


#include "kv8_rows.cuh"

Kv8 view(const loom_b200_kv8* c) {
    return {c->seqs, c->max_len, c->heads, c->dim, c->blocks, c->dim_k, c->dim_v, c->dim_o, c->k, c->v, c->k_top, c->v_top, c->k_open, c->v_open, c->placed, c->ctx->status_dev};
}

}  // namespace

template <typename P>
static cudaError_t launch_pdl(loom_b200_ctx* ctx, void (*kern)(P), dim3 grid, int threads, size_t smem, const P& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->opt_pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

constexpr int kAtMostCtasPerSm = 2;

template <int NK, int SETS, bool WIDE>
static int launch_attend(loom_b200_ctx* ctx, AttendParams p) {
    using S = AttendShape<NK, SETS>;
    p.ctas = ctx->sm_count * S::kPerSm;
    static_assert(S::kPerSm * (S::kSmem + 6 * 1024) <= 228 * 1024, "shared memory of an SM");
    p.part = (float*)((uint8_t*)p.cnt + (2 * (size_t)ctx->sm_count * kAtMostCtasPerSm + 1) * 4 / 16 * 16 + 16);
    const size_t smem = S::kSmem;
    LB_CUDA(ctx, cudaFuncSetAttribute(lb_kv8_attend_kernel<NK, SETS, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    LB_CUDA(ctx, launch_pdl(ctx, lb_kv8_attend_kernel<NK, SETS, WIDE>, dim3(p.ctas), kAtThreads, smem, p));
    ctx->launches++;
    return 0;
}

// (without the code for wide tiles one token's attention is 5 % faster)
template <int NK>
static int launch_few(loom_b200_ctx* ctx, const AttendParams& p, bool few, bool wide) {
    if (wide) return few ? launch_attend<NK, 1, true>(ctx, p) : launch_attend<NK, 2, true>(ctx, p);
    return few ? launch_attend<NK, 1, false>(ctx, p) : launch_attend<NK, 2, false>(ctx, p);
}

template <int NK>
static int launch_rows(loom_b200_ctx* ctx, AttendParams p) {
    using S = RowsShape<NK>;
    p.ctas = 2 * ctx->sm_count;
    p.part = (float*)((uint8_t*)p.cnt + (2 * (size_t)ctx->sm_count * kAtMostCtasPerSm + 1) * 4 / 16 * 16 + 16);
    LB_CUDA(ctx, cudaFuncSetAttribute(lb_kv8_rows_kernel<NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
    LB_CUDA(ctx, launch_pdl(ctx, lb_kv8_rows_kernel<NK>, dim3(p.ctas), kRwThreads, S::kSmem, p));
    ctx->launches++;
    return 0;
}

constexpr int kKvMaxSeqs = 4096;
constexpr int kKvMaxLen = 1 << 29;  // (a tile's load times its parts, of which there are no more than CTAs, in 32 bits)

extern "C" {

int loom_b200_kv8_create(loom_b200_ctx* ctx, int sequences, int max_len, int kv_heads, int head_dim, loom_b200_kv8** out) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "kv8_create: ctx is NULL");
    LB_REQUIRE(ctx, out != nullptr, "kv8_create: out is NULL");
    *out = nullptr;
    LB_REQUIRE(ctx, sequences > 0 && max_len > 0 && kv_heads > 0 && head_dim > 0, "kv8_create: %d sequences of %d positions, %d KV heads of %d", sequences, max_len, kv_heads, head_dim);
    if (sequences > kKvMaxSeqs || kv_heads > 65535 || head_dim > 256 || max_len > kKvMaxLen)
        return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "kv8_create: %d sequences (%d at most), %d positions (%d at most), %d KV heads of %d (256 at most)", sequences, kKvMaxSeqs, max_len, kKvMaxLen, kv_heads, head_dim);
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
    c->dim_o = (head_dim + 3) / 4 * 4;
    const size_t blocks = (size_t)sequences * kv_heads * c->blocks, open = (size_t)sequences * kv_heads * 2 * kKvBlock * c->dim_o * 4;
    const size_t ctas = (size_t)ctx->sm_count * kAtMostCtasPerSm;
    // counters, then parts: a few rows' of every CTA, or the tiles' of a portion
    const size_t dims = (head_dim + 31) / 32 * 32, few = (head_dim > 128 ? AttendShape<8, 1>::kTile : AttendShape<4, 2>::kTile) * (size_t)(c->dim_o + 4), many = head_dim > 128 ? 0 : kRwTile * (dims + 2);
    c->work_bytes = (2 * ctas + 1) * 4 + 32 + (2 * ctas + 1) * (few > many ? few : many) * 4;
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
    get((void**)&c->placed, (size_t)sequences * kv_heads * 4 * sizeof(int));
    get(&c->work, c->work_bytes);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->placed, 0xff, (size_t)sequences * kv_heads * 4 * sizeof(int), ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->work, 0, c->work_bytes, ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->k_open, 0, open, ctx->stream);  // (what rounds a row's dimensions up stays zero)
    if (e == cudaSuccess) e = cudaMemsetAsync(c->v_open, 0, open, ctx->stream);
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
    void* ptrs[] = {c->k, c->v, c->k_top, c->v_top, c->k_open, c->v_open, c->placed, c->work};
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

// a CTA for each item, as far as the blocks can be bounded here: a sequence's rows touch one more than their 64s, and at most one each
static dim3 row_grid(const RowParams& p) {
    long long blocks = p.rows;
    if (p.starts && blocks > (p.rows + 62LL * p.c.seqs) / kKvBlock + p.c.seqs) blocks = (p.rows + 62LL * p.c.seqs) / kKvBlock + p.c.seqs;
    if (blocks > 32768) blocks = 32768;
    return dim3(2 * p.c.heads, (unsigned)blocks);
}

int loom_b200_kv8_append(loom_b200_ctx* ctx, loom_b200_kv8* c, int rows, const int32_t* starts, const int32_t* lengths, const float* k, const float* v, long long ld) {
    if (int rc = kv8_ready(ctx, c, rows, starts, lengths, k, v, "kv8_append")) return rc;
    LB_REQUIRE(ctx, ld >= (long long)c->heads * c->dim, "kv8_append: %lld floats between rows of %d", ld, c->heads * c->dim);
    if (int rc = lb_set_device(ctx)) return rc;
    const bool wide = c->dim % 4 == 0 && ld % 4 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    const RowParams p{view(c), rows, starts, lengths, k, v, ld, nullptr, nullptr, wide};
    const dim3 grid = row_grid(p);
    LB_CUDA(ctx, launch_pdl(ctx, c->dim > 128 ? lb_kv8_append_kernel<2> : lb_kv8_append_kernel<1>, grid, kRowThreads, 0, p));
    ctx->launches++;
    return 0;
}

int loom_b200_kv8_read(loom_b200_ctx* ctx, loom_b200_kv8* c, int rows, const int32_t* starts, const int32_t* lengths, float* k, float* v) {
    if (int rc = kv8_ready(ctx, c, rows, starts, lengths, k, v, "kv8_read")) return rc;
    if (int rc = lb_set_device(ctx)) return rc;
    const bool wide = c->dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    const RowParams p{view(c), rows, starts, lengths, nullptr, nullptr, 0, k, v, wide};
    const dim3 grid = row_grid(p);
    LB_CUDA(ctx, launch_pdl(ctx, lb_kv8_read_kernel, grid, kRowThreads, 0, p));
    ctx->launches++;
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
    if (p.group > 32768) return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "kv8_attend: %d query heads a KV head, 32768 at most", p.group);
    p.group_inv = p.group > 1 ? (unsigned)((4294967296ull + p.group - 1) / p.group) : 0u;
    // the list of work is counted in 31 bits: blocks of tiles of eight rows, as if every sequence were full and had an open block
    if ((double)c->heads * (c->blocks + 1 + kAtOpenFew) * ((double)rows * p.group / 8 + 8.0 * c->seqs) >= kAtMostWork)
        return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "kv8_attend: %d rows of %d heads over sequences of up to %d positions: fewer rows a call", rows, heads, c->max_len);
    // and so are a portion's tiles, should every sequence have every row
    if ((double)c->heads * c->seqs * ((double)rows * p.group / kRwTile + 1) >= kAtMostWork)
        return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "kv8_attend: %d rows of %d heads for %d sequences: fewer rows a call", rows, heads, c->seqs);
    if (int rc = lb_set_device(ctx)) return rc;
    p.starts = starts;
    p.lengths = lengths;
    p.q = q;
    p.ldq = ldq;
    p.out = out;
    p.scale = (float)((scale > 0 ? scale : 1.0 / sqrt((double)c->dim)) * 1.4426950408889634);
    p.cnt = (unsigned*)c->work;
    p.part_ld = (c->dim + 3) / 4 * 4 + 4;
    // tiles of eight rows a warp where sequences have no more on the average (any number is right with either)
    const bool few = (long long)rows * p.group <= 8LL * (starts ? c->seqs : rows);
    // Sequences of many rows go to the kernel for portions, where the call has more than two rows a sequence on the average, or more than 256 rows
    // of a KV head's group: which sequences have them is on the device, and a cache may have many that take no part.  13 to 512 rows of 4 heads at
    // 2900: 43 to 83 us instead of 125 to 238; 200 rows of one of 256 sequences 71 instead of 118, 512 of them 97 instead of 351.  Its launch where there are
    // none takes up to 5 us: 16 sequences of one row 41.6 us instead of 36.4, 128 of one at 1000 97 instead of 91.
    const int nk = c->dim_k / 32;
    const long long group_rows = (long long)rows * p.group;
    const bool portions = nk <= kAtRowsNk && (starts ? group_rows > kAtWideRows && (rows > 2 * c->seqs || group_rows > kAtPortionRows) : p.group > kAtWideRows);
    const bool wide = !portions && (long long)(starts ? rows : 1) * p.group > kAtWideRows;
    int rc = 0;
    switch (nk) {
        case 1: rc = launch_few<1>(ctx, p, few, wide); break;
        case 2: rc = launch_few<2>(ctx, p, few, wide); break;
        case 3: rc = launch_few<3>(ctx, p, few, wide); break;
        case 4: rc = launch_few<4>(ctx, p, few, wide); break;
        case 5: rc = launch_attend<5, 1, true>(ctx, p); break;
        case 6: rc = launch_attend<6, 1, true>(ctx, p); break;
        case 7: rc = launch_attend<7, 1, true>(ctx, p); break;
        default: rc = launch_attend<8, 1, true>(ctx, p);
    }
    if (rc || !portions) return rc;
    return nk == 1 ? launch_rows<1>(ctx, p) : nk == 2 ? launch_rows<2>(ctx, p) : nk == 3 ? launch_rows<3>(ctx, p) : launch_rows<4>(ctx, p);
}

}  // extern "C"
