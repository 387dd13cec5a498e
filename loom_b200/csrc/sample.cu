// sample.cu -- the next token of every sequence from its row of logits: temperature, top-k, top-p and min-p, with random numbers that the
// caller gives.
//
// Definition, for a row l of `vocab` logits, temperature T, and m its largest value:
//   weight   w_i = exp((l_i - m) / T); not-a-numbers count as minus infinity, which has weight 0; where m is plus infinity those have weight 1
//            and all others 0
//   order    larger logit first, equal ones by index
//   kept     the first k of the order; of those the shortest run from the front whose weight is at least p times theirs (one token at
//            least); of those the ones with w_i >= min_p (above 1: as 1)
//   token    the first kept one, by index, whose weight and that of the kept ones in front of it exceed u times the kept weight
// T <= 0 is the first largest logit.  Weights are integers, round(w 2^S) with S such that a whole row's sum stays below 2^62: sums do not
// depend on their order then.  They are within vocab * 2^-S of the largest weight (S = 44 for 128,256 tokens: 7e-9) and 2^-32 of themselves of the
// real ones, the latter from the weights beyond four temperatures.
//
// One cluster of CTAs per row, each with a slice of the row in shared memory, so the row is read once and by one launch.  What is kept
// ends at a place in the order, a (logit, index) pair.  A place is found from a histogram -- of counts for top-k, of weights for
// top-p -- over linear bins of m - l: the values of the bin that the limit falls into are few, and are put in order by another one, down to
// what a handful of comparisons settles.  Three ways there, the cheapest that holds:
//   few     values that no kept one is below are gathered in the first CTA, which does the rest by itself while the others' places are
//           free for the next rows.  top-k: with G >= k groups of tokens, at least k values reach the smallest of the groups' largest
//           ones, of values in random order about G ln G do (270 for k up to 64); min-p: the values not below it; small vocabularies: all.  2048
//           values at most
//   cluster the CTAs' histograms are added up through distributed shared memory.  Weights enter them in units of 2^-22 of the largest, by
//           32-bit atomics: they say which bins to look at, and what lies in front of those is then added up exactly
//   whole   the same with exact weights, bins divided further by the bits of the values down to a single value, whose ties go by index: long
//           stretches of equal or nearly equal logits, top-p next to 1
//
// Weights are exp2 by a table and a polynomial (P. T. P. Tang, Table-driven implementation of the exponential function, ACM TOMS 15, 1989): near the
// largest in doubles, 32 entries, error 2^-48; the many others by 512 entries of 63 bits, a float32 polynomial of what is left and one integer
// product, of a distance that is exact.  (A float32 exponential, 2^-22 of a weight, moved the borders of 128,256 tokens of nearly equal weight by
// thousandths of one.  64 rows of 128,256: 91 us with that, 98 so, 103 with 32 entries and what they leave in pairs of floats.)
//
// Bound: latencies one behind the other, 1.2 to 2 us for an exchange over the cluster; the reads are 5 of the 92 to 98 us that 64 rows of 128,256
// take, a row of 32,000 by temperature, top-k and top-p takes 25 us.  So a row goes over as many CTAs as give 2048 logits each while there
// are SMs for them, and 16,384 each beyond (the CTAs of a row wait for one another, four rows share an SM's time); where every CTA read all bins
// instead of a share of them, 64 rows took 16 us more.
#include "common.cuh"

#include <math_constants.h>

#include <cstddef>

namespace {

constexpr int kSpThreads = 512;
constexpr int kSpWarps = kSpThreads / 32;
constexpr int kSpBins = 1024;
constexpr int kSpFine = 4096;       // bins of a cluster of four CTAs and more
constexpr int kSpCap = 1024;        // values of one bin that are ranked among each other
constexpr int kSpFew = 2048;        // values that the first CTA sorts
constexpr int kSpList = kSpFew / kSpWarps;  // values of a warp's list
constexpr int kSpStretch = 1024;   // places of a warp's list: its share of the bins' room
constexpr float kSpReach = 16.f;   // distances that histograms of weights take, in temperatures: beyond them a weight is less than half a unit
constexpr int kSpMaxSlice = 40960;  // logits of a CTA: 160 KB
constexpr int kSpMaxCluster = 16;

struct SampleParams {
    const float* logits;
    long long stride;
    int vocab, slice;  // slice: logits of a CTA, a multiple of 4
    int bits;          // S
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p, *uniform;
    int32_t* tokens;
    float* logprob;
};

using u64 = unsigned long long;

struct __align__(16) SampleShared {  // (the slice behind it is written sixteen bytes at a time)
    double exp2_32[32];      // 2^(j/32)
    u64 exp2_512[512];       // 2^(62 + j/512)
    u64 mass[kSpBins];       // bins of weights; running sums over this CTA's share of finer ones; with cand, values on their way to the first CTA
    u64 cand[kSpCap];        // values on their way, their weights
    union {
        u64 few[kSpFew];         // in the first CTA: all CTAs' values that are left, as places
        unsigned fine[kSpFine];  // finer bins
        struct {
            u64 share_mass[kSpBins];  // running sums over this CTA's share of the bins
            unsigned share_count[kSpBins];
            unsigned count[kSpBins];
        };
    };
    union {
        unsigned wlist[kSpFew];  // a bin's values
        u64 cand_w[kSpCap];
    };
    u64 xa[2][kSpMaxCluster], xb[2][kSpMaxCluster];  // a pair of words from every CTA, two exchanges alternating
    u64 ra[2], rb[2], rc[2];                          // an answer from one CTA
    u64 wsum[kSpWarps];
    float wf[kSpWarps];
    unsigned wcount[kSpWarps];
    unsigned n_cand;
};
// (declared again wherever it is used, so that the compiler knows the accesses for shared ones)
#define LB_SAMPLE_SHARED                                       \
    extern __shared__ __align__(16) uint8_t lb_sample_smem[]; \
    SampleShared& s = *reinterpret_cast<SampleShared*>(lb_sample_smem)
static_assert(sizeof(SampleShared) % 16 == 0, "alignment of the slice");
static_assert((kSpBins + kSpCap + kSpFew) * 8 >= kSpWarps * kSpStretch * 2 && offsetof(SampleShared, few) == offsetof(SampleShared, mass) + (kSpBins + kSpCap) * 8, "lists over the bins");
static_assert(kSpBins + kSpCap >= kSpFew, "the values that are left, in the place of the bins");
constexpr size_t kSpLeast = (size_t)kSpFew * 8;  // bytes of the slice's place, where the first CTA keeps weights later
static_assert(sizeof(SampleShared) + (size_t)kSpMaxSlice * 4 <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned ld_cluster_u32(uint32_t addr) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ unsigned add_cluster_u32(uint32_t addr, unsigned v) {
    unsigned old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
}

// larger logit, larger key
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// place in the order: larger first
__device__ __forceinline__ u64 place_of(float l, int index) { return (u64)key_of(l) << 32 | (unsigned)~index; }

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_max_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}
__device__ __forceinline__ u64 warp_scan_u64(u64 v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    return v;
}

// f * total, rounded down or up; 0 <= f < 1
__device__ __forceinline__ u64 part_of(float f, u64 total, bool up) {
    const unsigned b = __float_as_uint(f);
    const int e = (int)(b >> 23 & 255);
    const u64 m = (b & 0x7fffffu) | (e ? 0x800000u : 0u);
    const int shift = 150 - (e ? e : 1);  // f = m 2^-shift; shift >= 24 because f < 1
    const unsigned __int128 x = (unsigned __int128)total * m;
    if (shift >= 100) return up && x != 0 ? 1 : 0;  // (x < 2^86)
    const u64 q = (u64)(x >> shift);
    return q + (up && ((unsigned __int128)q << shift) != x ? 1 : 0);
}

struct Row {
    float top;     // the largest logit
    double inv_t;
    float inv_hi, inv_lo;  // log2(e) / temperature as two floats
    float bin_scale;
    float far;     // no weight beyond it: 48 temperatures
    float least;   // nor below this power of two: half of 2^-S
    int bits;

    __device__ __forceinline__ double distance(float l) const { return ((double)l - (double)top) * inv_t; }
    // round(2^S exp(d)), d <= 0
    __device__ __forceinline__ u64 weight_at(double d) const {
        const double y = d * 1.4426950408889634;                      // log2(e)
        if (!(y > -62.0)) return 0;                                   // (not a number: too)
        const double big = 6755399441055744.0 / 32;                   // 1.5 2^52 / 32: the sum's low word is y rounded to 32nds
        const double k = y + big;
        const int n = __double2loint(k);                              // 32 y
        // the rest in natural units, from d itself: 32nds of ln 2 in two parts, the first with 32 bits
        const double j = k - big;
        const double x = fma(j, -1.9082149292705877e-10, fma(j, -0.6931471803691238, d));
        double e = fma(x, 1.0 / 120, 1.0 / 24);
        e = fma(e, x, 1.0 / 6);
        e = fma(e, x, 0.5);
        e = fma(e, x, 1.0);
        LB_SAMPLE_SHARED;
        const double t = s.exp2_32[n & 31];
        e = fma(t * x, e, t);                                         // 2^(n % 32 / 32) exp(x)
        e = __hiloint2double(__double2hiint(e) + ((n >> 5) + bits) * (1 << 20), __double2loint(e));
        return __double2ull_rn(e);
    }
    // Beyond four temperatures: y + z = log2 of the weight, the 512ths of y by the table, 2^r - 1 of the rest (|r| <= 2^-10) as a float32 polynomial.
    // That is taken in 2^-32ths (the sums with 1.5 2^n have them as their low bits: no conversions): 2^-33 of the weight, and 2^-35 each from the
    // roundings of r and of the polynomial's last two steps, 2^-32 together; what equal values share of it adds up.  The distance itself is the exact
    // difference, as two floats.
    __device__ __forceinline__ u64 weight(float l) const {
        const float far_l = l - top;
        const float y = far_l * inv_hi;
        if (!(y <= -4.f * 1.442695f)) {  // near, equal or not a number
            if (l == top) return 1ull << bits;
            if (top == CUDART_INF_F || l == -CUDART_INF_F) return 0;
            return weight_at(distance(l));
        }
        if (!(y > least)) return 0;
        const float back = far_l - l, rest = (l - (far_l - back)) - (top + back);
        const float z = fmaf(rest, inv_hi, fmaf(far_l, inv_lo, fmaf(far_l, inv_hi, -y)));
        constexpr float kWhole = 24576.f, kPart = 0.0029296875f;  // 1.5 2^14 and 1.5 2^-9
        const float k = y + kWhole, r = (y - (k - kWhole)) + z;
        const float x = fmaf(fmaf(fmaf(0.055504109f, r, 0.24022651f), r, 0.69314718f), r, kPart);  // powers of ln 2 over factorials
        LB_SAMPLE_SHARED;
        const unsigned n = __float_as_uint(k);
        const u64 t = s.exp2_512[n & 511];
        const u64 w = t + (u64)((long long)(int)(t >> 32) * (__float_as_int(x) - 0x3b400000));  // (the table's top half will do: 2^-41 of the weight)
        return ((w >> (61 - bits + (0x46c00000 >> 9) - (int)(n >> 9))) + 1) >> 1;  // (a shift of 62 at most, since y > least)
    }
    __device__ __forceinline__ int bin(float l) const {
        const int b = (int)((top - l) * bin_scale);  // (not a number, from equal infinities: 0)
        return b < kSpBins - 1 ? b : kSpBins - 1;
    }
};

__device__ __forceinline__ uint32_t remote(const void* p, unsigned r) { return lb_cluster_addr(lb_smem_u32(p), r); }

struct Cluster {
    int n, first;    // this CTA's logits, and the first one's index in the row
    int n_most;      // logits of a CTA, at most
    unsigned rank, size;

    // a pair of words from every CTA to every CTA: s.xa[turn], s.xb[turn] by rank; all threads call
    __device__ __forceinline__ int exchange(int& turn, u64 a, u64 b) const {
        LB_SAMPLE_SHARED;
        turn ^= 1;
        if (threadIdx.x < size) {
            st_cluster_u64(remote(&s.xa[turn][rank], threadIdx.x), a);
            st_cluster_u64(remote(&s.xb[turn][rank], threadIdx.x), b);
        }
        lb_cluster_sync();
        return turn;
    }
    // one CTA's answer to every CTA (`mine`: whether this is the one; a, b, c are read from thread 0 .. size-1 of it)
    __device__ __forceinline__ int answer(int& turn, bool mine, u64 a, u64 b, u64 c) const {
        LB_SAMPLE_SHARED;
        turn ^= 1;
        if (mine && threadIdx.x < size) {
            st_cluster_u64(remote(&s.ra[turn], threadIdx.x), a);
            st_cluster_u64(remote(&s.rb[turn], threadIdx.x), b);
            st_cluster_u64(remote(&s.rc[turn], threadIdx.x), c);
        }
        lb_cluster_sync();
        return turn;
    }
};

struct Found {
    int bin;
    u64 base;        // count or weight in front of the bin
    unsigned values; // values in the bin
};

// The histogram of every CTA is complete: adds it up over the cluster, every CTA a share of the bins.  Returns the weight of all bins.
__device__ __noinline__ u64 add_bins(const Cluster c, bool mass, int& turn) {
    LB_SAMPLE_SHARED;
    const int share = kSpBins / c.size, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    lb_cluster_sync();
    u64 run_m = 0;
    unsigned run_c = 0;
    for (int b0 = 0; b0 < share; b0 += kSpThreads) {  // (share is a power of two; rounds of all threads, the first ones of it at work)
        const int b = b0 + threadIdx.x;
        u64 m = 0;
        unsigned n = 0;
        if (b < share) {
            const int at = c.rank * share + b;
            for (unsigned r = 0; r < c.size; ++r) {
                n += ld_cluster_u32(remote(&s.count[at], r));
                if (mass) m += ld_cluster_u64(remote(&s.mass[at], r));
            }
        }
        u64 sm = warp_scan_u64(m, lane);
        unsigned sn = (unsigned)warp_scan_u64(n, lane);
        if (lane == 31) {
            s.wsum[warp] = sm;
            s.wcount[warp] = sn;
        }
        __syncthreads();
        sm += run_m;
        sn += run_c;
        for (int w = 0; w < kSpWarps; ++w) {
            if (w < warp) {
                sm += s.wsum[w];
                sn += s.wcount[w];
            }
            run_m += s.wsum[w];
            run_c += s.wcount[w];
        }
        if (b < share) {
            s.share_mass[b] = sm;
            s.share_count[b] = sn;
        }
        __syncthreads();
    }
    c.exchange(turn, run_c, run_m);
    u64 total = 0;
    for (unsigned r = 0; r < c.size; ++r) total += s.xb[turn][r];
    return total;
}

// The first bin at which the count (mass: the weight) reaches `limit`; `turn` as add_bins left it.
__device__ __noinline__ Found find_bin(const Cluster c, bool mass, u64 limit, int& turn) {
    LB_SAMPLE_SHARED;
    const int share = kSpBins / c.size;
    u64 before = 0;
    unsigned owner = c.size - 1;
    for (unsigned r = 0; r < c.size; ++r) {
        const u64 v = mass ? s.xb[turn][r] : s.xa[turn][r];
        if (before + v >= limit) {
            owner = r;
            break;
        }
        if (r + 1 < c.size) before += v;
    }
    if (c.rank == owner) {
        if (threadIdx.x == 0) {
            s.cand[0] = share - 1;  // (nothing reaches it: the last bin; does not happen with limits up to the total)
        }
        __syncthreads();
        for (int b = threadIdx.x; b < share; b += kSpThreads) {
            const u64 to = before + (mass ? s.share_mass[b] : (u64)s.share_count[b]);
            const u64 from = b ? before + (mass ? s.share_mass[b - 1] : (u64)s.share_count[b - 1]) : before;
            if (to >= limit && from < limit) s.cand[0] = b;
        }
        __syncthreads();
    }
    u64 a = 0, b = 0, n = 0;
    if (c.rank == owner) {
        const int at = (int)s.cand[0];
        a = owner * share + at;
        b = at ? before + (mass ? s.share_mass[at - 1] : (u64)s.share_count[at - 1]) : before;
        n = s.share_count[at] - (at ? s.share_count[at - 1] : 0u);
    }
    const int t = c.answer(turn, c.rank == owner, a, b, n);
    return {(int)s.ra[t], s.rb[t], (unsigned)s.rc[t]};
}

// The place of the last value, among those at or in front of `cut` in the order, that the limit lets through: the limit-th one, or with
// `mass` the first one with which the weight reaches the limit.  limit >= 1 and at most what there is.  With mass and share > 0 the limit
// is that share of the weight.
__device__ __noinline__ u64 find_cut(const Cluster c, const Row row, int& turn, u64 cut, bool mass, u64 limit, float share) {
    LB_SAMPLE_SHARED;
    const float* const x = reinterpret_cast<const float*>(lb_sample_smem + sizeof(SampleShared));
    const unsigned top_key = key_of(row.top);
    int lin = -1;                              // the linear bin that the search has come to, then
    unsigned lo = 0, hi = 0xffffffffu;         // the stretch of top_key - key inside it
    u64 base = 0;
    unsigned values = 0;
    for (int level = 0;; ++level) {
        const int shift = level == 0 ? 0 : level == 1 ? 22 : level == 2 ? 12 : level == 3 ? 2 : 0;
        for (int b = threadIdx.x; b < kSpBins; b += kSpThreads) {
            s.count[b] = 0;
            s.mass[b] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < c.n; i += kSpThreads) {
            const float l = x[i];
            if (place_of(l, c.first + i) < cut) continue;
            int b = row.bin(l);
            if (level > 0) {
                const unsigned d = top_key - key_of(l);
                if (b != lin || d < lo || d > hi) continue;
                b = (int)((d - lo) >> shift);
            }
            atomicAdd(&s.count[b], 1u);
            if (mass) {
                const u64 w = row.weight(l);
                if (w) atomicAdd(&s.mass[b], w);
            }
        }
        const u64 total = add_bins(c, mass, turn);
        if (level == 0 && mass && share >= 0.f) {
            limit = part_of(share, total, true);
            if (limit == 0) limit = 1;
        }
        const Found f = find_bin(c, mass, limit - base, turn);
        base += f.base;
        values = f.values;
        if (level == 0) {
            lin = f.bin;
        } else {
            lo += (unsigned)f.bin << shift;
            hi = lo + ((1u << shift) - 1u);
        }
        if (values <= kSpCap || (level > 0 && shift == 0)) break;
    }
    if (values <= kSpCap) {
        // the values to CTA 0, which ranks them; their order in the list does not matter
        if (threadIdx.x == 0) s.n_cand = 0;
        lb_cluster_sync();
        for (int i = threadIdx.x; i < c.n; i += kSpThreads) {
            const float l = x[i];
            const u64 p = place_of(l, c.first + i);
            const unsigned d = top_key - key_of(l);
            if (p < cut || row.bin(l) != lin || d < lo || d > hi) continue;
            const unsigned at = add_cluster_u32(remote(&s.n_cand, 0), 1u);
            if (at < kSpCap) {
                st_cluster_u64(remote(&s.cand[at], 0), p);
                st_cluster_u64(remote(&s.cand_w[at], 0), mass ? row.weight(l) : 1ull);
            }
        }
        lb_cluster_sync();
        u64 last = ~0ull;
        if (c.rank == 0) {
            const int n = s.n_cand < kSpCap ? (int)s.n_cand : kSpCap;
            for (int i = threadIdx.x; i < n; i += kSpThreads) {
                const u64 p = s.cand[i];
                u64 before = base;
                for (int j = 0; j < n; ++j)
                    if (s.cand[j] > p) before += s.cand_w[j];
                if (before < limit && p < last) last = p;
            }
            last = ~warp_max_u64(~last);
            if ((threadIdx.x & 31) == 0) s.wsum[threadIdx.x >> 5] = last;
            __syncthreads();
            for (int w = 0; w < kSpWarps; ++w) last = s.wsum[w] < last ? s.wsum[w] : last;
        }
        const int t = c.answer(turn, c.rank == 0, last, 0, 0);
        return s.ra[t];
    }
    // one value that more than kSpCap tokens share: the tie-th of them by index
    const unsigned key = top_key - lo;
    const float value = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    u64 tie = limit - base;
    if (mass) {
        const u64 w = row.weight(value);
        tie = w ? (tie + w - 1) / w : 1;
    }
    const int per = ((c.n + kSpThreads - 1) / kSpThreads + 31) / 32 * 32 * 32;  // a warp's stretch of the slice
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int from = min(c.n, warp * per), to = min(c.n, from + per);
    const auto is_tie = [&](int i) { return key_of(x[i]) == key && place_of(x[i], c.first + i) >= cut; };
    unsigned mine = 0;
    for (int i = from + lane; i < to; i += 32) mine += is_tie(i);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) s.wcount[warp] = mine;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < kSpWarps; ++w) all += s.wcount[w];
    const int t0 = c.exchange(turn, all, 0);
    u64 before = 0;
    unsigned owner = 0;
    for (unsigned r = 0; r < c.size; ++r) {
        if (before + s.xa[t0][r] >= tie) {
            owner = r;
            break;
        }
        before += s.xa[t0][r];
    }
    if (c.rank == owner) {
        u64 ahead = before;
        for (int w = 0; w < warp; ++w) ahead += s.wcount[w];
        if (ahead < tie && ahead + s.wcount[warp] >= tie)
            for (int i0 = from; i0 < to; i0 += 32) {
                const int i = i0 + lane;
                const unsigned hit = __ballot_sync(0xffffffffu, i < to && is_tie(i));
                const unsigned need = (unsigned)(tie - ahead);
                if (__popc(hit) >= (int)need) {
                    if ((hit >> lane & 1u) && __popc(hit & ((2u << lane) - 1u)) == (int)need) s.cand[0] = place_of(x[i], c.first + i);
                    break;
                }
                ahead += __popc(hit);
            }
        __syncthreads();
    }
    const u64 at = c.rank == owner ? s.cand[0] : 0;
    const int t = c.answer(turn, c.rank == owner, at, 0, 0);
    return s.ra[t];
}

__device__ __forceinline__ float value_of_key(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ float value_of_place(u64 place) { return value_of_key((unsigned)(place >> 32)); }

// Sorts the n <= kSpFew places in s.few, into bins and then within them: by value, largest first, or by index.  By value, those further than `far`
// below the largest have no weight and are left out: how many there are then.  All of one CTA's threads.
template <bool INDEX>
__device__ __noinline__ int sort_few(int n, float far, int shift) {
    LB_SAMPLE_SHARED;
    u64* sorted = s.mass;  // and s.cand behind it
    unsigned *count = s.wlist, *start = s.wlist + kSpBins;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int E = kSpFew / kSpThreads, B = kSpBins / kSpThreads;
    u64 v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = tid + e * kSpThreads < n ? s.few[tid + e * kSpThreads] : 0;
    float top = -CUDART_INF_F, scale = 0.f;
    if (!INDEX) {
        float least = CUDART_INF_F;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (v[e]) {
                const float l = value_of_place(v[e]);
                top = fmaxf(top, l);
                least = fminf(least, l);
            }
        least = -lb_warp_max(-least);
        top = lb_warp_max(top);
        if (lane == 0) {
            s.wf[warp] = least;
            s.wcount[warp] = __float_as_uint(top);
        }
    }
    for (int b = tid; b < kSpBins; b += kSpThreads) count[b] = 0;
    __syncthreads();
    if (!INDEX) {
        float least = CUDART_INF_F;
        for (int w = 0; w < kSpWarps; ++w) {
            least = fminf(least, s.wf[w]);
            top = fmaxf(top, __uint_as_float(s.wcount[w]));
        }
        scale = 1.f / fminf(top - least, far);
    }
    int bin[E];
    unsigned slot[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        bin[e] = -1;
        if (v[e]) {
            if (INDEX) {
                bin[e] = (int)(~(unsigned)v[e] >> shift);
            } else {
                const float d = top - value_of_place(v[e]);
                // finer towards the far end, where most values are (not a number, from equal ones: 0)
                if (!(d > far)) bin[e] = kSpBins - 1 - min((int)(sqrtf(fmaxf(1.f - d * scale, 0.f)) * kSpBins), kSpBins - 1);
            }
            if (bin[e] >= 0) slot[e] = atomicAdd(&count[bin[e]], 1u);
        }
    }
    __syncthreads();
    unsigned m[B], sum = 0;
#pragma unroll
    for (int e = 0; e < B; ++e) {
        m[e] = count[tid * B + e];
        sum += m[e];
    }
    unsigned upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
    }
    if (lane == 31) s.wsum[warp] = upto;
    __syncthreads();
    unsigned all = 0, ahead = upto - sum;
    for (int w = 0; w < kSpWarps; ++w) {
        if (w < warp) ahead += (unsigned)s.wsum[w];
        all += (unsigned)s.wsum[w];
    }
#pragma unroll
    for (int e = 0; e < B; ++e) {
        start[tid * B + e] = ahead;
        ahead += m[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (bin[e] >= 0) sorted[start[bin[e]] + slot[e]] = v[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (bin[e] >= 0) {
            const unsigned from = start[bin[e]], to = from + count[bin[e]];
            unsigned at = from;
            for (unsigned j = from; j < to; ++j) at += INDEX ? (unsigned)sorted[j] > (unsigned)v[e] : sorted[j] > v[e];  // (the index' complement)
            s.few[at] = v[e];
        }
    __syncthreads();
    return (int)all;
}

// Weights of the first n of s.few, four neighbours a thread, and the sum in front of the thread's; the sum of all.
constexpr int kSpEach = kSpFew / kSpThreads;
__device__ __forceinline__ u64 weights_of_few(const Row& row, int n, u64 (&w)[kSpEach], u64& before) {
    LB_SAMPLE_SHARED;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < kSpEach; ++e) {
        const int i = tid * kSpEach + e;
        w[e] = i < n ? row.weight(value_of_place(s.few[i])) : 0;
        sum += w[e];
    }
    const u64 upto = warp_scan_u64(sum, lane);
    __syncthreads();
    if (lane == 31) s.wsum[warp] = upto;
    __syncthreads();
    u64 all = 0;
    before = upto - sum;
    for (int i = 0; i < kSpWarps; ++i) {
        if (i < warp) before += s.wsum[i];
        all += s.wsum[i];
    }
    return all;
}

// What the first CTA does with the n values that are left (in s.few): cuts, kept weight, token.  `given`: the weight that top-p wants, where that
// is a share of the whole row's; else 0.
__device__ __noinline__ void choose(const Row row, const SampleParams p, int r, int n, int k, float top_p, float min_p, u64 given) {
    LB_SAMPLE_SHARED;
    const int tid = threadIdx.x, lane = tid & 31;
    n = sort_few<false>(n, row.far, 0);
    u64 w[kSpEach], before;
    u64 mass = weights_of_few(row, n, w, before);
    const int first = k > 0 && k < n ? k : n;  // top-k
    if (first < n) {
        u64 upto = before;
#pragma unroll
        for (int e = 0; e < kSpEach; ++e) {
            upto += w[e];
            if (tid * kSpEach + e == first - 1) s.ra[0] = upto;
        }
        __syncthreads();
        mass = s.ra[0];
    }
    u64 need = ~0ull;
    if (top_p < 1.f) {
        need = given ? given : part_of(fmaxf(top_p, 0.f), mass, true);
        if (need == 0) need = 1;
    }
    if (tid == 0) s.n_cand = 0;
    const double log_min = min_p > 0.f ? log((double)min_p) : -CUDART_INF;
    // kept: a run from the front
    unsigned kept = 0;
#pragma unroll
    for (int e = 0; e < kSpEach; ++e) {
        const int i = tid * kSpEach + e;
        bool is = i < first && before < need && w[e] > 0;
        if (is && min_p > 0.f) {
            const float l = value_of_place(s.few[i]);
            if (l != row.top) {
                const double d = row.distance(l);
                is = d > log_min + 1e-6 || (d > log_min - 1e-6 && exp(d) >= (double)min_p);
            }
        }
        kept += is;
        before += w[e];
    }
    kept = __reduce_add_sync(0xffffffffu, kept);
    __syncthreads();
    if (lane == 0 && kept) atomicAdd(&s.n_cand, kept);
    __syncthreads();
    kept = s.n_cand;
    // by index
    int shift = 0;
    while ((p.vocab - 1) >> shift >= kSpBins) ++shift;
    sort_few<true>((int)kept, 0.f, shift);
    const u64 total = weights_of_few(row, (int)kept, w, before);
    const float u = __ldg(p.uniform + r);
    const u64 target = u >= 1.f ? total - 1 : u > 0.f ? part_of(u, total, false) : 0;
#pragma unroll
    for (int e = 0; e < kSpEach; ++e) {
        if (target >= before && target < before + w[e]) {
            const u64 place = s.few[tid * kSpEach + e];
            p.tokens[r] = (int)~(unsigned)place;
            if (p.logprob) {
                const float l = value_of_place(place);
                const double d = l == row.top ? 0.0 : row.distance(l);
                p.logprob[r] = (float)(d - log(ldexp((double)total, -p.bits)));
            }
        }
        before += w[e];
    }
}

// The place at which the limit (count, or with MASS a share of the weight) ends, among the row's values at or in front of `cut` that are
// not below `floor_l`; 0 where the search has to take the whole row; kSpDone where few values were left and the first CTA has seen to them.
constexpr u64 kSpDone = ~0ull;
template <bool MASS>
__device__ __noinline__ u64 cluster_cut(const Cluster c, const Row row, int& turn, u64 cut, float floor_l, u64 limit, float share, float reach, const SampleParams p, int r, int k, float top_p, float min_p) {
    LB_SAMPLE_SHARED;
    const float* const x = reinterpret_cast<const float*>(lb_sample_smem + sizeof(SampleShared));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float cut_l = fmaxf(floor_l, cut ? value_of_place(cut) : -CUDART_INF_F);
    const auto is_in = [&](float l, int i) { return l > cut_l || (l == cut_l && l > -CUDART_INF_F && place_of(l, c.first + i) >= cut); };
    const int bins = c.size >= 4 ? kSpFine : kSpBins, share_bins = bins / c.size;
    const float scale = (float)bins / reach;
    const auto bin_of = [&](float l) {
        const int b = (int)((row.top - l) * scale);
        return b < bins - 1 ? b : bins - 1;
    };
    int unit = row.bits - 22;
again:
    for (int b = tid; b < bins; b += kSpThreads) s.fine[b] = 0;
    __syncthreads();
    u64 sum = 0;
#pragma unroll 2
    for (int i = tid; i < c.n; i += kSpThreads) {
        const float l = x[i];
        if (!is_in(l, i)) continue;
        unsigned q = 1;
        if (MASS) {
            const u64 w = row.weight(l);
            sum += w;
            q = (unsigned)((w + (1ull << (unit - 1))) >> unit);
        }
        if (q) atomicAdd(&s.fine[bin_of(l)], q);
    }
    if (MASS) {
        sum = warp_sum_u64(sum);
        if (lane == 0) s.wsum[warp] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < kSpWarps; ++w) sum += s.wsum[w];
    }
    lb_cluster_sync();
    u64 run = 0;
    for (int b0 = 0; b0 < share_bins; b0 += kSpThreads) {  // this CTA's share of the bins, over the cluster
        const int b = b0 + tid;
        u64 n = 0;
        if (b < share_bins)
#pragma unroll
            for (unsigned r = 0; r < kSpMaxCluster; ++r)  // (all under way at once)
                if (r < c.size) n += ld_cluster_u32(remote(&s.fine[c.rank * share_bins + b], r));
        u64 upto = warp_scan_u64(n, lane);
        __syncthreads();
        if (lane == 31) s.wsum[warp] = upto;
        __syncthreads();
        upto += run;
        for (int w = 0; w < kSpWarps; ++w) {
            if (w < warp) upto += s.wsum[w];
            run += s.wsum[w];
        }
        if (b < share_bins) s.mass[b] = upto;
    }
    int t = c.exchange(turn, run, sum);
    u64 all = 0, counted = 0, most = 0;
    for (unsigned r = 0; r < c.size; ++r) {
        counted += s.xa[t][r];
        all += s.xb[t][r];
        most = s.xb[t][r] > most ? s.xb[t][r] : most;
    }
    if (MASS && (most >> unit) >= 0xf0000000ull) {  // (a bin may have passed 2^32: larger units, in which no CTA's sum does)
        int log2 = 14;
        while ((1 << log2) < c.n_most) ++log2;
        unit = row.bits - (31 - log2);
        goto again;
    }
    u64 need = limit;
    if (MASS) {
        limit = part_of(share, all, true);
        if (limit == 0) limit = 1;
        need = (limit >> unit) + 1;
    }
    if (counted < need) return 0;
    u64 before = 0;
    unsigned owner = 0;
    for (; owner + 1 < c.size && before + s.xa[t][owner] < need; ++owner) before += s.xa[t][owner];
    u64 found = 0, base = 0;
    if (c.rank == owner) {
        for (int b = tid; b < share_bins; b += kSpThreads) {
            const u64 to = before + s.mass[b], from = b ? before + s.mass[b - 1] : before;
            if (to >= need && from < need) {
                s.ra[t] = owner * share_bins + b;  // (this exchange's own words are free)
                s.rb[t] = from;
            }
        }
        __syncthreads();
        found = s.ra[t];
        base = s.rb[t];
    }
    t = c.answer(turn, c.rank == owner, found, base, 0);
    // weights: units may point a bin or two aside
    const int lo = (int)s.ra[t] - (MASS ? 3 : 0), hi = (int)s.ra[t] + (MASS ? 3 : 0);
    base = s.rb[t];
    if (tid == 0) s.n_cand = 0;
    __syncthreads();
    // the values down to that bin (the lowest value that can be in one saves the others' bins)
    const float low_l = hi >= bins - 1 ? -CUDART_INF_F : row.top - (float)(hi + 2) / scale;
    unsigned window = 0, mine = 0;
    unsigned* list = s.wlist + warp * kSpList;
#pragma unroll 2
    for (int i0 = 0; i0 < c.n; i0 += kSpThreads) {
        const int i = i0 + tid;
        const float l = i < c.n ? x[i] : -CUDART_INF_F;
        bool is = l >= low_l && is_in(l, i);
        if (is) {
            const int b = bin_of(l);
            is = b <= hi;
            window += is && b >= lo;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, is), at = mine + __popc(hit & ((1u << lane) - 1u));
        if (is && at < kSpList) list[at] = (unsigned)i;
        mine += __popc(hit);
    }
    const bool listed = mine <= kSpList;  // (this warp's)
    window = __reduce_add_sync(0xffffffffu, window);
    if (lane == 0) {
        s.wcount[warp] = window;
        s.wsum[warp] = mine;
    }
    const int all_listed = __syncthreads_and(listed);
    unsigned near = 0, ahead = 0;
    window = 0;
    for (int w = 0; w < kSpWarps; ++w) {
        window += s.wcount[w];
        if (w < warp) ahead += (unsigned)s.wsum[w];
        near += (unsigned)s.wsum[w];
    }
    if (!all_listed) near += kSpFew;  // (then there is no list to give away)
    t = c.exchange(turn, near, window);
    unsigned from = 0, wfrom = 0, members = 0, left = 0;
    for (unsigned q = 0; q < c.size; ++q) {
        if (q < c.rank) {
            from += (unsigned)s.xa[t][q];
            wfrom += (unsigned)s.xb[t][q];
        }
        left += (unsigned)s.xa[t][q];
        members += (unsigned)s.xb[t][q];
    }
    if (left <= kSpFew) {
        for (unsigned a = lane; a < mine; a += 32) st_cluster_u64(remote(&s.few[from + ahead + a], 0), place_of(x[list[a]], c.first + list[a]));
        lb_cluster_sync();
        bool ok = true;
        if (MASS) {
            if (c.rank == 0) {
                u64 mass = 0;
                for (unsigned i = tid; i < left; i += kSpThreads) mass += row.weight(value_of_place(s.few[i]));
                mass = warp_sum_u64(mass);
                __syncthreads();
                if (lane == 0) s.wsum[warp] = mass;
                __syncthreads();
                mass = 0;
                for (int i = 0; i < kSpWarps; ++i) mass += s.wsum[i];
                ok = mass >= limit;
            }
            t = c.answer(turn, c.rank == 0, ok, 0, 0);
            ok = s.ra[t] != 0;
        }
        if (ok) {
            if (c.rank == 0) choose(row, p, r, (int)left, k, top_p, min_p, MASS ? limit : 0);
            return kSpDone;
        }
        return 0;
    }
    if (members > kSpCap) return 0;
    // the weight in front of the bins exactly, and their values to the first CTA
    if (tid == 0) s.n_cand = 0;
    __syncthreads();
    sum = 0;
    for (int a = listed ? lane : tid; a < (listed ? (int)mine : c.n); a += listed ? 32 : kSpThreads) {
        const int i = listed ? (int)list[a] : a;
        const float l = x[i];
        if (!listed && !(l >= low_l && is_in(l, i))) continue;
        const int b = bin_of(l);
        if (b > hi) continue;
        if (b < lo) {
            if (MASS) sum += row.weight(l);
        } else {
            const unsigned at = atomicAdd(&s.n_cand, 1u);
            st_cluster_u64(remote(&s.few[wfrom + at], 0), place_of(l, c.first + i));
        }
    }
    if (MASS) {
        sum = warp_sum_u64(sum);
        if (lane == 0) s.wsum[warp] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < kSpWarps; ++w) sum += s.wsum[w];
        t = c.exchange(turn, 0, sum);
        base = 0;
        for (unsigned q = 0; q < c.size; ++q) base += s.xb[t][q];
        if (base >= limit) return 0;
    } else {
        lb_cluster_sync();
    }
    u64 at = 0;
    if (c.rank == 0) {
        const int n = sort_few<false>((int)members, CUDART_INF_F, 0);
        u64 w[kSpEach], before;
        if (tid == 0) s.rc[0] = 0;
        if (MASS) {
            weights_of_few(row, n, w, before);
        } else {
            before = (u64)tid * kSpEach;
            __syncthreads();
        }
        before += base;
#pragma unroll
        for (int e = 0; e < kSpEach; ++e) {
            const int i = tid * kSpEach + e;
            const u64 x = MASS ? w[e] : 1;
            if (i < n && before < limit && before + x >= limit) s.rc[0] = s.few[i];
            before += x;
        }
        __syncthreads();
        at = s.rc[0];
    }
    t = c.answer(turn, c.rank == 0, at, 0, 0);
    return s.ra[t];
}

__global__ void __launch_bounds__(kSpThreads, 2) lb_sample_kernel(const SampleParams p) {
    LB_SAMPLE_SHARED;
    float* x = reinterpret_cast<float*>(lb_sample_smem + sizeof(SampleShared));
    unsigned size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = lb_cluster_rank();
    const int first = (int)rank * p.slice, n = max(0, min(p.slice, p.vocab - first));
    lb_cluster_arrive();  // (waited for in front of the first access to another CTA's memory)
    static_assert(kSpThreads == 512, "a thread for each entry");
    const double entry = exp2((double)tid / 512);
    s.exp2_512[tid] = __double2ull_rn(entry * 4611686018427387904.0);
    if (tid % 16 == 0) s.exp2_32[tid / 16] = entry;
    lb_pdl_launch_dependents();
    lb_pdl_wait();
    const float* __restrict__ src = p.logits + (size_t)r * p.stride + first;
    const float temp = p.temperature ? __ldg(p.temperature + r) : 1.f;
    const int k_asked = p.top_k ? __ldg(p.top_k + r) : 0, k = k_asked > 0 && k_asked < p.vocab ? k_asked : 0;
    const float top_p = p.top_p ? __ldg(p.top_p + r) : 1.f;
    const float asked = p.min_p ? __ldg(p.min_p + r) : 0.f;
    const float min_p = asked > 0.f ? fminf(asked, 1.f) : 0.f;
    const Cluster c{n, first, p.slice, rank, size};
    int turn = 0;

    // the slice and its largest value
    float best = -CUDART_INF_F;
    const auto clean = [](float l) { return l != l ? -CUDART_INF_F : l + 0.0f; };  // (one zero)
    const int n4 = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? n / 4 : 0;
#pragma unroll 4
    for (int i = tid; i < n4; i += kSpThreads) {
        float4 v = __ldg(reinterpret_cast<const float4*>(src) + i);
        v = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
        *reinterpret_cast<float4*>(x + 4 * i) = v;
        best = fmaxf(best, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
#pragma unroll 4
    for (int i = n4 * 4 + tid; i < n; i += kSpThreads) {
        const float l = clean(__ldg(src + i));
        x[i] = l;
        best = fmaxf(best, l);
    }
    // what some lanes, a warp or some warps together have read is a group: the smallest of the groups' largest values
    int lanes = 32;  // lanes a group, then warps a group: as many as leave k groups
    while (lanes > 1 && (int)size * (kSpThreads / lanes) < k) lanes /= 2;
    float bound = best;
    for (int o = 1; o < lanes; o *= 2) bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
    bound = -lb_warp_max(-bound);
    best = lb_warp_max(best);
    if (lane == 0) {
        s.wf[warp] = best;
        s.wcount[warp] = __float_as_uint(bound);
    }
    __syncthreads();
    int per = 1;
    while (lanes == 32 && per < kSpWarps && (int)size * (kSpWarps / (per * 2)) >= k) per *= 2;
    bound = CUDART_INF_F;
    for (int w = 0; w < kSpWarps; w += per) {
        float group = __uint_as_float(s.wcount[w]);
        for (int v = 1; v < per; ++v) group = fmaxf(group, __uint_as_float(s.wcount[w + v]));
        bound = fminf(bound, group);
    }
    for (int w = 0; w < kSpWarps; ++w) best = fmaxf(best, s.wf[w]);
    lb_cluster_wait();
    const int t0 = c.exchange(turn, (u64)key_of(best), (u64)key_of(bound));
    unsigned best_key = key_of(best), bound_key = key_of(bound);
    for (unsigned q = 0; q < size; ++q) {
        best_key = max(best_key, (unsigned)s.xa[t0][q]);
        bound_key = min(bound_key, (unsigned)s.xb[t0][q]);
    }
    Row row;
    row.top = value_of_key(best_key);
    row.bits = p.bits;
    row.least = (float)(-1 - p.bits);
    if (row.top == -CUDART_INF_F) {  // nothing to choose
        if (rank == 0 && tid == 0) {
            p.tokens[r] = -1;
            if (p.logprob) p.logprob[r] = CUDART_NAN_F;
        }
        return;
    }
    if (!(temp > 0.f)) {  // (not a number: too) the first largest value
        unsigned at = 0xffffffffu;
        for (int i = tid; i < n; i += kSpThreads)
            if (x[i] == row.top) at = min(at, (unsigned)(first + i));
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) s.wcount[warp] = at;
        __syncthreads();
        for (int w = 0; w < kSpWarps; ++w) at = min(at, s.wcount[w]);
        const int t = c.exchange(turn, at, 0);
        for (unsigned q = 0; q < size; ++q) at = min(at, (unsigned)s.xa[t][q]);
        if (rank == 0 && tid == 0) {
            p.tokens[r] = (int)at;
            if (p.logprob) p.logprob[r] = 0.f;
        }
        return;
    }
    row.inv_t = 1.0 / (double)temp;
    row.inv_hi = (float)(1.4426950408889634 * row.inv_t);
    row.inv_lo = (float)(1.4426950408889634 * row.inv_t - (double)row.inv_hi);
    row.far = 48.f * temp;

    // a value that no kept one is below, where one is known
    float floor_l = -CUDART_INF_F;
    const bool groups = k && (int)size * kSpThreads >= k;
    bool few = false;  // whether not many values can be left
    if (p.vocab <= kSpFew && (k || top_p < 1.f || min_p > 0.f)) {
        few = true;
    } else if (k) {
        if (groups) floor_l = value_of_key(bound_key);
        few = k <= kSpFew / 8;
    } else if (min_p > 0.f && top_p >= 1.f && row.top < CUDART_INF_F) {
        few = true;
        floor_l = row.top + logf(min_p) * temp * 1.0001f - fabsf(row.top) * 1e-6f;
    }
    if (floor_l != floor_l) floor_l = -CUDART_INF_F;  // (no distance at an infinite temperature)
    if (few) {
        unsigned* list = s.wlist + warp * kSpList;
        unsigned mine = 0;
#pragma unroll 2
        for (int i0 = 0; i0 < n; i0 += kSpThreads) {
            const int i = i0 + tid;
            const bool is = i < n && x[i] >= floor_l;
            const unsigned hit = __ballot_sync(0xffffffffu, is), at = mine + __popc(hit & ((1u << lane) - 1u));
            if (is && at < kSpList) list[at] = (unsigned)i;
            mine += __popc(hit);
        }
        __syncthreads();
        if (lane == 0) s.wcount[warp] = mine;
        const int all_listed = __syncthreads_and(mine <= kSpList);
        unsigned ahead = 0, here = 0;
        for (int w = 0; w < kSpWarps; ++w) {
            if (w < warp) ahead += s.wcount[w];
            here += s.wcount[w];
        }
        if (!all_listed) here += kSpFew;  // (then there is no list to give away)
        const int t = c.exchange(turn, here, 0);
        unsigned from = 0, left = 0;
        for (unsigned q = 0; q < size; ++q) {
            if (q < rank) from += (unsigned)s.xa[t][q];
            left += (unsigned)s.xa[t][q];
        }
        if (left <= kSpFew) {
            for (unsigned a = lane; a < mine; a += 32) st_cluster_u64(remote(&s.few[from + ahead + a], 0), place_of(x[list[a]], first + list[a]));
            lb_cluster_sync();
            if (rank == 0) choose(row, p, r, (int)left, k, top_p, min_p, 0);
            return;
        }
    }

    // the whole row
    u64 cut = 0;
    float scale = 0.f;
    const auto whole_scale = [&]() {  // of the whole row's bins
        if (scale != 0.f) return;
        float least = CUDART_INF_F;
        for (int i = tid; i < n; i += kSpThreads)
            if (x[i] > -CUDART_INF_F) least = fminf(least, x[i]);
        least = -lb_warp_max(-least);
        __syncthreads();
        if (lane == 0) s.wf[warp] = least;
        __syncthreads();
        for (int w = 0; w < kSpWarps; ++w) least = fminf(least, s.wf[w]);
        const int t = c.exchange(turn, __float_as_uint(least), 0);
        for (unsigned q = 0; q < size; ++q) least = fminf(least, __uint_as_float((unsigned)s.xa[t][q]));
        row.bin_scale = scale = (float)kSpBins / fminf(32.f * temp, row.top - least);
    };
    const bool plain = row.top < CUDART_INF_F;
    if (k) {
        if (plain && groups && floor_l > -CUDART_INF_F) cut = cluster_cut<false>(c, row, turn, 0, floor_l, (u64)k, 0.f, row.top - floor_l, p, r, k, top_p, min_p);
        if (cut == kSpDone) return;
        if (cut == 0) {
            whole_scale();
            cut = find_cut(c, row, turn, 0, false, (u64)k, -1.f);
        }
    }
    if (top_p < 1.f) {
        u64 at = 0;
        if (plain) at = cluster_cut<true>(c, row, turn, cut, -CUDART_INF_F, 0, fmaxf(top_p, 0.f), kSpReach * temp, p, r, 0, top_p, min_p);
        if (at == kSpDone) return;
        if (at == 0) {
            whole_scale();
            at = find_cut(c, row, turn, cut, true, 1, fmaxf(top_p, 0.f));
        }
        cut = at;
    }
    const float cut_l = cut ? value_of_place(cut) : -CUDART_INF_F;
    const double log_min = min_p > 0.f ? log((double)min_p) : -CUDART_INF;
    const auto kept = [&](int i) -> u64 {
        const float l = x[i];
        if (l < cut_l || (l == cut_l && place_of(l, first + i) < cut)) return 0;
        if (min_p > 0.f) {
            if (row.top == CUDART_INF_F ? l != row.top : l == -CUDART_INF_F) return 0;
            const double d = l == row.top ? 0.0 : row.distance(l);
            if (d < log_min - 1e-6) return 0;
            if (d < log_min + 1e-6 && exp(d) < (double)min_p) return 0;
        }
        return row.weight(l);
    };
    // kept weight by warp, whose stretches follow one another
    const int stretch = (n + kSpWarps * 32 - 1) / (kSpWarps * 32) * 32;
    const int from = min(n, warp * stretch), to = min(n, from + stretch);
    // (few of a row's values are kept once it has been cut: their places first, so that weights are computed for full warps)
    unsigned short* list = reinterpret_cast<unsigned short*>(s.mass) + warp * kSpStretch;
    const bool listed = cut != 0 && stretch <= kSpStretch;
    int kept_n = 0;
    __syncthreads();
    if (listed)
        for (int i0 = from; i0 < to; i0 += 32) {
            const int i = i0 + lane;
            const float l = i < to ? x[i] : -CUDART_INF_F;
            const bool is = i < to && (l > cut_l || (l == cut_l && place_of(l, first + i) >= cut));
            const unsigned hit = __ballot_sync(0xffffffffu, is);
            if (is) list[kept_n + __popc(hit & ((1u << lane) - 1u))] = (unsigned short)(i - from);
            kept_n += __popc(hit);
        }
    __syncwarp();
    const int begin = listed ? 0 : from, end = listed ? kept_n : to;
    const auto at_of = [&](int j) { return listed ? from + list[j] : j; };
    u64 mine = 0;
    for (int j = begin + lane; j < end; j += 32) mine += kept(at_of(j));
    mine = warp_sum_u64(mine);
    __syncthreads();
    if (lane == 0) s.wsum[warp] = mine;
    __syncthreads();
    u64 here = 0;
    for (int w = 0; w < kSpWarps; ++w) here += s.wsum[w];
    const int t = c.exchange(turn, here, 0);
    u64 total = 0, ahead = 0;
    for (unsigned q = 0; q < size; ++q) {
        if (q < rank) ahead += s.xa[t][q];
        total += s.xa[t][q];
    }
    const float u = __ldg(p.uniform + r);
    const u64 target = u >= 1.f ? total - 1 : u > 0.f ? part_of(u, total, false) : 0;
    if (target < ahead || target >= ahead + here) return;
    for (int w = 0; w < warp; ++w) ahead += s.wsum[w];
    if (target < ahead || target >= ahead + s.wsum[warp]) return;
    for (int j0 = begin; j0 < end; j0 += 32) {
        const int i = j0 + lane < end ? at_of(j0 + lane) : 0;
        const u64 w = j0 + lane < end ? kept(i) : 0;
        const u64 upto = ahead + warp_scan_u64(w, lane);
        if (upto > target && upto - w <= target) {
            p.tokens[r] = first + i;
            if (p.logprob) {
                const double d = x[i] == row.top ? 0.0 : row.distance(x[i]);
                p.logprob[r] = (float)(d - log(ldexp((double)total, -p.bits)));
            }
        }
        ahead = __shfl_sync(0xffffffffu, upto, 31);
        if (ahead > target) return;
    }
}

}  // namespace

// CTAs of a row's cluster: 2048 logits each for few rows, up to 16,384 where the rows fill the device
static int sample_cluster(const loom_b200_ctx* ctx, int rows, int vocab) {
    int size = 1;
    while (size < kSpMaxCluster && (vocab + size - 1) / size > ((long long)rows * size <= ctx->sm_count ? 2048 : 16384)) size *= 2;
    return size;
}

int lb_launch_sample(loom_b200_ctx* ctx, int rows, int vocab, const float* logits, long long stride, const float* temperature, const int32_t* top_k,
                     const float* top_p, const float* min_p, const float* uniform, int32_t* tokens, float* logprob) {
    SampleParams p;
    p.logits = logits;
    p.stride = stride;
    p.vocab = vocab;
    const int size = sample_cluster(ctx, rows, vocab);
    p.slice = ((vocab + size - 1) / size + 3) / 4 * 4;
    int log2 = 0;
    while (((long long)1 << log2) < (long long)vocab + 1) ++log2;
    p.bits = 61 - log2;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.uniform = uniform;
    const size_t slice = (size_t)p.slice * 4, smem = sizeof(SampleShared) + (slice > kSpLeast ? slice : kSpLeast);
    if (!(ctx->func_attr_mask2 & (1u << 28))) {
        LB_CUDA(ctx, cudaFuncSetAttribute(lb_sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(SampleShared) + (size_t)kSpMaxSlice * 4)));
        LB_CUDA(ctx, cudaFuncSetAttribute(lb_sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        ctx->func_attr_mask2 |= 1u << 28;
    }
    for (int r0 = 0; r0 < rows; r0 += 65535) {  // (a grid's second dimension)
        const int some = rows - r0 < 65535 ? rows - r0 : 65535;
        p.logits = logits + (size_t)r0 * stride;
        p.temperature = temperature ? temperature + r0 : nullptr;
        p.top_k = top_k ? top_k + r0 : nullptr;
        p.top_p = top_p ? top_p + r0 : nullptr;
        p.min_p = min_p ? min_p + r0 : nullptr;
        p.uniform = uniform + r0;
        p.tokens = tokens + r0;
        p.logprob = logprob ? logprob + r0 : nullptr;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(size, some);
        cfg.blockDim = dim3(kSpThreads);
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
        LB_CUDA(ctx, cudaLaunchKernelEx(&cfg, lb_sample_kernel, p));
        ctx->launches++;
    }
    return 0;
}

extern "C" int loom_b200_sample(loom_b200_ctx* ctx, int rows, int vocab, const float* logits, long long stride, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform, int32_t* tokens, float* logprob) {
    if (!ctx) return lb_fail(nullptr, LOOM_B200_ERR_INVALID, "sample: ctx is NULL");
    LB_REQUIRE(ctx, rows > 0 && vocab > 0, "sample: %d rows of %d logits", rows, vocab);
    LB_REQUIRE(ctx, logits && uniform && tokens, "sample: NULL buffer");
    LB_REQUIRE(ctx, stride >= vocab || (rows == 1 && stride >= 0), "sample: stride %lld of %d logits", stride, vocab);
    if (vocab > kSpMaxSlice * kSpMaxCluster)
        return lb_fail(ctx, LOOM_B200_ERR_UNSUPPORTED, "sample: %d logits in a row, %d at most", vocab, kSpMaxSlice * kSpMaxCluster);
    if (int rc = lb_set_device(ctx)) return rc;
    return lb_launch_sample(ctx, rows, vocab, logits, stride, temperature, top_k, top_p, min_p, uniform, tokens, logprob);
}
