// sample.cu -- the next token of every sequence from its row of logits: temperature, top-k, top-p and min-p, with random numbers that the
// caller gives.
//
// Definition, for a row l of `vocab` logits, temperature T, and m its largest value:
//   weight   w_i = exp((l_i - m) / T); not-a-numbers count as minus infinity, which has weight 0; where m is plus infinity those have weight 1
//            and all others 0
//   order    larger logit first, equal ones by index
//   kept     the first k of the order; of those the shortest run from the front whose weight is at least p times theirs (one token at
//            least); of those the ones with w_i >= min_p
//   token    the first kept one, by index, whose weight and that of the kept ones in front of it exceed u times the kept weight
// T <= 0 is the first largest logit.  Weights are integers, round(w 2^S) with S such that a whole row's sum stays below 2^62: sums do not
// depend on their order then, and are within vocab * 2^-S of the real ones (S = 44 for 128,256 tokens: 7e-9 of the largest weight).
//
// One cluster of CTAs per row, each with a slice of the row in shared memory, so the row is read once and by one launch.  What the kept
// set ends with is one place in the order -- a (logit, index) pair: top-k finds it from a histogram of counts over 1024 linear bins of
// m - l, top-p from one of weights; the bins are added up across the cluster through distributed shared memory, the few values of
// the bin that the limit falls into are gathered in one CTA and ranked there among each other.  A bin with more than 1024 values (long
// stretches of equal or nearly equal logits) is divided further by the bits of the values, down to a single value, whose ties go by index.
#include "common.cuh"

#include <math_constants.h>

namespace {

constexpr int kSpThreads = 512;
constexpr int kSpWarps = kSpThreads / 32;
constexpr int kSpBins = 1024;
constexpr int kSpCap = 1024;        // values that are ranked among each other
constexpr int kSpMaxSlice = 46080;  // logits of a CTA: 180 KB
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

struct SampleShared {
    u64 mass[kSpBins];
    u64 cand[kSpCap], cand_w[kSpCap];
    u64 share_mass[kSpBins];  // running sums over this CTA's share of the bins
    u64 xa[2][kSpMaxCluster], xb[2][kSpMaxCluster];  // a pair of words from every CTA, two exchanges alternating
    u64 ra[2], rb[2], rc[2];                          // an answer from one CTA
    u64 wsum[kSpWarps];
    unsigned count[kSpBins];
    unsigned share_count[kSpBins];
    unsigned wcount[kSpWarps];
    unsigned n_cand;
    int flag;
};

static_assert(sizeof(SampleShared) + (size_t)kSpMaxSlice * 4 <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned ld_cluster_u32(uint32_t addr) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
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
    float bin_scale;
    int bits;

    __device__ __forceinline__ double distance(float l) const { return ((double)l - (double)top) * inv_t; }
    // round(exp(d) 2^S).  Below exp(-15) = 2^-21.6 the float exponential's error, 2^-22 of the value, is 2^-43 of the largest weight.
    __device__ __forceinline__ u64 weight(float l) const {
        if (l == top) return 1ull << bits;
        if (top == CUDART_INF_F || l == -CUDART_INF_F) return 0;
        const double d = distance(l);
        if (d < -44.0) return 0;  // exp(-44) < 2^-63
        if (d < -15.0) return __float2ull_rn(ldexpf(expf((float)d), bits));
        return __double2ull_rn(ldexp(exp(d), bits));
    }
    __device__ __forceinline__ int bin(float l) const {
        const int b = (int)((top - l) * bin_scale);  // (not a number, from equal infinities: 0)
        return b < kSpBins - 1 ? b : kSpBins - 1;
    }
};

struct Cluster {
    SampleShared& s;
    const float* x;  // this CTA's slice
    int n, first;    // its logits, and the first one's index in the row
    unsigned rank, size;
    int turn;

    __device__ __forceinline__ uint32_t remote(const void* p, unsigned r) const { return lb_cluster_addr(lb_smem_u32(p), r); }

    // a pair of words from every CTA to every CTA: s.xa[turn], s.xb[turn] by rank; all threads call
    __device__ __forceinline__ int exchange(u64 a, u64 b) {
        turn ^= 1;
        if (threadIdx.x < size) {
            st_cluster_u64(remote(&s.xa[turn][rank], threadIdx.x), a);
            st_cluster_u64(remote(&s.xb[turn][rank], threadIdx.x), b);
        }
        lb_cluster_sync();
        return turn;
    }
    // one CTA's answer to every CTA (`mine`: whether this is the one; a, b, c are read from thread 0 .. size-1 of it)
    __device__ __forceinline__ int answer(bool mine, u64 a, u64 b, u64 c) {
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
__device__ u64 add_bins(Cluster& c, bool mass, int& turn) {
    SampleShared& s = c.s;
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
                n += ld_cluster_u32(c.remote(&s.count[at], r));
                if (mass) m += ld_cluster_u64(c.remote(&s.mass[at], r));
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
    turn = c.exchange(run_c, run_m);
    u64 total = 0;
    for (unsigned r = 0; r < c.size; ++r) total += s.xb[turn][r];
    return total;
}

// The first bin at which the count (mass: the weight) reaches `limit`; `turn` as add_bins left it.
__device__ Found find_bin(Cluster& c, bool mass, u64 limit, int turn) {
    SampleShared& s = c.s;
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
            s.flag = 0;
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
    const int t = c.answer(c.rank == owner, a, b, n);
    return {(int)s.ra[t], s.rb[t], (unsigned)s.rc[t]};
}

// The place of the last value, among those at or in front of `cut` in the order, that the limit lets through: the limit-th one, or with
// `mass` the first one with which the weight reaches the limit.  limit >= 1 and at most what there is.  With mass and share > 0 the limit
// is that share of the weight.
__device__ u64 find_cut(Cluster& c, const Row& row, u64 cut, bool mass, u64 limit, float share) {
    SampleShared& s = c.s;
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
            const float l = c.x[i];
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
        int turn;
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
            const float l = c.x[i];
            const u64 p = place_of(l, c.first + i);
            const unsigned d = top_key - key_of(l);
            if (p < cut || row.bin(l) != lin || d < lo || d > hi) continue;
            const unsigned at = add_cluster_u32(c.remote(&s.n_cand, 0), 1u);
            if (at < kSpCap) {
                st_cluster_u64(c.remote(&s.cand[at], 0), p);
                st_cluster_u64(c.remote(&s.cand_w[at], 0), mass ? row.weight(l) : 1ull);
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
        const int t = c.answer(c.rank == 0, last, 0, 0);
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
    const auto is_tie = [&](int i) { return key_of(c.x[i]) == key && place_of(c.x[i], c.first + i) >= cut; };
    unsigned mine = 0;
    for (int i = from + lane; i < to; i += 32) mine += is_tie(i);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) s.wcount[warp] = mine;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < kSpWarps; ++w) all += s.wcount[w];
    const int t0 = c.exchange(all, 0);
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
                    if ((hit >> lane & 1u) && __popc(hit & ((2u << lane) - 1u)) == (int)need) s.cand[0] = place_of(c.x[i], c.first + i);
                    break;
                }
                ahead += __popc(hit);
            }
        __syncthreads();
    }
    const u64 at = c.rank == owner ? s.cand[0] : 0;
    const int t = c.answer(c.rank == owner, at, 0, 0);
    return s.ra[t];
}

__global__ void __launch_bounds__(kSpThreads) lb_sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw);
    float* x = reinterpret_cast<float*>(smem_raw + sizeof(SampleShared));
    unsigned size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned rank = lb_cluster_rank();
    const int first = (int)rank * p.slice, n = max(0, min(p.slice, p.vocab - first));
    const float* __restrict__ src = p.logits + (size_t)r * p.stride + first;
    Cluster c{s, x, n, first, rank, size, 0};

    // the slice, its first largest value and its smallest finite one
    u64 best = 0;
    float least = CUDART_INF_F;
    const auto take = [&](int i, float l) {
        l = l != l ? -CUDART_INF_F : l + 0.0f;  // (one zero)
        x[i] = l;
        const u64 at = place_of(l, first + i);
        best = at > best ? at : best;
        if (l > -CUDART_INF_F) least = fminf(least, l);
    };
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        for (int i = threadIdx.x; i < n / 4; i += kSpThreads) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(src) + i);
            take(4 * i, v.x);
            take(4 * i + 1, v.y);
            take(4 * i + 2, v.z);
            take(4 * i + 3, v.w);
        }
        for (int i = n / 4 * 4 + threadIdx.x; i < n; i += kSpThreads) take(i, __ldg(src + i));
    } else {
        for (int i = threadIdx.x; i < n; i += kSpThreads) take(i, __ldg(src + i));
    }
    best = warp_max_u64(best);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
    if (lane == 0) {
        s.wsum[warp] = best;
        s.wcount[warp] = __float_as_uint(least);
    }
    __syncthreads();
    for (int w = 0; w < kSpWarps; ++w) {
        best = s.wsum[w] > best ? s.wsum[w] : best;
        least = fminf(least, __uint_as_float(s.wcount[w]));
    }
    lb_cluster_sync();  // every CTA of the cluster runs: its shared memory may be written
    const int t0 = c.exchange(best, __float_as_uint(least));
    for (unsigned q = 0; q < size; ++q) {
        best = s.xa[t0][q] > best ? s.xa[t0][q] : best;
        least = fminf(least, __uint_as_float((unsigned)s.xb[t0][q]));
    }
    const unsigned best_key = (unsigned)(best >> 32);
    Row row;
    row.top = __uint_as_float(best_key & 0x80000000u ? best_key & 0x7fffffffu : ~best_key);
    row.bits = p.bits;
    const float temp = p.temperature ? __ldg(p.temperature + r) : 1.f;
    const bool writes = rank == 0 && threadIdx.x == 0;
    if (row.top == -CUDART_INF_F) {  // nothing to choose
        if (writes) {
            p.tokens[r] = -1;
            if (p.logprob) p.logprob[r] = CUDART_NAN_F;
        }
        return;
    }
    if (!(temp > 0.f)) {  // (not a number: too)
        if (writes) {
            p.tokens[r] = (int)~(unsigned)best;
            if (p.logprob) p.logprob[r] = 0.f;
        }
        return;
    }
    row.inv_t = 1.0 / (double)temp;
    row.bin_scale = (float)kSpBins / fminf(32.f * temp, row.top - least);

    u64 cut = 0;
    const int k = p.top_k ? __ldg(p.top_k + r) : 0;
    if (k > 0 && k < p.vocab) cut = find_cut(c, row, cut, false, (u64)k, -1.f);
    const float top_p = p.top_p ? __ldg(p.top_p + r) : 1.f;
    if (top_p < 1.f) cut = find_cut(c, row, cut, true, 1, fmaxf(top_p, 0.f));
    const float asked = p.min_p ? __ldg(p.min_p + r) : 0.f;
    const float min_p = asked > 0.f ? fminf(asked, 1.f) : 0.f;
    const double log_min = min_p > 0.f ? log((double)min_p) : -CUDART_INF;
    const auto kept = [&](int i) -> u64 {
        const float l = x[i];
        if (place_of(l, first + i) < cut) return 0;
        if (min_p > 0.f) {
            if (row.top == CUDART_INF_F ? l != row.top : l == -CUDART_INF_F) return 0;
            const double d = l == row.top ? 0.0 : row.distance(l);
            if (d < log_min - 1e-6) return 0;
            if (d < log_min + 1e-6 && exp(d) < (double)min_p) return 0;
        }
        return row.weight(l);
    };
    // kept weight by warp, whose stretches follow one another
    const int per = (n + kSpWarps * 32 - 1) / (kSpWarps * 32) * 32;
    const int from = min(n, warp * per), to = min(n, from + per);
    u64 mine = 0;
    for (int i = from + lane; i < to; i += 32) mine += kept(i);
    mine = warp_sum_u64(mine);
    __syncthreads();
    if (lane == 0) s.wsum[warp] = mine;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < kSpWarps; ++w) all += s.wsum[w];
    const int t = c.exchange(all, 0);
    u64 total = 0, ahead = 0;
    for (unsigned q = 0; q < size; ++q) {
        if (q < rank) ahead += s.xa[t][q];
        total += s.xa[t][q];
    }
    const float u = __ldg(p.uniform + r);
    const u64 target = u >= 1.f ? total - 1 : u > 0.f ? part_of(u, total, false) : 0;
    if (target < ahead || target >= ahead + all) return;
    for (int w = 0; w < warp; ++w) ahead += s.wsum[w];
    if (target < ahead || target >= ahead + s.wsum[warp]) return;
    for (int i0 = from; i0 < to; i0 += 32) {
        const int i = i0 + lane;
        const u64 w = i < to ? kept(i) : 0;
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

// bytes of shared memory and CTAs of a row's cluster
static int sample_cluster(int vocab) {
    int size = 1;
    while (size < kSpMaxCluster && (vocab + size - 1) / size > 8192) size *= 2;
    return size;
}

int lb_launch_sample(loom_b200_ctx* ctx, int rows, int vocab, const float* logits, long long stride, const float* temperature, const int32_t* top_k,
                     const float* top_p, const float* min_p, const float* uniform, int32_t* tokens, float* logprob) {
    SampleParams p;
    p.logits = logits;
    p.stride = stride;
    p.vocab = vocab;
    const int size = sample_cluster(vocab);
    p.slice = ((vocab + size - 1) / size + 3) / 4 * 4;
    int log2 = 0;
    while (((long long)1 << log2) < (long long)vocab + 1) ++log2;
    p.bits = 61 - log2;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.uniform = uniform;
    const size_t smem = sizeof(SampleShared) + (size_t)p.slice * 4;
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
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
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
