// kv8_rows.cuh -- attention of a portion's rows over the 8-bit cache, on the 5th-generation tensor cores (tcgen05, kind::f16).
//
// A tile is 128 rows of one KV head's group; a thread has a row (its TMEM lane).  For every block of 64 positions:
//     S = Q K^T   [128][64] in tensor memory
//     p           the row's scores, its running maximum and sum, weights over S in tensor memory, from where the second product takes them
//     O = P V     [128][dimensions] in tensor memory, then times the block's factors onto the row's result in registers
//
// Codes are float16 numbers as they are.  A float32 query, times the power of two that brings its row's largest value to 2^14 .. 2^15, is the
// sum of two float16 numbers but for 2^-24 of it, and so is a weight, which runs from 2^14 down: two products each, the lower part's first,
// and sums that start anew with every block, so that a float32 accumulator takes few terms.  (On integer digits, as the kernel for few
// rows has it, three accumulators each have to be put together: 2000 instructions a row and block instead of 700.)
//
// Four warps have the rows, four make float16 numbers of the next block's codes and issue the products: S of block b + 1, while the rows have
// their weights of block b, then O of block b, which the rows take up after their scores of block b + 1.
//
// The open block's float32 rows become two float16 numbers too, each row with a power of two of its own.  Three products of parts (the fourth is
// 2^-24 of the first); the keys' factors go to the scores, the values' to the weights, which are then taken relative to the row's largest.
//
// Work is a list: sequences, KV heads, tiles, parts of a tile's blocks, every CTA its place and those a grid further on.  Parts are put together
// by twos, so that results repeat bit for bit.
//
// Bound: a block costs two CTAs of an SM 2.7 us: weights 0.8 and 0.5, results 0.5, waiting for S 0.5 (its MMAs come 94 clocks apart, with an operand A
// of 4 KB of shared memory for 64 columns), the tensor pipe counted as active 14 % and issue slots 33 % of the kernel.  300 rows of 20 heads over 5 of 128 dimensions at position 2900: 63.6 us (without these
// tiles, on integer instructions, 93 us; with them on integer digits 89 us; with one set of warps for both kinds of work 66 us), of which 12 are the list and
// the queries, 28 the blocks, 15 the parts' joining; 2048 rows at 8000: 755 us (1690), 2048 from the start 135 us (354).
constexpr int kRwThreads = 256;
constexpr int kRwWarps = kRwThreads / 32;
constexpr int kRwHalf = kRwThreads / 2;
constexpr int kRwRegs = 216, kRwFeedRegs = 40;  // a thread's, of 128 at the launch
static_assert(kRwRegs + kRwFeedRegs == 256, "what the launch has, and no more");
constexpr int kRwTile = 128;
constexpr int kRwCols = 256;    // of tensor memory: S twice, O
constexpr int kRwSizes = 8;     // sizes of parts that are tried
constexpr int kRwFixed = 4;     // what a part costs beside its blocks, in blocks, and putting two together
constexpr int kRwLevel = 2;
constexpr int kRwLeast = 4;     // blocks of a part, at least (13 rows of 4 heads at 2900: 43 us; with 3 the same, with 6 45 us, with 13 55 us)
constexpr float kRwWeight = 16384.f;
constexpr float kRwLag = 8.f;  // a row's results are scaled anew where a block's largest score is so far above theirs, as a power of two (by as much may they overflow sooner)

template <int NK>
struct RowsShape {
    static constexpr int DK = 32 * NK, KC = 4 * NK;  // dimensions; 16-byte columns of a row of them
    // Bytes from one 16-byte column to the next, where a warp writes a row at a time: sixteen over a multiple of 128, so that its columns are in
    // different banks.  Keys and values made of codes are written eight rows at a time.
    static constexpr int kQCol = kRwTile * 16 + 16;
    static constexpr int kOpenCol = kKvBlock * 16 + 16;
    static constexpr int kOpenRows = 128 + 16;       // of the open block's values, from eight dimensions to the next
    static constexpr int kQ = KC * kQCol;            // a part of Q, a block of keys or values, the open block's parts, a block's codes
    static constexpr int kB = kKvBlock * DK * 2;
    static constexpr int kOpenK = KC * kOpenCol;
    static constexpr int kOpenV = 8 * (DK / 8) * kOpenRows;
    static constexpr int kRaw = kKvBlock * DK;
    static constexpr size_t kSmem = 2 * kQ + 2 * kB + 2 * kRaw;
    static_assert(2 * (kOpenK > kOpenV ? kOpenK : kOpenV) + 2 * kKvBlock * 4 <= 2 * kB + 2 * kRaw, "room for the open block");
    static constexpr size_t kPart = (size_t)kRwTile * (DK + 2);  // floats of a part: [DK / 4][128][4], largest scores, sums
};

// float32 sums, float16 operands, B K-major
__host__ __device__ constexpr uint32_t idesc_f16(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRwTile >> 4) << 24); }
// A in tensor memory: a lane's row, two values a column
__device__ __forceinline__ void mma_f16_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two values as float16, and what is left of them as float16
__device__ __forceinline__ void halves_of(float a, float b, uint32_t& high, uint32_t& low) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
    high = *reinterpret_cast<const uint32_t*>(&h);
    low = *reinterpret_cast<const uint32_t*>(&r);
}
// sixteen codes as float16: 1024 + (code + 128) as a bit pattern, less 1152
__device__ __forceinline__ void put_codes(uint8_t* to, uint4 w) {
    const uint32_t in[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    uint32_t out[8];
    const __half2 zero = __half2half2(__ushort_as_half(0x6480));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t x = __byte_perm(in[i >> 1], 0x64646464u, i & 1 ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), zero);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(out[0], out[1], out[2], out[3]);
    *reinterpret_cast<uint4*>(to + 128) = make_uint4(out[4], out[5], out[6], out[7]);
}

// a row's largest magnitude as bits (above those of every number: not finite), four values a lane
__device__ __forceinline__ uint32_t row_top(const float4& f) {
    const uint32_t a = max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu), b = max(__float_as_uint(f.z) & 0x7fffffffu, __float_as_uint(f.w) & 0x7fffffffu);
    return __reduce_max_sync(0xffffffffu, max(a, b));
}
// the power of two that brings such a row to 2^14 .. 2^15 (the smallest rows below that), as an exponent's field
__device__ __forceinline__ uint32_t row_field(uint32_t bits) { return min(268u - min(bits >> 23, 254u), 253u); }
__device__ __forceinline__ float row_factor(uint32_t bits) { return __uint_as_float((254u - row_field(bits)) << 23); }  // and back
// four values of it in two parts
__device__ __forceinline__ void row_parts(const float4& f, uint32_t bits, uint2 (&part)[2]) {
    const float mul = __uint_as_float(row_field(bits) << 23);
    halves_of(f.x * mul, f.y * mul, part[0].x, part[1].x);
    halves_of(f.z * mul, f.w * mul, part[0].y, part[1].y);
    if (bits >= 0x7f800000u) part[0] = part[1] = make_uint2(0u, 0u);  // (of no consequence for other rows: its factor makes it not a number)
}

template <int NK>
__global__ void __launch_bounds__(kRwThreads, 2) lb_kv8_rows_kernel(const AttendParams p) {
    using S = RowsShape<NK>;
    constexpr int DK = S::DK, KC = S::KC;
    extern __shared__ __align__(128) uint8_t rows_smem[];
    uint8_t* sq = rows_smem;             // [2][KC][128 rows][16 bytes] Q
    uint8_t* sk = sq + 2 * S::kQ;        // [64 positions / 8][KC][8][16 bytes] keys; the open block's, in two parts, over both
    uint8_t* sv = sk + S::kB;            // [dimensions / 8][8][8][16 bytes] values
    uint8_t* raw = sv + S::kB;           // [2][64 x dimensions] codes on their way: keys, values
    float* s_ks = reinterpret_cast<float*>(raw + 2 * S::kRaw) - 2 * kKvBlock;  // (the open block's factors, when no codes are)
    float* s_vs = s_ks + kKvBlock;
    __shared__ unsigned s_scan[kRwWarps][kRwSizes], s_first[2], s_most[kRwWarps];
    __shared__ int s_seq[2], s_last;
    __shared__ uint32_t s_tmem;
    __shared__ __align__(8) uint64_t s_bar[4];  // S (of an even block, of an odd one: the next but one may be there before a row has waited), O, the weights
    const Kv8& c = p.c;
    const int hd = c.dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    lb_pdl_wait();

    // ---- the list of work: sequences, KV heads, tiles, parts ----
    struct Seq {
        Span a;
        int blocks, tiles;  // blocks (the open one included) that its last row sees
    };
    const auto seq_of = [&](int s) {
        Seq q;
        q.a = span_of(p.starts, p.lengths, p.rows, s);
        q.blocks = q.tiles = 0;
        if (q.a.count > 0 && fits(c, q.a) && q.a.count * p.group > kAtWideRows) {
            q.tiles = (q.a.count * p.group + kRwTile - 1) / kRwTile;
            q.blocks = (q.a.pos + q.a.count - 1) / kKvBlock + 1;
        }
        return q;
    };
    bool some = false;
    for (int i = tid; i < c.seqs; i += kRwThreads) some = some || seq_of(i).tiles > 0;
    if (!__syncthreads_or(some)) return;
    if (tid == 0) {
        lb_mbar_init(&s_bar[0], 1);
        lb_mbar_init(&s_bar[1], 1);
        lb_mbar_init(&s_bar[2], 1);
        lb_mbar_init(&s_bar[3], kRwHalf / 32);
        lb_fence_mbar_init();
    }
    // blocks of a part: the size of those tried for which rounds of parts times their length is least (more work than 32 bits hold, by sequences that
    // share rows, gives a share beyond every sequence's blocks: parts are tiles then, which 31 bits do hold)
    const int my_size = lane % kRwSizes;
    unsigned size = 0, most = 0, parts = 0;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        unsigned v = 0, longest = 0;
#pragma unroll 1
        for (int i = warp * (32 / kRwSizes) + lane / kRwSizes; i < c.seqs; i += kRwThreads / kRwSizes) {
            const Seq q = seq_of(i);
            v = add_work(v, c.heads * q.tiles * (pass == 0 ? (unsigned)q.blocks : (q.blocks + size - 1) / size));
            longest = max(longest, (unsigned)q.blocks);
        }
#pragma unroll
        for (int o = kRwSizes; o < 32; o <<= 1) v = add_work(v, __shfl_xor_sync(0xffffffffu, v, o));
        longest = __reduce_max_sync(0xffffffffu, longest);
        __syncthreads();
        if (lane < kRwSizes) s_scan[warp][lane] = v;
        if (lane == 0) s_most[warp] = longest;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < kRwWarps; ++w) v = add_work(v, s_scan[w][my_size]);
        if (pass == 0) {
#pragma unroll
            for (int w = 0; w < kRwWarps; ++w) most = max(most, s_most[w]);
            const unsigned share = v / p.ctas + 1;
            const unsigned eighths = 0xca987650u >> (4 * my_size) & 15;  // 5/8 .. 12/8 of an equal share; first, no cuts
            size = my_size == 0 ? most : min(most, max((unsigned)kRwLeast, (unsigned)((unsigned long long)share * eighths / 8) + 1));
        } else {
            const unsigned long long cost = (unsigned long long)((v + p.ctas - 1) / p.ctas) * (size + kRwFixed) + kRwLevel * (32 - __clz((int)((most + size - 1) / size) - 1));
            unsigned best = size < most && v > 2u * p.ctas ? 0xfffffff0u : (unsigned)min(cost << 3, 0xffffffe0ull);  // (there is room for so many parts)
            best = __reduce_min_sync(0xffffffffu, best / kRwSizes * kRwSizes + my_size) % kRwSizes;
            size = __shfl_sync(0xffffffffu, size, best);
            parts = __shfl_sync(0xffffffffu, v, best);
        }
    }

    if (blockIdx.x >= parts) return;

    // ---- tensor memory, before any later kernel's CTA may come and want its own ----
    if (warp == 0) lb_tmem_alloc(&s_tmem, kRwCols);
    lb_tc_fence_before();
    __syncthreads();
    lb_tc_fence_after();
    lb_pdl_launch_dependents();
    const uint32_t tmem = s_tmem;
    const uint64_t desc_q = lb_smem_desc(lb_smem_u32(sq), S::kQCol, 128), desc_k = lb_smem_desc(lb_smem_u32(sk), 128, 128 * KC), desc_v = lb_smem_desc(lb_smem_u32(sv), 128, 1024);
    uint32_t phases = 0;
    bool alive = true;  // no wait has run out
    const auto wait_for = [&](int which) {
        if (alive && !lb_mbar_wait_bounded(&s_bar[which], phases >> which & 1)) {
            atomicExch(c.status, 1);
            alive = false;
        }
        phases ^= 1u << which;
        __syncwarp();
        lb_tc_fence_after();
    };

    const int role = warp >= kRwHalf / 32, tr = tid % kRwHalf, wr = warp % (kRwHalf / 32);  // in its half
    const auto half_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + role), "r"(kRwHalf) : "memory"); };
    // part n: for a whole half
    struct Part {
        Span a;
        size_t head;  // of its blocks
        int s, h, r0, nr, cut, cuts, b0, bend, closed, token0, head0;
        bool open;
    };
    const auto token_of = [&](const Part& t, int r) { return t.token0 + (p.group_inv ? (int)__umulhi((unsigned)(t.head0 + r), p.group_inv) : r); };
    const auto row_at = [&](const Part& t, int r, long long ld) {
        const int token = token_of(t, r);
        return (size_t)(t.a.row + token) * ld + (size_t)(t.h * p.group + t.r0 + r - token * p.group) * hd;
    };
    const auto part_at = [&](unsigned n) {
        unsigned before = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < c.seqs; s0 += kRwHalf) {
            unsigned mine = 0;
            if (s0 + tr < c.seqs) {
                const Seq q = seq_of(s0 + tr);
                mine = c.heads * q.tiles * ((q.blocks + size - 1) / size);
            }
            unsigned sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            half_sync();
            if (lane == 31) s_scan[warp][0] = sum;
            half_sync();
            unsigned all = 0;
#pragma unroll
            for (int w = 0; w < kRwHalf / 32; ++w) {
                const unsigned u = s_scan[role * (kRwHalf / 32) + w][0];
                if (w < wr) sum += u;
                all += u;
            }
            sum += before;
            before += all;
            if (n < sum && n >= sum - mine) {
                s_seq[role] = s0 + tr;
                s_first[role] = sum - mine;
            }
        }
        half_sync();
        Part t;
        t.s = s_seq[role];
        const Seq q = seq_of(t.s);
        t.a = q.a;
        t.cuts = (int)((q.blocks + size - 1) / size);
        const int rel = (int)(n - s_first[role]), unit = rel / t.cuts;
        t.cut = rel - unit * t.cuts;
        t.h = unit / q.tiles;
        t.r0 = (unit - t.h * q.tiles) * kRwTile;
        t.nr = min(kRwTile, q.a.count * p.group - t.r0);  // rows i = token * group + head
        t.token0 = t.r0 / p.group;
        t.head0 = t.r0 - t.token0 * p.group;
        t.closed = (q.a.pos + q.a.count) / kKvBlock;  // whole blocks
        const int blocks = (q.a.pos + token_of(t, t.nr - 1)) / kKvBlock + 1;  // of this tile
        const int b1 = (int)((long long)blocks * (t.cut + 1) / t.cuts);
        t.b0 = (int)((long long)blocks * t.cut / t.cuts);
        t.bend = min(b1, t.closed);
        t.open = b1 == blocks && t.closed < blocks;
        t.head = c.head_of(t.s, t.h) * c.blocks;
        return t;
    };
    const auto tm_s = [&](int which) { return tmem + 64 * which; };
    // S (+)= a part of Q times keys, and O (+)= a part of the weights times values; by one thread.  (A descriptor's address is in sixteens of
    // bytes; `step`: from sixteen values of all rows to the next, two columns.)
    const auto mma_s = [&](int which, int part, uint64_t keys, int step, bool more) {
        const uint64_t dq = desc_q + (part * S::kQ >> 4);
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i) lb_mma_f16(tm_s(which), dq + i * (2 * S::kQCol >> 4), keys + i * (step >> 4), idesc_f16(kKvBlock), more || i > 0);
    };
    const auto mma_o = [&](int which, int part, uint64_t values, int step, bool more) {
#pragma unroll
        for (int i = 0; i < kKvBlock / 16; ++i) mma_f16_tmem(tmem + 128, tm_s(which) + 32 * part + 8 * i, values + i * (step >> 4), idesc_f16(DK), more || i > 0);
    };
    const auto shared_written = [&]() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); };  // for the tensor core to read

    if (role == 1) {
        // ---- codes into operands, and the tensor core's work ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRwFeedRegs));
#pragma unroll 1
        for (unsigned n = blockIdx.x; n < parts; n += gridDim.x) {
            const Part t = part_at(n);
            // A block's codes on their way, 16 bytes a thread and step, and as float16 numbers where the tensor core reads them: a thread makes
            // them of what it has asked for itself.
            struct Place {
                int code, half;  // bytes: in the block as the cache holds it, and in its float16 numbers
            };
            const auto key_place = [&](int i) -> Place {
                const int u = i * kRwHalf + tr, j = u / (16 * NK), r = u % (16 * NK), end = r - NK / 2 * 32;
                const int row = r % 8, col = end < 0 ? r / 32 * 4 + r % 32 / 8 : NK / 2 * 4 + end / 8;
                return {j * 8 * DK + (end < 0 ? r / 32 * 512 + row * 64 + r % 32 / 8 * 16 : NK / 2 * 512 + row * 32 + end / 8 * 16), (j * KC + 2 * col) * 128 + row * 16};
            };
            const auto value_place = [&](int i) -> Place {
                const int u = i * kRwHalf + tr, row = u % 8, col = u % 32 / 8;
                return {u / 32 * 512 + row * 64 + col * 16, (u / 32 * 8 + 2 * col) * 128 + row * 16};
            };
            const int v_bytes = kKvBlock * c.dim_v;
            const uint8_t *k_from = c.k + t.head * S::kRaw, *v_from = c.v + t.head * v_bytes;
            const auto copy_keys = [&](int b) {
                if (b < t.bend)
#pragma unroll
                    for (int i = 0; i < NK; ++i) copy16(raw + key_place(i).code, k_from + (size_t)b * S::kRaw + key_place(i).code);
                copies_commit();
            };
            const auto copy_values = [&](int b) {
                if (b < t.bend)
#pragma unroll
                    for (int i = 0; i < NK; ++i)
                        if (value_place(i).code < v_bytes) copy16(raw + S::kRaw + value_place(i).code, v_from + (size_t)b * v_bytes + value_place(i).code);
                copies_commit();
            };
            const auto make_keys = [&]() {
#pragma unroll
                for (int i = 0; i < NK; ++i) put_codes(sk + key_place(i).half, *reinterpret_cast<const uint4*>(raw + key_place(i).code));
            };
            const auto make_values = [&]() {
#pragma unroll
                for (int i = 0; i < NK; ++i)
                    if (value_place(i).code < v_bytes) put_codes(sv + value_place(i).half, *reinterpret_cast<const uint4*>(raw + S::kRaw + value_place(i).code));
            };
            copy_keys(t.b0);
            copy_values(t.b0);
            if (t.b0 < t.bend) {
                copies_wait<1>();
                make_keys();
                shared_written();
            }
            copy_keys(t.b0 + 1);
            __syncthreads();  // the queries are there too
            if (tr == 0 && t.b0 < t.bend) {
                mma_s(0, 1, desc_k, 256, false);
                mma_s(0, 0, desc_k, 256, true);
                lb_mma_commit(&s_bar[0]);
            }
            __syncwarp();
#pragma unroll 1
            for (int b = t.b0; b < t.bend; ++b) {
                const int which = (b - t.b0) & 1;
                copies_wait<0>();
                wait_for(which);  // (the keys have been read)
                if (b + 1 < t.bend) make_keys();
                if (b > t.b0) wait_for(2);  // (and the values)
                make_values();
                shared_written();  // (in front of the copies: a fence waits for what is on its way)
                half_sync();
                copy_values(b + 1);
                copy_keys(b + 2);
                if (tr == 0) {
                    if (b + 1 < t.bend) {
                        mma_s(which ^ 1, 1, desc_k, 256, false);
                        mma_s(which ^ 1, 0, desc_k, 256, true);
                        lb_mma_commit(&s_bar[which ^ 1]);
                    }
                    if (alive && !lb_mbar_wait_bounded(&s_bar[3], phases >> 3 & 1)) {
                        atomicExch(c.status, 1);
                        alive = false;
                    }
                    lb_tc_fence_after();
                    mma_o(which, 1, desc_v, 256, false);
                    mma_o(which, 0, desc_v, 256, true);
                    lb_mma_commit(&s_bar[2]);
                }
                phases ^= 8;
                __syncwarp();
            }
            copies_wait<0>();
            if (t.b0 < t.bend) wait_for(2);
            if (t.open) {  // (the other half's work, on the same barriers)
                phases ^= 1 | 4;
            }
            __syncthreads();
        }
    } else {
        // ---- the rows' half ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRwRegs));
        const uint32_t my_tmem = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll 1
        for (unsigned n = blockIdx.x; n < parts; n += gridDim.x) {
            const Part t = part_at(n);
            const Span& a = t.a;
            const int nr = t.nr, closed = t.closed;

            // ---- queries in two parts, a warp its own rows ----
            float m = -CUDART_INF_F, l = 0.f, qs = 0.f;
            const bool q_wide = ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)p.ldq * 4 | (uintptr_t)hd * 4) & 15) == 0;
            const size_t my_row = row_at(t, min(tid, nr - 1), p.ldq);
            // four dimensions of a row in memory, zeros behind its end
            const auto four = [&](const float* row, bool is, bool wide) {
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                const int d = 4 * lane;
                if (!is || d >= hd) return f;
                if (wide) return __ldg(reinterpret_cast<const float4*>(row + d));
                f.x = __ldg(row + d);
                if (d + 1 < hd) f.y = __ldg(row + d + 1);
                if (d + 2 < hd) f.z = __ldg(row + d + 2);
                if (d + 3 < hd) f.w = __ldg(row + d + 3);
                return f;
            };
            float4 next[8];
            const auto ask = [&](int i0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) next[i] = four(p.q + __shfl_sync(0xffffffffu, my_row, (i0 + i) & 31), i0 < 32 && warp * 32 + i0 + i < nr, q_wide);
            };
            ask(0);
#pragma unroll 1
            for (int i0 = 0; i0 < 32; i0 += 8) {
                float4 f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = next[i];
                ask(i0 + 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = warp * 32 + i0 + i;
                    const uint32_t bits = row_top(f[i]);
                    uint2 part[2];
                    row_parts(f[i], bits, part);
                    if (lane == i0 + i) {
                        qs = row_factor(bits);
                        if (bits >= 0x7f800000u) l = CUDART_NAN_F;
                    }
                    if (lane < DK / 4)
#pragma unroll
                        for (int k = 0; k < 2; ++k) *reinterpret_cast<uint2*>(sq + k * S::kQ + (lane >> 1) * S::kQCol + r * 16 + (lane & 1) * 8) = part[k];
                }
            }
            const int see = tid < nr ? a.pos + token_of(t, tid) : -1;  // the row's last position
            const int first_seen = a.pos + t.token0;
            const float cr = p.scale * qs * (1.f / 127.f);
            float o[DK], sc[kKvBlock];
#pragma unroll
            for (int d = 0; d < DK; ++d) o[d] = 0.f;

            const auto my_s = [&](int which) { return my_tmem + 64 * which; };
            const auto load_scores = [&](int which) {
#pragma unroll
                for (int i = 0; i < kKvBlock; i += 16) lb_tmem_ld16(my_s(which) + i, sc + i);
                lb_tmem_wait_ld();
            };
            // weights in two parts over the scores, in the order of the values' positions
            const auto put_weights = [&](int which) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    uint32_t high[8], low[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) halves_of(sc[8 * j + 2 * t], sc[8 * j + 2 * t + 1], high[j], low[j]);
                    tmem_st8(my_s(which) + 8 * t, high);
                    tmem_st8(my_s(which) + 32 + 8 * t, low);
                }
                tmem_wait_st();
            };
            const auto rescale = [&](float old) {
                if (__any_sync(0xffffffffu, old != 1.f))
#pragma unroll
                    for (int d = 0; d < DK; ++d) o[d] *= old;
            };
            const auto add_values = [&](float mul) {
                wait_for(2);
#pragma unroll
                for (int d = 0; d < DK; d += 32) {
                    float f[32];
                    lb_tmem_ld16(my_tmem + 128 + d, f);
                    lb_tmem_ld16(my_tmem + 128 + d + 16, f + 16);
                    lb_tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[d + i] = fmaf(f[i], mul, o[d + i]);
                }
            };

            shared_written();
            __syncthreads();  // the first keys are there too

            // ---- whole blocks ----
            float kt = 0.f, vt = 0.f, mul = 0.f;
            if (t.b0 < t.bend) {
                kt = __ldg(c.k_top + t.head + t.b0);
                vt = __ldg(c.v_top + t.head + t.b0);
            }
#pragma unroll 1
            for (int b = t.b0; b < t.bend; ++b) {
                const int which = (b - t.b0) & 1;
                float kt1 = 0.f, vt1 = 0.f;
                if (b + 1 < t.bend) {
                    kt1 = __ldg(c.k_top + t.head + b + 1);
                    vt1 = __ldg(c.v_top + t.head + b + 1);
                }
                wait_for(which);
                load_scores(which);
                const int last = see - b * kKvBlock;
                if ((b + 1) * kKvBlock - 1 > first_seen) {
#pragma unroll
                    for (int i = 0; i < kKvBlock; ++i) sc[i] = i > last ? -CUDART_INF_F : sc[i];
                }
                float top = -CUDART_INF_F;
#pragma unroll
                for (int i = 0; i < kKvBlock; ++i) top = fmaxf(top, sc[i]);
                const bool any = last >= 0;  // the row sees a part of the block
                const float cs = fmaxf(cr * kt, 1e-37f);  // (0 times a masked score)
                top = any ? top * cs : 0.f;
                float sum[4] = {};
#pragma unroll
                for (int i = 0; i < kKvBlock; ++i) {
                    sc[i] = exp2_of(fmaf(sc[i], cs, 14.f - top));
                    sum[i & 3] += sc[i];
                }
                if (b > t.b0) add_values(mul);  // (the block before, while the scores were on their way)
                put_weights(which);
                lb_tc_fence_before();
                __syncwarp();
                if (lane == 0) lb_mbar_arrive(&s_bar[3]);
                float old = 1.f;
                mul = 0.f;
                if (any) {
                    const float both = top > m + kRwLag ? top : m;
                    old = m == both ? 1.f : exp2_of(m - both);
                    const float now = exp2_of(top - both) * (1.f / kRwWeight);
                    l = fmaf(l, old, ((sum[0] + sum[1]) + (sum[2] + sum[3])) * now);
                    if (!(fabsf(kt) <= CUDART_MAX_NORMAL_F)) l = CUDART_NAN_F;
                    m = both;
                    mul = now * (1.f / 127.f) * vt;
                }
                rescale(old);
                kt = kt1;
                vt = vt1;
            }
            if (t.b0 < t.bend) add_values(mul);

            // ---- the open block ----
            if (t.open) {
                const int n_open = a.pos + a.count - closed * kKvBlock;
                const auto parts_in = [&](const float* rows, bool values, float* factors) {  // sixteen rows a warp, by pairs
#pragma unroll 1
                    for (int j0 = warp * 16; j0 < warp * 16 + 16; j0 += 4) {
                        float4 f[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) f[i] = four(rows + (size_t)(j0 + i) * c.dim_o, j0 + i < n_open, true);
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const int j = j0 + i;
                            uint2 part[2][2];  // [row][part]
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t bits = row_top(f[i + e]);
                                row_parts(f[i + e], bits, part[e]);
                                if (lane == 0) factors[j + e] = bits < 0x7f800000u ? row_factor(bits) : CUDART_NAN_F;
                            }
                            if (lane < DK / 4)
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    if (values) {  // dimensions 4 lane .. 4 lane + 3 of both rows
                                        const uint32_t w[4] = {__byte_perm(part[0][k].x, part[1][k].x, 0x5410), __byte_perm(part[0][k].x, part[1][k].x, 0x7632),
                                                               __byte_perm(part[0][k].y, part[1][k].y, 0x5410), __byte_perm(part[0][k].y, part[1][k].y, 0x7632)};
#pragma unroll
                                        for (int e = 0; e < 4; ++e) {
                                            const int d = 4 * lane + e;
                                            *reinterpret_cast<uint32_t*>(sk + k * S::kOpenV + ((2 * (j >> 1 & 3) + (j >> 5)) * (DK / 8) + (d >> 3)) * S::kOpenRows + (d & 7) * 16 + (j >> 3 & 3) * 4) = w[e];
                                        }
                                    } else {
#pragma unroll
                                        for (int e = 0; e < 2; ++e)
                                            *reinterpret_cast<uint2*>(sk + k * S::kOpenK + (lane >> 1) * S::kOpenCol + (j + e) * 16 + (lane & 1) * 8) = part[e][k];
                                    }
                                }
                        }
                    }
                };
                half_sync();  // (every thread's products are through)
                parts_in(c.open_row(c.k_open, t.s, t.h, closed * kKvBlock), false, s_ks);
                shared_written();
                lb_tc_fence_before();
                half_sync();
                lb_tc_fence_after();
                if (tid == 0) {
                    const uint64_t keys = lb_smem_desc(lb_smem_u32(sk), S::kOpenCol, 128);
                    mma_s(0, 1, keys, 2 * S::kOpenCol, false);
                    mma_s(0, 0, keys + (S::kOpenK >> 4), 2 * S::kOpenCol, true);
                    mma_s(0, 0, keys, 2 * S::kOpenCol, true);
                    lb_mma_commit(&s_bar[0]);
                }
                wait_for(0);
                half_sync();  // (for every thread: the keys have been read)
                parts_in(c.open_row(c.v_open, t.s, t.h, closed * kKvBlock), true, s_vs);
                shared_written();
                half_sync();
                load_scores(0);
                const int last = see - closed * kKvBlock;
                const bool any = last >= 0;
                const float cs = p.scale * qs;
                float top = -CUDART_INF_F;
#pragma unroll
                for (int i = 0; i < kKvBlock; ++i) {
                    sc[i] = i > last ? -CUDART_INF_F : sc[i] * (cs * s_ks[i]);
                    top = fmaxf(top, sc[i]);
                }
                top = any ? top : 0.f;
                float sum = 0.f, most_y = 0.f, odd = 0.f;
#pragma unroll
                for (int i = 0; i < kKvBlock; ++i) {
                    const float w = exp2_of(sc[i] - top);
                    sum += w;
                    sc[i] = i <= last ? w * s_vs[i] : 0.f;
                    most_y = fmaxf(most_y, sc[i]);
                    odd += sc[i] * 0.f;  // (not a number, from one)
                }
                // (from 2^-112 down the weights get smaller with the values: a larger factor would overflow)
                most_y = fmaxf(most_y, 0x1p-112f);
                const float inv = __fdiv_rn(kRwWeight, most_y);
#pragma unroll
                for (int i = 0; i < kKvBlock; ++i) sc[i] *= inv;
                put_weights(0);
                lb_tc_fence_before();
                half_sync();
                lb_tc_fence_after();
                if (tid == 0) {
                    constexpr int kCol = DK / 8 * S::kOpenRows;
                    const uint64_t values = lb_smem_desc(lb_smem_u32(sk), kCol, S::kOpenRows);
                    mma_o(0, 1, values, 2 * kCol, false);
                    mma_o(0, 0, values + (S::kOpenV >> 4), 2 * kCol, true);
                    mma_o(0, 0, values, 2 * kCol, true);
                    lb_mma_commit(&s_bar[2]);
                }
                float old = 1.f;
                mul = 0.f;
                if (any) {
                    const float both = top > m + kRwLag ? top : m;
                    old = m == both ? 1.f : exp2_of(m - both);
                    const float now = exp2_of(top - both);
                    l = fmaf(l, old, sum * now);
                    m = both;
                    mul = now * (1.f / kRwWeight) * most_y + odd;
                }
                rescale(old);
                add_values(mul);
            }

            // ---- the parts together, by twos: the CTA that comes second takes both on; the operands' order is that of the parts ----
            bool mine = true;
#pragma unroll 1
            for (int level = 0; mine && 1 << level < t.cuts; ++level) {
                const int half = 1 << level, right = (t.cut >> (level + 1) << (level + 1)) + half;  // the right one's first part
                if (right >= t.cuts) continue;
                unsigned* cnt = p.cnt + (n - t.cut + right);
                const bool is_right = (t.cut & half) != 0;
                const auto slot = [&](int part) { return p.part + (size_t)(n - t.cut + part) * S::kPart; };
                if (tid == 0) s_last = __ldcg(cnt) != 0;  // (and then for good)
                half_sync();
                if (!s_last) {
                    float* to = slot(is_right ? right : right - half);
                    if (tid < nr) {
#pragma unroll
                        for (int d = 0; d < DK; d += 4) __stcg(reinterpret_cast<float4*>(to + (size_t)d * kRwTile) + tid, make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]));
                        __stcg(to + DK * kRwTile + tid, m);
                        __stcg(to + (DK + 1) * kRwTile + tid, l);
                    }
                    __threadfence();
                    half_sync();
                    if (tid == 0) s_last = atomicAdd(cnt, 1u) != 0;
                    half_sync();
                }
                mine = s_last != 0;
                half_sync();
                if (!mine) break;
                __threadfence();
                if (tid == 0) *cnt = 0;
                if (tid >= nr) continue;
                const float* from = slot(is_right ? right - half : right);
                const float m1 = __ldcg(from + DK * kRwTile + tid), l1 = __ldcg(from + (DK + 1) * kRwTile + tid), both = fmaxf(m, m1);
                const float f = m == -CUDART_INF_F ? 0.f : exp2_of(m - both), f1 = m1 == -CUDART_INF_F ? 0.f : exp2_of(m1 - both);
                const auto join = [&](float own, float other) { return is_right ? fmaf(other, f1, own * f) : fmaf(own, f, other * f1); };
                m = both;
                l = join(l, l1);
#pragma unroll
                for (int d0 = 0; d0 < DK; d0 += 32) {
                    float4 x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = __ldcg(reinterpret_cast<const float4*>(from + (size_t)(d0 + 4 * i) * kRwTile) + tid);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        o[d0 + 4 * i] = join(o[d0 + 4 * i], x[i].x);
                        o[d0 + 4 * i + 1] = join(o[d0 + 4 * i + 1], x[i].y);
                        o[d0 + 4 * i + 2] = join(o[d0 + 4 * i + 2], x[i].z);
                        o[d0 + 4 * i + 3] = join(o[d0 + 4 * i + 3], x[i].w);
                    }
                }
            }
            if (mine && tid < nr) {
                const bool o_wide = (hd & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
                float* to = p.out + row_at(t, tid, (long long)p.q_heads * hd);
                const float inv = __fdiv_rn(1.f, l);
#pragma unroll
                for (int d = 0; d < DK; d += 4) {
                    if (o_wide) {
                        if (d < hd) *reinterpret_cast<float4*>(to + d) = make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (d + e < hd) to[d + e] = o[d + e] * inv;
                    }
                }
            }
            lb_tc_fence_before();
            __syncthreads();
            lb_tc_fence_after();
        }
    }
    __syncthreads();
    if (warp == 0) lb_tmem_dealloc(tmem, kRwCols);
}
