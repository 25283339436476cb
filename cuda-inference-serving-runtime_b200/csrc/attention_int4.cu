// Attention over a cache held in 4 bits (int4_cache.cuh): a few new tokens per request (one in a decode step), all query heads of a
// key head at once, key ranges in parallel, the weights of the keys added up where that is asked for.
// Specialised by HEAD_DIM (32, 64, 96, 128) and the queries' type (STORAGE_BF16).
//
// With codes n = c + 8, steps s and t the place of a key, of one query row q:
//   score   scale log2(e) sum_g s_g(t) (sum_{d in g} q_d n_d - 8 sum_{d in g} q_d)          groups g of 32 dimensions
//   output  sum_t p_t s_g(t) n_d(t) - 8 sum_t p_t s_g(t),     p = 2^(score - max), divided by sum_t p_t
// The cache is read once, 9 D / 8 bytes a key for both planes, 3.6 times less than in bfloat16; at the rate of memory that is some 44 values a
// clock and SM, so what has to be small here is the number of instructions per value:
//   * A code is a float16 operand by one mask: the low half byte of a 16-bit half is the subnormal n 2^-24, the next one n 2^-20, which
//     the matrix instructions take exactly; the two upper half bytes follow after one shift by 8.  Five integer instructions for
//     8 values, none of them a conversion.  The factor 16 is taken out of the query (exactly) or of the finished output.
//   * The offset 8 is never subtracted from a code: a score's share, -8 sum_g s_g sum q, is the product of a key's steps with the queries'
//     sums (two float16 terms), the output's share the product of the probabilities with a constant operand: one matrix instruction per
//     16 keys, and one per group of them.
//   * A is the cache (16 keys by 16 dimensions of K; 16 dimensions by 16 keys of V), B the queries or probabilities, of which 8 columns are
//     the least there is: a group of 3 or 4 query heads fills half of them, where it as A would fill a quarter.
//   * Steps of K are applied to the score of a group (float), those of V to the probabilities (float16 pairs).
// Operands other than codes are float16: of queries, normed by a power of two per row, exactly what bfloat16 holds (elements below 2^-24 of
// the row's largest lose digits); of probabilities 11 bits.  Float queries take two float16 terms (22 bits) for both.
// Scores, running maxima, sums and outputs are float.
//
// What bounds it: with many long requests no unit alone, but each warp's chain of products, exponentials, transpositions and products, of which
// 128 registers a thread leave four to a scheduler: 64 requests of 4000 to 8000 rows, 32 heads over 8 of 128, 97 us where memory takes 68 and
// the instructions (219 per 16 keys and warp at head size 128 and up to 8 rows) 37; counters: DRAM 56 %, issue slots 52 %, tensor pipe 36 %.  Float
// queries, whose products are two, take twice as long.  Several tokens, in tiles of 24 rows, have 255 registers and two warps to a scheduler (DRAM 11 %,
// issue 32 %, tensor pipe 16 %).  With few or short requests it is the way from one trip to memory to the next, some 5 us of a block
// (one request of 700 rows 8 to 10 us, of 8000 12).  Besides (us, 32 heads over 8 of 128): 32 x 4000 rows 38 (memory 22), 48 x 3000 41 (25), 64 x 500 16 (6);
// five tokens each of 8 requests of 3000 rows 24.
#include <climits>

#include "int4_cache.cuh"

#ifndef HEAD_DIM
#define HEAD_DIM 128
#endif
#ifndef STORAGE_BF16
#define STORAGE_BF16 1
#endif

namespace {
constexpr int D = HEAD_DIM, NG = D / 32;
static_assert(D % 32 == 0 && D >= 32 && D <= 128, "head sizes of whole groups up to 128");
#if STORAGE_BF16
typedef __nv_bfloat16 T;
constexpr int TERMS = 1;
#else
typedef float T;
constexpr int TERMS = 2;
#endif
// Keys of a warp's tile.  A warp has one tile in shared memory, its keys and its values apart: the next tile's keys are on their way while this
// one's values are worked on, and the other way round.
template <int NT> constexpr int tile_keys() { return NT == 1 ? 64 : 32; }
constexpr int BLOCK_BYTES = int4_block_bytes(D);
constexpr float LOG2E = 1.4426950408889634f;
// The running maximum follows a score only where that is 2^SLACK times its weight above it, which after a warp's first tile is rare (each time
// costs 50 multiplications a lane).  Probabilities are held times 2^9: with steps of V below 8 (values below 56) no product of the two overflows
// a float16, and products down to 2^-23 keep all their digits (smaller ones are off by 2^-34 at most).  A warp whose sums come out not finite
// does its keys again with bfloat16 operands, which no step can overflow: codes, which they hold exactly, and products of a probability and a
// step, made in float, as two terms (16 digits; for float queries three, 24).  So it does not matter to a small group that another one is large.
// (32 requests of 4000 rows, all of whose values are large: 90 us instead of 36; with float16 and weights times 2^-5, which took 61, groups beside a large
// one came out up to 2e-3 off.  Looking at every step instead took 8 instructions per 16 keys.)
constexpr float SLACK = 4.f, SHIFT = 9.f;
constexpr int MAX_CLUSTER = 8;                                     // thread blocks of a portable cluster
constexpr int MAX_RANKED = 128;                                    // requests that are put in order of length, a thread each

// Thread blocks of four warps, and for bfloat16 queries of up to 8 rows also of eight (`Shape` chooses); blocks of an SM by a warp's registers.
constexpr int MOST_WARPS = TERMS == 1 ? 8 : 4;
template <int NT, int WARPS> constexpr int blocks_of() { return NT == 1 ? (TERMS == 1 ? 16 / WARPS : 3) : 2; }

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same without sums from before, and with 8 of K.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_8_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {        // of an 8 x 8 matrix of 16-bit elements spread over a warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Two codes n, subnormals n 2^-24 (EXPONENT 15) or n 2^-20 (11), as (n - 8) 2^-9: exact, in one instruction.
template <int EXPONENT> __device__ __forceinline__ uint32_t centred(uint32_t n) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&n), __float2half2_rn((float)(1 << EXPONENT)), __float2half2_rn(-8.f / 512.f));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Two codes n, one in each half's low four bits, as bfloat16 (n - 8) 2^-DOWN: 128 + n is one by its bits, and the rest is exact, in one instruction.
template <int DOWN> __device__ __forceinline__ uint32_t centred_bf16(uint32_t n) {
    const uint32_t x = n | 0x43004300u;
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(1.f / (1 << DOWN)), __float2bfloat162_rn(-136.f / (1 << DOWN)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float low_half(uint32_t x) { return __half2float(__ushort_as_half((unsigned short)(x & 0xffff))); }
__device__ __forceinline__ float high_half(uint32_t x) { return __half2float(__ushort_as_half((unsigned short)(x >> 16))); }

template <int N> struct Share { uint32_t w[(N + 3) / 4]; };         // N neighbouring bytes of shared memory, as wide as they are aligned
template <int N> __device__ __forceinline__ Share<N> load_share(const unsigned char* p) {
    Share<N> s;
    if constexpr (N == 16) { const uint4 v = *reinterpret_cast<const uint4*>(p); s.w[0] = v.x; s.w[1] = v.y; s.w[2] = v.z; s.w[3] = v.w; }
    else if constexpr (N == 8) { const uint2 v = *reinterpret_cast<const uint2*>(p); s.w[0] = v.x; s.w[1] = v.y; }
    else if constexpr (N % 4 == 0) { for (int i = 0; i < N / 4; ++i) s.w[i] = reinterpret_cast<const uint32_t*>(p)[i]; }
    else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
        for (int i = 0; i < N / 2; i += 2) s.w[i / 2] = h[i] | (i + 1 < N / 2 ? (uint32_t)h[i + 1] << 16 : 0u);
    }
    return s;
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {      // zeros where it is not there
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

struct Args {
    const T* q; T* out;
    const unsigned char* k_cache; const unsigned char* v_cache;
    const int* req_slot; const int* table; int width;
    const int* q_start; const int* q_len; const int* ctx_len;
    float* partial;      // [tile][kv head][row][split][D], where the splits are not one cluster
    float* stats;        // [tile][kv head][row][split or 1][2]: largest score (base 2, less the shift), sum; null where no other kernel wants them
    float* scores;       // [tile][kv head][longest][row_stride], base 2, or null
    float* mass;         // added to by this kernel itself, or null
    int max_queries, tiles, row_stride, n_splits, cluster, longest;
    int hq, hkv, page_size, window, keep_first;
    Divider by_page, by_group, by_tiles, by_heads;
    int group, n_req, ranked, rank_threads;       // rank_threads: a power of two of n_req or more
    float scale, sink_all; const float* sink_heads;
    int* error;
};

// What the rows of one (request, tile of 8 NT query rows) see, as tiles of TK keys: those of the first keys that stay in sight behind a
// window, then those from the first key inside the first row's window to the last row's own.  They are walked from the `lead`th on, the
// others last: then the tiles that some row does not see whole are the last ones, and the first `plain` need no masks.
template <int TK> struct Span {
    int req, n, ctx, slot, tok0, group, row0, rows, first_pos, last_pos;
    int kept_tiles, window_base, tiles, lead, plain;
    __device__ __forceinline__ int key(int t) const {
        t += lead;
        t -= t >= tiles ? tiles : 0;
        return t < kept_tiles ? t * TK : window_base + (t - kept_tiles) * TK;
    }
};
template <int ROWS, int TK> __device__ __forceinline__ bool find_span(Span<TK>& s, const Args& a, int x) {
    static_assert(TK - 1 + ROWS - 1 < 2 * TK, "with one query head per key head a tile's rows are as many tokens, whose windows begin in two tiles of keys");
    s.req = a.by_tiles(x);
    const int tile = x - s.req * a.tiles;
    s.n = a.q_len[s.req]; s.ctx = a.ctx_len[s.req]; s.slot = a.req_slot[s.req]; s.tok0 = a.q_start[s.req];      // one trip to memory
    s.group = a.group; s.row0 = tile * ROWS;
    s.rows = min(ROWS, s.n * s.group - s.row0);
    if (s.n > a.max_queries || s.rows <= 0) return false;           // another kernel's request, or no such tile
    if (s.ctx > a.longest) {                                        // more rows than the scratch was made for
        if (threadIdx.x == 0) atomicExch(a.error, 6);
        return false;
    }
    s.first_pos = s.ctx - s.n + a.by_group(s.row0);
    s.last_pos = s.ctx - s.n + a.by_group(s.row0 + s.rows - 1);
    s.kept_tiles = 0; s.window_base = 0;
    const int begin = s.first_pos - a.window + 1;
    if (a.window > 0 && begin >= TK) {
        s.kept_tiles = min((min(a.keep_first, begin) + TK - 1) / TK, begin / TK);
        s.window_base = begin & ~(TK - 1);
    }
    s.tiles = s.last_pos < 0 ? 0 : s.kept_tiles + (s.last_pos - s.window_base) / TK + 1;
    s.lead = a.window > 0 && s.last_pos >= a.window ? min(s.tiles, s.kept_tiles + 2) : 0;      // the rows' windows begin within ROWS keys
    s.plain = min(s.tiles - s.lead, max(0, s.first_pos + 1 < s.window_base ? 0 : (s.first_pos + 1 - s.window_base) / TK + s.kept_tiles - s.lead));
    return true;
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ float load_cluster(const float* p, uint32_t rank) {      // of another thread block's shared memory
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A part of a row's keys joins the others: sums, largest score and denominator.  A part without a largest score has no keys in sight, or
// scores that are not numbers, of which its denominator tells.
struct Joined {
    float m = -INFINITY, num = 0.f, den = 0.f;
    __device__ __forceinline__ float weight(float part_m) const { return part_m == -INFINITY ? 0.f : exp2_fast(part_m - m); }
    __device__ __forceinline__ void add(float part_m, float part_num, float part_den) {
        if (part_m != -INFINITY) {
            const float w = weight(part_m);
            num = fmaf(w, part_num, num);
            den = fmaf(w, part_den, den);
        } else if (!(part_den == 0.f)) {
            den = NAN;
        }
    }
    // with the sink: one more term of the denominator, no value
    __device__ __forceinline__ float whole(float sink) const { return sink > -INFINITY ? den + exp2f(fmaf(sink, LOG2E, -m)) : den; }
    // the logarithm (base 2) of that, by which a score becomes a weight; of a row that sees nothing one by which every weight is 0
    __device__ __forceinline__ float logarithm(float sink) const { return den == 0.f ? INFINITY : m + log2f(whole(sink)); }
};

// NT: columns of 8 query rows.  Where there are two or three, or float queries, codes serve two matrix instructions, and the offset is
// subtracted from them (and the subnormals made normal) by one instruction for two.  The matrix instructions align their
// products by the operands' exponent fields, so that a sum over subnormals keeps some 2^-18 of its largest term only: far below the
// rounding of a bfloat16 output, but not of a float one.
template <int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, blocks_of<NT, WARPS>()) attn_int4_kernel(const __grid_constant__ Args a) {
    constexpr int ROWS = 8 * NT, THREADS = 32 * WARPS;
    constexpr bool OFFSET = NT == 1 && TERMS == 1;       // the offset as a product with a constant
    constexpr bool Q_SHARED = NT > 2;                    // the queries' operands stay in shared memory
    constexpr float SECOND = OFFSET ? 0.0625f : 1.f;     // of operands that meet codes n 2^-20
    constexpr int MERGE_STRIDE = D + 4;                  // rows of whole 16 bytes
    constexpr int TK = tile_keys<NT>(), HALVES = TK / 16, PLANE_BYTES = TK / INT4_BLOCK * BLOCK_BYTES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float others[MAX_CLUSTER][ROWS][2], lse[ROWS];       // a cluster's largest scores and denominators; the row's logarithm of its sum
    __shared__ float weight[WARPS][ROWS];                           // of a warp's sums among the block's
    __shared__ __align__(16) float sums[ROWS * MERGE_STRIDE];                     // this block's, for its cluster
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    // The key heads of a request's tile of rows are neighbours in the order of thread blocks (a page's heads lie side by side), and where
    // not all blocks run at once the longest requests come first, so that the last blocks to end are short ones: 64 requests of 4000 to
    // 8000 rows 96 us, in the order of requests 111.
    const int split = blockIdx.z, id = blockIdx.x + gridDim.x * blockIdx.y;
    int unit_of = a.by_heads(id);
    const int kvh = id - unit_of * a.hkv;
    pdl_trigger();
    // Lengths, places in q and the table are older than the kernel before this one (which brings queries and rows): they are read beside its end.
    if (a.ranked) {
        __shared__ int lens[MAX_RANKED], before[MAX_RANKED], chosen;
        for (int i = tid; i < a.n_req; i += THREADS) { lens[i] = a.ctx_len[i]; before[i] = 0; }
        __syncthreads();
        const int rank = a.by_tiles(unit_of), threads_each = THREADS / a.rank_threads, i = tid & (a.rank_threads - 1);
        if (i < a.n_req) {                                          // how many come before request i, counted by several threads
            const int mine = lens[i];
            int n = 0;
            for (int j = tid / a.rank_threads; j < a.n_req; j += threads_each) n += lens[j] > mine || (lens[j] == mine && j < i);
            if (n) atomicAdd(&before[i], n);
        }
        __syncthreads();
        if (tid < a.n_req && before[tid] == rank) chosen = tid;
        __syncthreads();
        unit_of += (chosen - rank) * a.tiles;
    }
    Span<TK> span;
    if (!find_span<ROWS>(span, a, unit_of)) return pdl_wait();      // the same for a whole cluster
    const size_t base_row = ((size_t)unit_of * a.hkv + kvh) * a.row_stride;
    const int* pages = a.table + (size_t)span.slot * a.width;
    const int tok0 = span.tok0;
    const int share = (span.tiles + a.n_splits - 1) / a.n_splits;   // tiles of a split: the request's own, so that a cluster ends together
    const int t0 = split * share, n_tiles = max(0, min(share, span.tiles - t0));

    unsigned char* ks = smem + (size_t)warp * 2 * PLANE_BYTES;
    unsigned char* vs = ks + PLANE_BYTES;
    // A tile's keys or values: 16 bytes a lane at a time, some lanes a block.  (A bulk copy per page took less address arithmetic but a loop
    // of some 15 instructions for each copy.)  Its page is looked up one tile ahead.  Blocks behind the last key and pages that are
    // not there become zeros.
    constexpr int CHUNKS = BLOCK_BYTES / 16, LANES = 32 / (TK / INT4_BLOCK);
    const uint32_t page_chunks = (uint32_t)(a.hkv * (a.page_size / INT4_BLOCK) * CHUNKS);
    const size_t lane_bytes = (size_t)kvh * (a.page_size / INT4_BLOCK) * BLOCK_BYTES + (lane % LANES) * 16;
    const uint32_t landing = (uint32_t)__cvta_generic_to_shared(ks) + (lane / LANES) * BLOCK_BYTES + (lane % LANES) * 16;
    const auto look_up = [&](int t) {                               // the block's place in a plane, in 16 bytes, or all ones
        const int pos = span.key(t0 + t) + (lane / LANES) * INT4_BLOCK, logical = a.by_page(pos);
        const int page = t < n_tiles && pos <= span.last_pos && logical < a.width ? pages[logical] : -1;
        return page < 0 ? ~0u : page * page_chunks + (pos - logical * a.page_size) / INT4_BLOCK * CHUNKS;
    };
    const auto fetch = [&](const unsigned char* plane, uint32_t to, uint32_t found, bool any) {
        if (any) {
            const bool there = found != ~0u;
            const unsigned char* from = plane + lane_bytes + (there ? (size_t)found * 16 : 0);
#pragma unroll
            for (int i = 0; i < CHUNKS; i += LANES)
                if (i + LANES <= CHUNKS || i + lane % LANES < CHUNKS) copy16(to + i * 16, from + i * 16, there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t here, next;                                            // of this tile, of the next one
    here = look_up(warp); next = look_up(warp + WARPS);             // on their way at once
    pdl_wait();
    const auto begin = [&] {
        fetch(a.k_cache, landing, here, warp < n_tiles);
        fetch(a.v_cache, landing + PLANE_BYTES, here, warp < n_tiles);
    };

    // Queries as B: lane (g, c) has dimensions 32 j + 8 c + 0 .. 7 of row g, in the order of the half bytes: pairs (0, 4), (1, 5) / 16 and,
    // after the shift, (2, 6), (3, 7) / 16.  All warps need the same: each makes some groups' operands and they exchange them.
    constexpr int TURNS = (NT * NG + WARPS - 1) / WARPS;
    __shared__ uint4 operand[NT * NG][TERMS][32];
    __shared__ uint32_t largest[ROWS][NG];
    __shared__ float group_sum[ROWS][NG];
    uint4 raw[TURNS][TERMS];                                        // asked for before the first tiles' look-ups are waited for
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
        const int i = min(warp + turn * WARPS, NT * NG - 1), nt = i / NG, j = i - nt * NG, r = nt * 8 + g;
        const int row = span.row0 + (r < span.rows ? r : 0), token = a.by_group(row);
        const T* q = a.q + ((size_t)(tok0 + token) * a.hq + kvh * span.group + row - token * span.group) * D + 32 * j + 8 * c;
#pragma unroll
        for (int i = 0; i < TERMS; ++i) raw[turn][i] = reinterpret_cast<const uint4*>(q)[i];
    }
    begin();
    float x[TURNS][8];
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
        const int i = warp + turn * WARPS, nt = i / NG, j = i - nt * NG, r = nt * 8 + g;
        if (i >= NT * NG) continue;
        const bool there = r < span.rows;
#pragma unroll
        for (int i = 0; i < TERMS; ++i) {
            const uint32_t w[4] = {raw[turn][i].x, raw[turn][i].y, raw[turn][i].z, raw[turn][i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#if STORAGE_BF16
                x[turn][2 * e] = __uint_as_float(w[e] << 16); x[turn][2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
#else
                x[turn][4 * i + e] = __uint_as_float(w[e]);
#endif
            }
        }
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!there) x[turn][e] = 0.f;
            top = max(top, __float_as_uint(x[turn][e]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (c == 0) largest[r][j] = top;
    }
    __syncthreads();
    const auto exponent = [&](int r) {                              // the row times 2 to it is below 2^15
        uint32_t top = largest[r][0];
#pragma unroll
        for (int j = 1; j < NG; ++j) top = max(top, largest[r][j]);
        return min(14 - ((int)(top >> 23) - 127), 120);
    };
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
        const int i = warp + turn * WARPS, nt = i / NG, j = i - nt * NG, r = nt * 8 + g;
        if (i >= NT * NG) continue;
        const float factor = copysignf(__uint_as_float((uint32_t)(exponent(r) + 127) << 23), a.scale);
        float sum = 0.f;
        uint32_t w[TERMS][4];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float p0 = x[turn][2 * k + h] * factor * (h ? SECOND : 1.f), p1 = x[turn][2 * k + h + 4] * factor * (h ? SECOND : 1.f);
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    w[term][2 * k + h] = pack_f16(p0, p1);
                    const float lo = low_half(w[term][2 * k + h]), hi = high_half(w[term][2 * k + h]);
                    sum += (h ? 1.f / SECOND : 1.f) * (lo + hi);
                    p0 -= lo; p1 -= hi;
                }
            }
#pragma unroll
        for (int term = 0; term < TERMS; ++term) operand[i][term][lane] = make_uint4(w[term][0], w[term][1], w[term][2], w[term][3]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (c == 0) group_sum[r][j] = sum;
    }
    __syncthreads();
    uint4 qf[Q_SHARED ? 1 : NT][NG][TERMS];
    uint32_t qs[NT];                                                // -8 2^-24 sum q of two groups, the first float16 term (c below 2) or the second
    float unit[NT][2];                                              // of a column's sums, in the softmax's exponent (base 2); positive
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int term = 0; term < TERMS; ++term)
                if constexpr (!Q_SHARED) qf[nt][j][term] = operand[nt * NG + j][term][lane];
        if constexpr (OFFSET) {
            const int j0 = 2 * (c & 1);
            const float s0 = j0 < NG ? -0x1p-21f * group_sum[nt * 8 + g][j0 < NG ? j0 : 0] : 0.f, s1 = j0 + 1 < NG ? -0x1p-21f * group_sum[nt * 8 + g][j0 + 1 < NG ? j0 + 1 : 0] : 0.f;
            qs[nt] = pack_f16(s0, s1);
            if (c >= 2) qs[nt] = pack_f16(s0 - low_half(qs[nt]), s1 - high_half(qs[nt]));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            unit[nt][h] = fmaxf(fabsf(a.scale) * LOG2E * (OFFSET ? 0x1p24f : 0x1p9f) * __uint_as_float((uint32_t)(127 - exponent(nt * 8 + 2 * c + h)) << 23), 0x1p-126f);
    }
    float o[D / 16][NT][4], r_off[OFFSET ? NG : 1][NT][4], m_run[NT][2], l_run[NT][2];
    float limit[NT][2];                                             // scores above it move the maximum
    int own_pos[NT][2];                                             // a column's place, for tiles with masks
    uint32_t eights[4];                                             // the constant operand, kept in registers: as an immediate it was loaded again for every product
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, 0x00080008;" : "=r"(eights[i]));
    // alpha of column h into everything that is summed
    const auto rescale = [&](int nt, float a0, float a1) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) { o[i][nt][0] *= a0; o[i][nt][1] *= a1; o[i][nt][2] *= a0; o[i][nt][3] *= a1; }
        if constexpr (OFFSET) {
#pragma unroll
            for (int i = 0; i < NG; ++i) { r_off[i][nt][0] *= a0; r_off[i][nt][1] *= a1; r_off[i][nt][2] *= a0; r_off[i][nt][3] *= a1; }
        }
        l_run[nt][0] *= a0; l_run[nt][1] *= a1;
    };

    float* scores = a.scores ? a.scores + ((size_t)unit_of * a.hkv + kvh) * a.longest * a.row_stride : nullptr;
    // A tile: scores, running maxima, sums.  EDGE: some row does not see some of its keys.  LARGE: 16 keys of one that is there (the `part`th),
    // with products with steps as bfloat16.  (A whole tile of them was so much code that a captured step of 30 layers took 18 us more, although it
    // never ran.)
    const auto step = [&](auto is_edge, auto is_large, int t, int part) {
        constexpr bool EDGE = decltype(is_edge)::value, LARGE = decltype(is_large)::value;
        constexpr int PARTS = LARGE ? TERMS + 1 : TERMS;
        constexpr bool HALVES_PRODUCT = TERMS == 1 && !LARGE;       // of probability and step, in float16
        constexpr int COUNT = LARGE ? 1 : HALVES;
        const int k0 = span.key(t0 + t) + 16 * part;
        const unsigned char *keys = ks + 2 * part * BLOCK_BYTES, *values = vs + 2 * part * BLOCK_BYTES;
        float s[COUNT][NT][4];
        if constexpr (!LARGE) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");    // the keys
            __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < COUNT; ++h) {                           // 16 keys: blocks 2 h and 2 h + 1
            const unsigned char* b0 = keys + 2 * h * BLOCK_BYTES;
            const unsigned char* b1 = b0 + BLOCK_BYTES;
            const Share<4 * NG> w0 = load_share<4 * NG>(b0 + g * (D / 2) + c * 4 * NG), w1 = load_share<4 * NG>(b1 + g * (D / 2) + c * 4 * NG);
            const Share<2 * NG> s0 = load_share<2 * NG>(b0 + 4 * D + g * 2 * NG), s1 = load_share<2 * NG>(b1 + 4 * D + g * 2 * NG);
            if constexpr (OFFSET) {
                const uint32_t a0 = c & 1 ? (NG > 2 ? s0.w[(NG - 1) / 2] : 0u) : s0.w[0], a1 = c & 1 ? (NG > 2 ? s1.w[(NG - 1) / 2] : 0u) : s1.w[0];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_8_new(s[h][nt], a0, a1, qs[nt]);
            }
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                float acc[NT][4];
                uint4 query[NT][TERMS];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) query[nt][term] = Q_SHARED ? operand[nt * NG + j][term][lane] : qf[Q_SHARED ? 0 : nt][j][term];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t x = k ? w0.w[j] >> 8 : w0.w[j], y = k ? w1.w[j] >> 8 : w1.w[j];
                    uint32_t a0 = x & 0x000f000fu, a1 = y & 0x000f000fu, a2 = x & 0x00f000f0u, a3 = y & 0x00f000f0u;
                    if constexpr (!OFFSET) { a0 = centred<15>(a0); a1 = centred<15>(a1); a2 = centred<11>(a2); a3 = centred<11>(a3); }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int term = 0; term < TERMS; ++term) {
                            const uint4& q = query[nt][term];
                            if (k || term) mma_f16(acc[nt], a0, a1, a2, a3, k ? q.z : q.x, k ? q.w : q.y);
                            else mma_f16_new(acc[nt], a0, a1, a2, a3, q.x, q.y);
                        }
                }
                const float f0 = j & 1 ? high_half(s0.w[j / 2]) : low_half(s0.w[j / 2]), f1 = j & 1 ? high_half(s1.w[j / 2]) : low_half(s1.w[j / 2]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[h][nt][e] = OFFSET || j ? fmaf(e < 2 ? f0 : f1, acc[nt][e], s[h][nt][e]) : (e < 2 ? f0 : f1) * acc[nt][e];
            }
        }
        const bool again = t + WARPS < n_tiles;
        if constexpr (!LARGE) {
            __syncwarp();                                           // every lane has read the keys
            fetch(a.k_cache, landing, next, again);
        }
        bool more = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < COUNT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (EDGE) {
                        const int key = k0 + 16 * h + g + 8 * (e >> 1), pos = own_pos[nt][e & 1];
                        const bool seen = key <= pos && (a.window <= 0 || pos - key < a.window || key < a.keep_first);
                        if (!seen) s[h][nt][e] = -INFINITY;
                    }
                    more |= s[h][nt][e] > limit[nt][e & 1];
                }
        if (!LARGE && scores) {
#pragma unroll
            for (int h = 0; h < COUNT; ++h)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const int key = k0 + 16 * h + g + 8 * (e >> 1), col = nt * 8 + 2 * c;
                        if (key <= span.last_pos && col < span.rows)
                            *reinterpret_cast<float2*>(scores + (size_t)key * a.row_stride + col) = make_float2(s[h][nt][e] * unit[nt][0], s[h][nt][e + 1] * unit[nt][1]);
                    }
        }
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float alpha[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = s[0][nt][e];
#pragma unroll
                    for (int h = 0; h < COUNT; ++h) mx = fmaxf(mx, fmaxf(s[h][nt][e], s[h][nt][e + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float m_new = fmaxf(m_run[nt][e], mx);
                    alpha[e] = m_run[nt][e] == m_new ? 1.f : exp2_fast((m_run[nt][e] - m_new) * unit[nt][e]);
                    m_run[nt][e] = m_new;
                    limit[nt][e] = m_new + SLACK / unit[nt][e];
                }
                rescale(nt, alpha[0], alpha[1]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float top = SHIFT - (m_run[nt][e] == -INFINITY ? 0.f : m_run[nt][e] * unit[nt][e]);
#pragma unroll
                for (int h = 0; h < COUNT; ++h) {
                    float p0 = exp2_fast(fmaf(s[h][nt][e], unit[nt][e], top)), p1 = exp2_fast(fmaf(s[h][nt][e + 2], unit[nt][e], top));
                    l_run[nt][e] += p0 + p1;
                    if constexpr (EDGE) {                                     // a key out of sight gets -0, by which it is told from one of no weight
                        if (s[h][nt][e] == -INFINITY) p0 = -0.f;
                        if (s[h][nt][e + 2] == -INFINITY) p1 = -0.f;
                    }
                    s[h][nt][e] = p0; s[h][nt][e + 2] = p1;
                }
            }
        if constexpr (!LARGE) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");    // the values
            __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < COUNT; ++h) {
            // probabilities as B: rows of the product above are keys, here columns: two 8 x 8 transpositions per 16 keys
            uint32_t pt[NT][2];
            if constexpr (HALVES_PRODUCT) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    pt[nt][0] = transposed(pack_f16(s[h][nt][0], s[h][nt][1]));
                    pt[nt][1] = transposed(pack_f16(s[h][nt][2], s[h][nt][3]));
                }
            }
            const unsigned char* b0 = values + 2 * h * BLOCK_BYTES;
            const unsigned char* b1 = b0 + BLOCK_BYTES;
            Share<4 * NG> sv[2];                                    // the steps of two neighbouring keys side by side
#pragma unroll
            for (int b = 0; b < 2; ++b) sv[b] = load_share<4 * NG>(values + (2 * h + b) * BLOCK_BYTES + 4 * D + c * 4 * NG);
            const int turned = (g ^ int4_value_turn<D>(c)) * 2 * NG;
            const Share<2 * NG> u0 = load_share<2 * NG>(b0 + c * (D / 2) + turned), u1 = load_share<2 * NG>(b0 + (4 + c) * (D / 2) + turned);
            const Share<2 * NG> u2 = load_share<2 * NG>(b1 + c * (D / 2) + turned), u3 = load_share<2 * NG>(b1 + (4 + c) * (D / 2) + turned);
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                // B of this group: probability times step, of two keys a register
                uint32_t pb[NT][PARTS][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if constexpr (HALVES_PRODUCT) {
                            uint32_t v = mul_f16x2(pt[nt][b], sv[b].w[j]);
                            if constexpr (EDGE) v &= ~__vcmpeq2(pt[nt][b], 0x80008000u);      // out of sight: nothing, whatever the step there is
                            pb[nt][0][b] = v;
                        } else {
                            // before the transposition a lane has keys of row g: its step is half of the word of the pair of rows g / 2
                            const uint32_t pair = __shfl_sync(0xffffffffu, sv[b].w[j], g >> 1);
                            const float step = g & 1 ? high_half(pair) : low_half(pair);
                            float v0 = s[h][nt][2 * b] * step, v1 = s[h][nt][2 * b + 1] * step;
                            if constexpr (EDGE) {
                                if (__float_as_uint(s[h][nt][2 * b]) == 0x80000000u) v0 = 0.f;
                                if (__float_as_uint(s[h][nt][2 * b + 1]) == 0x80000000u) v1 = 0.f;
                            }
#pragma unroll
                            for (int part = 0; part < PARTS; ++part) {
                                const uint32_t term = LARGE ? pack_bf16(v0, v1) : pack_f16(v0, v1);
                                pb[nt][part][b] = transposed(term);
                                v0 -= LARGE ? __uint_as_float(term << 16) : low_half(term);
                                v1 -= LARGE ? __uint_as_float(term & 0xffff0000u) : high_half(term);
                            }
                        }
                    }
                const uint32_t r0 = __byte_perm(u0.w[j / 2], u1.w[j / 2], j & 1 ? 0x7632 : 0x5410);      // keys 2 c and 2 c + 1 of the first block
                const uint32_t r1 = __byte_perm(u2.w[j / 2], u3.w[j / 2], j & 1 ? 0x7632 : 0x5410);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t x = k ? r0 >> 8 : r0, y = k ? r1 >> 8 : r1;
                    if constexpr (LARGE) {
                        constexpr int DOWN = OFFSET ? 24 : 9, SECOND_DOWN = OFFSET ? 20 : 9;      // the units of the usual sums
                        const uint32_t a0 = centred_bf16<DOWN>(x & 0x000f000fu), a1 = centred_bf16<SECOND_DOWN>((x >> 4) & 0x000f000fu), a2 = centred_bf16<DOWN>(y & 0x000f000fu),
                                       a3 = centred_bf16<SECOND_DOWN>((y >> 4) & 0x000f000fu);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int part = 0; part < PARTS; ++part) mma_bf16(o[2 * j + k][nt], a0, a1, a2, a3, pb[nt][part][0], pb[nt][part][1]);
                        continue;
                    }
                    uint32_t a0 = x & 0x000f000fu, a1 = x & 0x00f000f0u, a2 = y & 0x000f000fu, a3 = y & 0x00f000f0u;
                    if constexpr (!OFFSET) { a0 = centred<15>(a0); a1 = centred<11>(a1); a2 = centred<15>(a2); a3 = centred<11>(a3); }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int term = 0; term < TERMS; ++term) mma_f16(o[2 * j + k][nt], a0, a1, a2, a3, pb[nt][term][0], pb[nt][term][1]);
                }
                if constexpr (OFFSET && !LARGE) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int term = 0; term < TERMS; ++term)
                            mma_f16(r_off[j][nt], eights[0], eights[1], eights[2], eights[3], pb[nt][term][0], pb[nt][term][1]);
                }
            }
        }
        if constexpr (!LARGE) {
            __syncwarp();                                           // every lane has read the values
            here = next;
            fetch(a.v_cache, landing + PLANE_BYTES, here, again);
            next = look_up(t + 2 * WARPS);
        }
    };

    const auto clear = [&] {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
            for (int i = 0; i < (OFFSET ? NG : 1); ++i) r_off[i][nt][0] = r_off[i][nt][1] = r_off[i][nt][2] = r_off[i][nt][3] = 0.f;
            m_run[nt][0] = m_run[nt][1] = limit[nt][0] = limit[nt][1] = -INFINITY;
            l_run[nt][0] = l_run[nt][1] = 0.f;
        }
    };
    for (bool large = false;; large = true) {
        clear();
        if (large) {
            here = look_up(warp);
            for (int t = warp; t < n_tiles; t += WARPS) {
                next = look_up(t + WARPS);
                begin();
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                __syncwarp();
#pragma unroll 1
                for (int part = 0; part < HALVES; ++part) step(std::true_type(), std::true_type(), t, part);
                __syncwarp();
                here = next;
            }
            break;
        }
        int t = warp;
        for (const int plain = min(n_tiles, span.plain - t0); t < plain; t += WARPS) step(std::false_type(), std::false_type(), t, 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) own_pos[nt][h] = span.ctx - span.n + a.by_group(span.row0 + min(nt * 8 + 2 * c + h, span.rows - 1));
        for (; t < n_tiles; t += WARPS) step(std::true_type(), std::false_type(), t, 0);
        float all = 0.f;                                            // an overflow is in the sums of the constant operand too
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < (OFFSET ? NG : D / 16); ++i) {
                const float* v = OFFSET ? r_off[OFFSET ? i : 0][nt] : o[i][nt];
                all += (v[0] + v[1] + (OFFSET ? 0.f : v[2] + v[3])) * 0.f;
            }
        if (!__any_sync(0xffffffffu, all != 0.f)) break;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                                // every warp is done with its tiles: their place becomes the merge area
    float* merge = reinterpret_cast<float*>(smem);                  // [warp][ROWS][D + 2]: sums, largest score, denominator
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float l = l_run[nt][h];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            float* row = merge + ((size_t)warp * ROWS + nt * 8 + 2 * c + h) * MERGE_STRIDE;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const float off = OFFSET ? r_off[OFFSET ? j : 0][nt][h] : 0.f;
                constexpr float whole = OFFSET ? 0x1p24f : 0x1p9f;
                *reinterpret_cast<float4*>(row + 32 * j + 4 * g) =
                    make_float4((o[2 * j][nt][h] - off) * whole, (o[2 * j][nt][2 + h] * SECOND - off) * whole, (o[2 * j + 1][nt][h] - off) * whole,
                                (o[2 * j + 1][nt][2 + h] * SECOND - off) * whole);
            }
            if (g == 0) { row[D] = m_run[nt][h] == -INFINITY ? -INFINITY : fmaf(m_run[nt][h], unit[nt][h], -SHIFT); row[D + 1] = l; }
        }
    __syncthreads();
    // The warps' sums joined, in their order: into the first warp's place for the cluster, or to where they go.
    const bool alone = a.n_splits == 1, clustered = a.cluster > 1;
    const auto place = [&](int r) {                                 // of row r in q and out
        const int row = span.row0 + r, token = a.by_group(row);
        return ((size_t)(tok0 + token) * a.hq + kvh * span.group + row - token * span.group) * D;
    };
    const auto sink_of = [&](int r) { return a.sink_heads ? a.sink_heads[kvh * span.group + (span.row0 + r) % span.group] : a.sink_all; };
    if (tid < WARPS * ROWS) {
        const int w = tid / ROWS, r = tid - w * ROWS;
        Joined j;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) j.m = fmaxf(j.m, merge[((size_t)i * ROWS + r) * MERGE_STRIDE + D]);
        weight[w][r] = j.weight(merge[((size_t)w * ROWS + r) * MERGE_STRIDE + D]);
        if (w == 0) {
#pragma unroll
            for (int i = 0; i < WARPS; ++i) j.add(merge[((size_t)i * ROWS + r) * MERGE_STRIDE + D], 0.f, merge[((size_t)i * ROWS + r) * MERGE_STRIDE + D + 1]);
            sums[r * MERGE_STRIDE + D] = j.m; sums[r * MERGE_STRIDE + D + 1] = j.den;
            if (!clustered && r < span.rows) {
                if (a.stats) {
                    float* st = a.stats + ((base_row + r) * a.n_splits + split) * 2;
                    st[0] = j.m; st[1] = j.den;
                }
                lse[r] = j.logarithm(sink_of(r));
            }
        }
    }
    __syncthreads();
    for (int e = tid; e < span.rows * (D / 4); e += THREADS) {
        const int r = e / (D / 4), d = 4 * (e - r * (D / 4));
        float num[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(merge + ((size_t)w * ROWS + r) * MERGE_STRIDE + d);
            const float part = weight[w][r];
            num[0] = fmaf(part, v.x, num[0]); num[1] = fmaf(part, v.y, num[1]); num[2] = fmaf(part, v.z, num[2]); num[3] = fmaf(part, v.w, num[3]);
        }
        if (clustered) {
            *reinterpret_cast<float4*>(sums + r * MERGE_STRIDE + d) = make_float4(num[0], num[1], num[2], num[3]);
        } else if (alone) {
            Joined j;
            j.m = sums[r * MERGE_STRIDE + D]; j.den = sums[r * MERGE_STRIDE + D + 1];
            const float whole = j.whole(sink_of(r));
            T* to = a.out + place(r) + d;
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = from_float<T>(j.den == 0.f ? 0.f : num[i] / whole);
        } else {
            *reinterpret_cast<float4*>(a.partial + ((base_row + r) * a.n_splits + split) * D + d) = make_float4(num[0], num[1], num[2], num[3]);
        }
    }
    if (clustered) {
        // A thread block finishes a slice of the output's dimensions of every row, from all the others' sums.
        cluster_barrier();
        const int rank = (int)cluster_rank(), parts = a.cluster;
        for (int e = tid; e < 2 * span.rows * parts; e += THREADS) {
            const int p = e / (2 * span.rows), i = e - p * 2 * span.rows;
            others[p][i >> 1][i & 1] = load_cluster(sums + (i >> 1) * MERGE_STRIDE + D + (i & 1), (uint32_t)p);
        }
        __syncthreads();
        const int cols = (D + parts - 1) / parts;
        for (int e = tid; e < span.rows * cols; e += THREADS) {
            const int r = e / cols, d = rank * cols + e - r * cols;
            if (d >= D) continue;
            float v[MAX_CLUSTER];
#pragma unroll
            for (int p = 0; p < MAX_CLUSTER; ++p) v[p] = p < parts ? load_cluster(sums + r * MERGE_STRIDE + d, (uint32_t)p) : 0.f;
            Joined j;
#pragma unroll
            for (int p = 0; p < MAX_CLUSTER; ++p) if (p < parts) j.m = fmaxf(j.m, others[p][r][0]);
#pragma unroll
            for (int p = 0; p < MAX_CLUSTER; ++p) if (p < parts) j.add(others[p][r][0], v[p], others[p][r][1]);
            a.out[place(r) + d] = from_float<T>(j.den == 0.f ? 0.f : j.num / j.whole(sink_of(r)));
        }
        if (tid < span.rows) {
            Joined j;
            for (int p = 0; p < parts; ++p) j.m = fmaxf(j.m, others[p][tid][0]);
            for (int p = 0; p < parts; ++p) j.add(others[p][tid][0], 0.f, others[p][tid][1]);
            lse[tid] = j.logarithm(sink_of(tid));
            if (a.stats && rank == 0) {
                float* st = a.stats + (base_row + tid) * 2;
                st[0] = j.m; st[1] = j.den;
            }
        }
        cluster_barrier();                                          // nobody leaves while its sums may be read
    }
    // The weights of this block's keys, from the scores that it has just written: the rows in their order.
    if (a.mass) {
        __syncthreads();
        constexpr int AT_ONCE = 4;                                  // keys of a thread on their way together
        for (int i0 = tid; i0 < n_tiles * TK; i0 += AT_ONCE * THREADS) {
            float* to[AT_ONCE];
            float w[AT_ONCE];
            const float* score[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int i = i0 + u * THREADS, key = i < n_tiles * TK ? span.key(t0 + i / TK) + i % TK : INT_MAX;
                const bool there = key <= span.last_pos;
                const int logical = there ? a.by_page(key) : 0, at = there && logical < a.width ? pages[logical] : -1;
                to[u] = at < 0 ? nullptr : a.mass + ((size_t)at * a.hkv + kvh) * a.page_size + key - logical * a.page_size;
                score[u] = scores + (there ? (size_t)key * a.row_stride : 0);
                w[u] = 0.f;
            }
            for (int r = 0; r < span.rows; r += 2) {
                const float first = lse[r], second = lse[r + 1 < span.rows ? r + 1 : r];
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    if (!to[u]) continue;
                    const float2 v = *reinterpret_cast<const float2*>(score[u] + r);
                    w[u] += exp2_fast(v.x - first);
                    if (r + 1 < span.rows) w[u] += exp2_fast(v.y - second);
                }
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) if (to[u] && w[u] != 0.f) atomicAdd(to[u], w[u]);      // (requests may share a page)
        }
    }
}

// Splits of a row put together where they are no cluster: a thread per output dimension, the splits in their order.
template <int ROWS>
__global__ void __launch_bounds__(D) attn_int4_merge_kernel(const __grid_constant__ Args a) {
    pdl_wait();
    Span<32> span;                                                  // (of its tiles nothing is used here)
    if (!find_span<ROWS>(span, a, blockIdx.x)) return;
    const int r = blockIdx.z, kvh = blockIdx.y, d = threadIdx.x;
    if (r >= span.rows) return;
    const size_t base = (((size_t)blockIdx.x * a.hkv + kvh) * a.row_stride + r) * a.n_splits;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + base;
    Joined j;
    for (int i = 0; i < a.n_splits; ++i) j.m = fmaxf(j.m, stats[i].x);
    for (int i0 = 0; i0 < a.n_splits; i0 += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i0 + i < a.n_splits ? a.partial[(base + i0 + i) * D + d] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < a.n_splits) {
                const float2 st = stats[i0 + i];
                j.add(st.x, v[i], st.y);
            }
    }
    const int row = span.row0 + r, head = kvh * span.group + row % span.group;
    const float whole = j.whole(a.sink_heads ? a.sink_heads[head] : a.sink_all);
    a.out[((size_t)(a.q_start[span.req] + row / span.group) * a.hq + head) * D + d] = from_float<T>(j.den == 0.f ? 0.f : j.num / whole);
}

// The weights of the keys where several tiles of rows, or splits that are no cluster, share them: every key of a request gets the sum over the
// key head's query rows of 2^(score - max) / denominator added to its number in `mass` [pages][hkv][page_size].  The rows in their order,
// so the sum does not change from run to run.
constexpr int MASS_THREADS = 256, MASS_ROWS = 128;                  // rows whose denominators are at hand at a time
template <int ROWS>
__global__ void __launch_bounds__(MASS_THREADS) attn_int4_mass_kernel(const __grid_constant__ Args a, float* __restrict__ mass, int keys_per_block) {
    __shared__ float lse[MASS_ROWS];
    pdl_wait();
    const int req = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    const int n = a.q_len[req], ctx = a.ctx_len[req], group = a.hq / a.hkv, rows = n * group;
    if (n > a.max_queries || n <= 0 || ctx > a.longest) return;
    const int parts = a.cluster > 1 ? 1 : a.n_splits;
    const int lo = blockIdx.z * keys_per_block, hi = min(lo + keys_per_block, ctx);
    if (lo >= hi) return;
    const int* pages = a.table + (size_t)a.req_slot[req] * a.width;
    float w[4] = {0.f, 0.f, 0.f, 0.f};                              // keys_per_block is 4 MASS_THREADS at most
    for (int row0 = 0; row0 < rows; row0 += MASS_ROWS) {
        __syncthreads();
        for (int r = tid; r < min(MASS_ROWS, rows - row0); r += MASS_THREADS) {
            const int row = row0 + r, tile = row / ROWS;
            const size_t base = ((((size_t)req * a.tiles + tile) * a.hkv + kvh) * a.row_stride + row - tile * ROWS) * parts;
            const float2* stats = reinterpret_cast<const float2*>(a.stats) + base;
            Joined j;
            for (int i = 0; i < parts; ++i) j.m = fmaxf(j.m, stats[i].x);
            for (int i = 0; i < parts; ++i) j.add(stats[i].x, 0.f, stats[i].y);
            const int head = kvh * group + row % group;
            lse[r] = j.logarithm(a.sink_heads ? a.sink_heads[head] : a.sink_all);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = lo + i * MASS_THREADS + tid;
            if (key >= hi) continue;
            for (int r = 0; r < min(MASS_ROWS, rows - row0); ++r) {
                const int row = row0 + r, tile = row / ROWS, pos = ctx - n + row / group;
                if (key > pos || (a.window > 0 && pos - key >= a.window && key >= a.keep_first)) continue;
                w[i] += exp2_fast(a.scores[((((size_t)req * a.tiles + tile) * a.hkv + kvh) * a.longest + key) * a.row_stride + row - tile * ROWS] - lse[r]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = lo + i * MASS_THREADS + tid;
        if (key >= hi || a.by_page(key) >= a.width) continue;
        const int page = pages[a.by_page(key)];
        if (page >= 0 && w[i] != 0.f) atomicAdd(mass + ((size_t)page * a.hkv + kvh) * a.page_size + key % a.page_size, w[i]);
    }
}

bool g_pdl = false;
int* g_error = nullptr;

template <int NT, int WARPS> constexpr size_t dynamic_smem() {
    constexpr size_t ring = (size_t)WARPS * 2 * (tile_keys<NT>() / INT4_BLOCK) * BLOCK_BYTES, merge = sizeof(float) * WARPS * 8 * NT * (D + 4);
    return ring > merge ? ring : merge;
}

constexpr int MAX_DEVICES = 64;
int sm_count(int device) {
    static int known[MAX_DEVICES] = {};
    if (!known[device]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) return 1;
        known[device] = n;
    }
    return known[device];
}

// Lets the kernel take its shared memory on a device, once.
template <int NT, int WARPS> cudaError_t prepare_kernel(int device) {
    static bool done[MAX_DEVICES] = {};
    if (done[device]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(attn_int4_kernel<NT, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dynamic_smem<NT, WARPS>());
    done[device] = e == cudaSuccess;
    return e;
}

// Thread blocks of the kernel that run at once on a device in clusters of `size`: a cluster lies in one part of the chip, whose
// last places it may not fill (48 clusters of 6 took two rounds where 296 blocks have places).
template <int NT, int WARPS> int places(int device, int size) {
    static int known[MAX_DEVICES][MAX_CLUSTER + 1] = {};
    if (!known[device][size]) {
        constexpr size_t SMEM = dynamic_smem<NT, WARPS>();
        int n = 0;
        if (prepare_kernel<NT, WARPS>(device) != cudaSuccess) return size;
        if (size == 1) {
            if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_int4_kernel<NT, WARPS>, 32 * WARPS, SMEM) != cudaSuccess) n = 0;
            n *= sm_count(device);
        } else {
            cudaLaunchConfig_t config = {};
            config.gridDim = dim3(1, 1, size); config.blockDim = dim3(32 * WARPS); config.dynamicSmemBytes = SMEM;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = (unsigned)size;
            config.attrs = attr; config.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, attn_int4_kernel<NT, WARPS>, &config) != cudaSuccess) n = 0;
            n *= size;
        }
        cudaGetLastError();
        known[device][size] = n > 0 ? n : size;
    }
    return known[device][size];
}

// What a launch has of everything: query rows of a tile (8, or 16 or 24 where requests bring more), tiles per request, rows that scratch is kept
// for (even, so that pairs are aligned), splits of a request's keys and whether they are one cluster.
struct Shape {
    int rows, tiles, stride, splits, cluster, warps;
    bool ranked;
    int room;                        // thread blocks that run at once, without clusters
    long long units;                 // requests by tiles by key heads by rows
    long long keys;
    int room_of(int device, int w, int size) const {
#if STORAGE_BF16
        if (rows == 24) return places<3, 4>(device, size);
#endif
        if (rows == 16) return places<2, 4>(device, size);
        return w == MOST_WARPS ? places<1, MOST_WARPS>(device, size) : places<1, 4>(device, size);
    }
    // How long `blocks` of w warps take, `tiles` to a warp, in the time that an SM takes for one warp's tile when it is full (0.22 us of 64
    // keys of 128 for bfloat16, 0.38 for float, 0.16 and 0.27 of 32 keys for 16 rows).  A tile of a warp alone takes LATENCY of that, a
    // block's start and end FIXED, the launch and a cluster's joining some more.  Blocks beyond those that run at once come in rounds.
    // Fitted to 1 to 128 requests of 150 to 8000 keys in 1 to 8 splits; right within a fifth, and in the order of what it compares: us of
    // 8 and 4 warps, 8 key heads of 128: 48 x 3000 keys 49 and 41, 64 x 500 22.6 and 16.1, 32 x 4000 38 and 41, in two splits 49 and 41.
    // The units are those of head size 128; at the smaller ones, where a tile is less work, the same constants choose as well: of 77 launches (single
    // tokens, 1 to 128 requests of 150 to 4000 keys, head sizes 32 to 128, float at 64) 70 take at most 7 % longer than the best of all forms, 75 at most
    // 12 %, and two of few blocks at head size 64 16 and 21 % (3 key heads, 32 x 4000 keys: 15.9 us, in four splits 13.1; float 18.7 and 16.1).
    double estimate(long long blocks, int room, int sms, int w, double tiles_of_warp, int parts) const {
        const double FIXED = rows == 8 ? (TERMS == 1 ? 29 : 18) : rows == 24 ? 50 : (TERMS == 1 ? 63 : 51), LATENCY = rows == 8 ? (TERMS == 1 ? 8 : 5) : 5;
        const auto round = [&](long long n) {                       // of n blocks
            const double sharing = (double)w * ((n + sms - 1) / sms);
            return FIXED + tiles_of_warp * (sharing > LATENCY ? sharing : LATENCY);
        };
        return 12 + (parts > 1 ? 10 : 0) + (double)(blocks / room) * round(room) + (blocks % room ? round(blocks % room) : 0);
    }
    // Eight warps unless four are clearly better: of requests of unlike lengths the larger blocks' last round is shorter than estimated (64 of 4000
    // to 8000 keys: 95 us, with four warps 104 to 114, where equal ones are 123 and 117).
    static constexpr double FEWER_WARPS = 0.9;
    // Warps and splits for tiles of `height` rows, and how long they take.
    double choose(int device, int height, int needed, int n_req, int hkv, long long reach) {
        rows = height;
        tiles = (needed + rows - 1) / rows;
        stride = ((needed < rows ? needed : rows) + 1) & ~1;
        const long long pairs = (long long)n_req * tiles * hkv;
        const int sms = sm_count(device);
        double best = 0;
        long long most = 0;
        warps = 0;
        for (int w = rows == 8 ? MOST_WARPS : 4; w >= 4; w /= 2) {
            const int per_block = (rows == 8 ? tile_keys<1>() : tile_keys<2>()) * w;                  // keys of a tile for every warp
            const long long parts = (reach + per_block - 1) / per_block;
            double least = 0;
            int n_least = 1;
            for (int n = 1; n <= (parts < MAX_CLUSTER ? parts : MAX_CLUSTER); ++n) {
                const double time = estimate(pairs * n, room_of(device, w, n), sms, w, (parts + n - 1) / n, n);
                if (n == 1 || time < least) { least = time; n_least = n; }
            }
            if (warps == 0 || least < FEWER_WARPS * best) { best = least; splits = n_least; warps = w; most = parts; }
        }
        room = room_of(device, warps, 1);
        if (splits == MAX_CLUSTER && pairs * MAX_CLUSTER < room / 2) {                                // SMs idle: as many as there are places for
            const long long want = (room + pairs - 1) / pairs;
            splits = (int)(want < most ? want : most);
            if (splits > 64) splits = 64;
        }
        return best;
    }
    Shape(int device, int n_req, int max_queries, int longest, int hq, int hkv, int window, int keep_first) {
        const int needed = max_queries * (hq / hkv);
        long long reach = longest;
        if (window > 0 && (long long)window + keep_first + max_queries < reach) reach = (long long)window + keep_first + max_queries;
        const double time = choose(device, needed > 8 ? 16 : 8, needed, n_req, hkv, reach);
#if STORAGE_BF16
        // A tile of 24 rows takes 1.3 times as long as one of 16 and unpacks the keys once for all: us, 32 heads over 8 of 128, 20 rows of 32
        // requests of 2500 keys 47 and 72, of 8 of 3000 23.5 and 29; 56 rows (64 over 8 of 64) of 8 of 3000 37 and 31.
        if (needed > 16) {
            Shape high = *this;
            if (1.3 * high.choose(device, 24, needed, n_req, hkv, reach) < time) *this = high;
        }
#endif
        const long long pairs = (long long)n_req * tiles * hkv;
        cluster = splits <= MAX_CLUSTER ? splits : 1;
        ranked = n_req > 1 && n_req <= MAX_RANKED && pairs * splits > room;
        units = pairs * stride;
        keys = longest;
    }
    bool merged_by_kernel() const { return splits > 1 && cluster == 1; }
    bool mass_by_kernel() const { return merged_by_kernel() || tiles > 1; }
    long long partial() const { return merged_by_kernel() ? units * splits * D : 0; }
    long long stats(bool mass) const { return merged_by_kernel() ? units * splits * 2 : mass && tiles > 1 ? units * 2 : 0; }
    long long scores(bool mass) const { return mass ? units * keys : 0; }
    int launches(bool mass) const { return 1 + merged_by_kernel() + (mass && mass_by_kernel()); }
};

template <int NT, int WARPS> int launch(int device, Args& a, const Shape& shape, int n_req, float* mass, bool early, cudaStream_t s) {
    constexpr size_t SMEM = dynamic_smem<NT, WARPS>();
    if (const cudaError_t e = prepare_kernel<NT, WARPS>(device); e != cudaSuccess) return (int)e;
    const dim3 grid((unsigned)(n_req * a.tiles), (unsigned)a.hkv, (unsigned)a.n_splits);
    a.mass = shape.mass_by_kernel() ? nullptr : mass;
    int status = launch_kernel_cluster(attn_int4_kernel<NT, WARPS>, grid, dim3(32 * WARPS), SMEM, s, early, a.cluster, a);
    if (status) return status;
    if (shape.merged_by_kernel()) {
        status = launch_kernel(attn_int4_merge_kernel<8 * NT>, dim3(grid.x, grid.y, (unsigned)a.row_stride), dim3(D), 0, s, true, a);
        if (status) return status;
    }
    if (mass && shape.mass_by_kernel()) {
        const int per = 4 * MASS_THREADS;
        status = launch_kernel(attn_int4_mass_kernel<8 * NT>, dim3((unsigned)n_req, (unsigned)a.hkv, (unsigned)((a.longest + per - 1) / per)), dim3(MASS_THREADS), 0, s, true, a, mass, per);
    }
    return status;
}
}  // namespace

CISR_EXPORT void cisr_attn_int4_set_pdl(int on) { g_pdl = on != 0; }
CISR_EXPORT int cisr_attn_int4_head_dim() { return D; }
// `error_flag`: one zeroed int in device memory that the kernels set when a request is longer than they were told.
CISR_EXPORT int cisr_attn_int4_init(int* error_flag) { g_error = error_flag; return 0; }

// Floats of scratch that a call with these sizes on the current device takes (partial sums and statistics of the ranges, with `mass` also the
// scores).  The kernels that it launches: a million million times their number is added.
CISR_EXPORT long long cisr_attn_int4_scratch(int n_req, int max_queries, int longest, int hq, int hkv, int window, int keep_first, int with_mass) {
    int device = 0;
    if (n_req <= 0 || max_queries <= 0 || hkv <= 0 || longest <= 0 || cudaGetDevice(&device) != cudaSuccess || device >= MAX_DEVICES) return 0;
    const Shape s(device, n_req, max_queries, longest, hq, hkv, window, keep_first);
    return s.partial() + s.stats(with_mass != 0) + s.scores(with_mass != 0) + 1000000000000ll * s.launches(with_mass != 0);
}

// A call's arguments, packed by the host in this order (as one address it is a third of the time in the interpreter).
struct AttnInt4Call {
    const void *q; void* out; const void *k_cache, *v_cache; const int *req_slot, *block_table, *q_start, *q_len, *ctx_len; float *scratch, *mass; const float* sink_heads;
    void* stream;
    double scale, sink;
    int width, n_req, max_queries, longest, hq, hkv, page_size, window, keep_first, new_lists;
};

// q, out [tokens][hq][D]; request r brings q_len[r] tokens from row q_start[r] on and has ctx_len[r] rows with them; those with more than
// `max_queries` are left alone, and none may have more than `longest` rows (one that has sets the error flag).  new_lists: the kernel launched just
// before may be the one that writes the lists or the table, which are else read beside its end: this one then starts behind it.
CISR_EXPORT int cisr_attn_int4(const AttnInt4Call* call) {
    const AttnInt4Call& c = *call;
    if (c.n_req <= 0 || c.max_queries <= 0) return 0;
    if (!g_error) return -13;
    if (c.hkv <= 0 || c.hkv > 65535 || c.hq % c.hkv || !isfinite((float)c.scale) || c.longest <= 0 || c.page_size <= 0 || c.page_size % INT4_BLOCK ||
        (long long)c.max_queries * (c.hq / c.hkv) > 1 << 20) return -2;
    if (((uintptr_t)c.q | (uintptr_t)c.k_cache | (uintptr_t)c.v_cache) & 15 || (uintptr_t)c.scratch & 15) return -2;      // rows are read by 16 bytes
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= MAX_DEVICES) return -2;
    const Shape shape(device, c.n_req, c.max_queries, c.longest, c.hq, c.hkv, c.window, c.keep_first);
    if (shape.splits > 65535 || (long long)c.n_req * shape.tiles >= 1ll << 31) return -2;
    const int group = c.hq / c.hkv;
    const bool mass = c.mass != nullptr, early = g_pdl && !c.new_lists;
    Args a{};
    a.q = (const T*)c.q; a.out = (T*)c.out; a.k_cache = (const unsigned char*)c.k_cache; a.v_cache = (const unsigned char*)c.v_cache;
    a.req_slot = c.req_slot; a.table = c.block_table; a.width = c.width; a.q_start = c.q_start; a.q_len = c.q_len; a.ctx_len = c.ctx_len;
    a.partial = c.scratch; a.stats = shape.stats(mass) ? c.scratch + shape.partial() : nullptr; a.scores = mass ? c.scratch + shape.partial() + shape.stats(mass) : nullptr;
    a.max_queries = c.max_queries; a.tiles = shape.tiles; a.row_stride = shape.stride; a.n_splits = shape.splits; a.cluster = shape.cluster;
    a.by_page = Divider((uint32_t)c.page_size); a.by_group = Divider((uint32_t)group); a.by_tiles = Divider((uint32_t)shape.tiles); a.by_heads = Divider((uint32_t)c.hkv);
    a.group = group; a.n_req = c.n_req; a.ranked = shape.ranked;
    a.rank_threads = 1;
    while (a.rank_threads < c.n_req && a.rank_threads < MAX_RANKED) a.rank_threads *= 2;
    a.longest = c.longest; a.hq = c.hq; a.hkv = c.hkv; a.page_size = c.page_size; a.window = c.window; a.keep_first = c.keep_first;
    a.scale = (float)c.scale; a.sink_all = (float)c.sink; a.sink_heads = c.sink_heads; a.error = g_error;
#if STORAGE_BF16
    if (shape.rows == 24) return launch<3, 4>(device, a, shape, c.n_req, c.mass, early, (cudaStream_t)c.stream);
#endif
    const auto run = shape.rows == 16 ? launch<2, 4> : shape.warps == MOST_WARPS ? launch<1, MOST_WARPS> : launch<1, 4>;
    return run(device, a, shape, c.n_req, c.mass, early, (cudaStream_t)c.stream);
}
