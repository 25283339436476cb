// Rows of a cache held in 4 bits (int4_cache.cuh): new keys and values brought in, rows handed back as values, and the rows
// that attention has looked at least taken out.
//
// All of these move memory, a row of keys and values of 4 D bytes as bfloat16 and 9 D / 8 as held, and all but the writing out of whole requests
// take longer than that, for what each says.  Head sizes 32, 64, 96 and 128.
#include <type_traits>

#include "int4_cache.cuh"

namespace {
constexpr int THREADS = 256;

// Where a step's rows lie: token t is place positions[t] of request token_req[t].
struct Place { const int* token_req; const int* positions; const int* req_slot; Pages pages; Divider by_heads; };

__device__ __forceinline__ float widened(const float* x, int i) { return x[i]; }
__device__ __forceinline__ float widened(const uint32_t* x, int i) { return __uint_as_float(i & 1 ? x[i >> 1] & 0xffff0000u : x[i >> 1] << 16); }
// N neighbours as they are stored: bfloat16 two to a word.
template <int N> __device__ __forceinline__ void load_raw(const float* p, float* x, bool wide) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if (wide) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        } else {
            for (int e = 0; e < 4; ++e) x[i + e] = p[i + e];
        }
    }
}
template <int N> __device__ __forceinline__ void load_raw(const __nv_bfloat16* p, uint32_t* x, bool wide) {
    if (wide && N == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        x[0] = v.x; x[1] = v.y; x[N / 2 - 2] = v.z; x[N / 2 - 1] = v.w;
    } else if (wide) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        x[0] = v.x; x[1] = v.y;
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < N; i += 2) x[i / 2] = h[i] | (uint32_t)h[i + 1] << 16;
    }
}
// The largest magnitude's bits, as a float's: as whole numbers they order like the magnitudes, NaN above infinity.
template <int N> __device__ __forceinline__ uint32_t largest(const float* x) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    return top;
}
template <int N> __device__ __forceinline__ uint32_t largest(const uint32_t* x) {
    uint32_t two = 0;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) two = __vmaxu2(two, x[i] & 0x7fff7fffu);
    return max(two << 16, two & 0xffff0000u);
}
template <typename T> struct Raw { typedef float type; static constexpr int PER = 1; };
template <> struct Raw<__nv_bfloat16> { typedef uint32_t type; static constexpr int PER = 2; };

__device__ __forceinline__ void store8(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(__half* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 two = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ __half step_of(uint32_t top) {
    if (top >= 0x7f800000u) return __ushort_as_half((unsigned short)0x7e00u);
    return __float2half_rn(fminf(__uint_as_float(top) * (1.f / 7.f), 65504.f));
}
// x / s to the nearest whole number, ties to even, within -7 .. 7; `inv` is 1 / s.  The product x inv is off by an ulp or two, which could
// tip a quotient next to a half: the remainder x - t s is a float without rounding (t s has at most 15 digits and x lies within
// a step of it) and says whether the next whole number is nearer.
__device__ __forceinline__ uint32_t code_of(float x, float s, float inv) {
    float t = rintf(x * inv);
    const float r = fmaf(-t, s, x), twice = 2.f * fabsf(r);
    if (twice > s || (twice == s && ((int)t & 1))) t += copysignf(1.f, r);
    t = s > 0.f ? fminf(fmaxf(t, -7.f), 7.f) : 0.f;
    return (uint32_t)((int)t + 8);
}
// N codes of a group, lowest half byte first.  A bfloat16 over a float16 is a half or at least 2^-12 away from one, so that rounding the
// product to 2^-18 (48 is added: floats there are 2^-18 apart) puts it on the half or leaves it on its side; then 1.5 2^23 - 40 makes
// it the whole number c + 8 in a float's low digits, and the digits above, the same for all, are taken off the sum of N at once.
template <int N, typename R> __device__ __forceinline__ uint32_t codes_of(const R* x, float s, uint32_t top) {
    const float inv = s > 0.f ? 1.f / s : 0.f;
    uint32_t w = 0;
    if (sizeof(R) == 4 && std::is_same<R, uint32_t>::value && __uint_as_float(top) * inv < 7.49f) {
        constexpr float whole = 12582912.f - 40.f;
        uint32_t above = 0;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            w = w * 16 + __float_as_uint((widened(x, i) * inv + 48.f) + whole);
            above = above * 16 + 0x4b400000u;
        }
        return w - above;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) w |= code_of(widened(x, i), s, inv) << (4 * i);
    return w;
}

template <int N> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };
// `BYTES` neighbouring bytes (a lane's share of a row), as wide as they are aligned; 6 and 12 (head size 96) as their thirds.
template <int BYTES> __device__ __forceinline__ void copy_share(void* to, const void* from) {
    constexpr int PART = BYTES % 3 ? BYTES : BYTES / 3;
    typedef typename Word<PART>::type W;
    for (int i = 0; i < BYTES / PART; ++i) reinterpret_cast<W*>(to)[i] = reinterpret_cast<const W*>(from)[i];
}

// Four lanes a row, lane c with the 8 neighbours 32 j + 8 c of every group j: its codes are a quarter of the row, written by one store, and a
// group's largest magnitude is two shuffles away.  (With eight lanes a row of values the arithmetic on places was half of the work.)
constexpr int LANES = 4, PER = 8;
// A quarter row of keys as it is kept is a word per group; of values first the low halves of those words, then the high ones.
template <int NG> __device__ __forceinline__ void to_value_order(uint32_t* w) {
    uint32_t t[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) t[j] = w[j];
    unsigned short h[2 * NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) { h[j] = (unsigned short)t[j]; h[NG + j] = (unsigned short)(t[j] >> 16); }
#pragma unroll
    for (int j = 0; j < NG; ++j) w[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
}
template <int NG> __device__ __forceinline__ void from_value_order(uint32_t* w) {
    unsigned short h[2 * NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) { h[2 * j] = (unsigned short)w[j]; h[2 * j + 1] = (unsigned short)(w[j] >> 16); }
#pragma unroll
    for (int j = 0; j < NG; ++j) w[j] = h[j] | (uint32_t)h[NG + j] << 16;
}
template <int D, typename T, bool VALUES>
__device__ __forceinline__ void store_rows(const T* __restrict__ x, long long token_stride, long long head_stride, unsigned char* __restrict__ cache, float* __restrict__ mass, const Place& at,
                                           int tokens, int hkv, bool wide, int unit) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x % LANES;
    const int row = unit * (THREADS / LANES) + threadIdx.x / LANES;      // token * hkv + head
    const bool inside = row < tokens * hkv;
    const int token = at.by_heads(inside ? row : 0), head = inside ? row - token * hkv : 0;
    const T* from = x + token * token_stride + head * head_stride;
    typename Raw<T>::type v[NG][PER / Raw<T>::PER];
    uint32_t top[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) load_raw<PER>(from + 32 * j + PER * lane, v[j], wide);       // before the row's page is waited for
    const int pos = at.positions[token];
    const long long block = inside ? int4_block_at(at.pages, at.req_slot[at.token_req[token]], pos, head) : -1;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
        top[j] = largest<PER>(v[j]);
#pragma unroll
        for (int o = 1; o < LANES; o *= 2) top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
    }
    if (block < 0) return;
    alignas(16) __half step[NG];
    alignas(16) uint32_t code[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
        step[j] = step_of(top[j]);
        code[j] = codes_of<PER>(v[j], __half2float(step[j]), top[j]);
    }
    const int r = pos % INT4_BLOCK;
    unsigned char* to = cache + block * int4_block_bytes(D);
    if (VALUES) {
        const int slot = int4_value_slot(r);
        to_value_order<NG>(code);
        copy_share<4 * NG>(to + slot * (D / 2) + (lane ^ int4_value_turn<D>(slot) / 2) * 4 * NG, code);
        if (lane < NG) {
            __half mine = step[0];
#pragma unroll
            for (int j = 1; j < NG; ++j) if (lane == j) mine = step[j];
            reinterpret_cast<__half*>(to + 4 * D)[((r >> 1) * NG + lane) * 2 + (r & 1)] = mine;
        }
    } else {
        copy_share<4 * NG>(to + r * (D / 2) + lane * 4 * NG, code);
        if (lane == 0) {
            copy_share<2 * NG>(to + 4 * D + r * 2 * NG, step);
            if (mass) mass[block * INT4_BLOCK + r] = 0.f;
        }
    }
}

// The first half of the thread blocks for the keys, the second for the values.  8192 tokens of 8 heads of 128: 12.4 us in bfloat16 and 20.6 in
// float, at memory's rate 6.6 and 11.7.  Neither memory nor issue slots are full then (bfloat16, counters: DRAM 25 %, issue 52 %, 63 % of the warps): it is
// 1.7 rounds of thread blocks, each of which waits for its rows and their pages, converts and stores, and 2.5 us are the launch's start and
// end.  A few tokens are the launch alone.
template <int D, typename T>
__global__ void __launch_bounds__(THREADS) int4_store_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_token, long long k_head, long long v_token,
                                                             long long v_head, unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache, float* __restrict__ mass,
                                                             Place at, int tokens, int hkv, int wide) {
    pdl_wait();
    pdl_trigger();
    const long long rows = (long long)tokens * hkv;
    const int key_units = (int)((rows + THREADS / LANES - 1) / (THREADS / LANES));
    if ((int)blockIdx.x < key_units) store_rows<D, T, false>(k, k_token, k_head, k_cache, mass, at, tokens, hkv, wide & 1, blockIdx.x);
    else store_rows<D, T, true>(v, v_token, v_head, v_cache, mass, at, tokens, hkv, wide & 2, blockIdx.x - key_units);
}

// Rows as values.  `out` is [tokens][heads] with strides of their own; places without a page, and with `ends` those behind a
// request's end, give zeros.  float16 (three binary digits times eleven, rounded to eleven): divided by the key head's factor (int4_top_kernel).
// Whole requests as bfloat16 are bound by memory: 24 x 2048 rows of 8 heads of 128 43 us of 39 (counters: issue 78 % as well).  As float 101
// of 70: nine tenths of the bytes are those written, by a warp to eight rows at a time.  8192 rows as bfloat16 10.4 us of 6.6, as float 20.6 of 11.7, where issue
// slots (58 %) and the launch's start and end count more than memory (DRAM 9 %: the rows lie in L2).
constexpr int READ_ROWS = 1;         // of a thread, and eight thread blocks to an SM: with four rows on their way together, and so fewer threads, 47 and 130
                                     // (the same lines without the arrays spilled registers: 24 x 2048 rows 46 us)
template <int D, typename T, bool VALUES>
__device__ __forceinline__ void read_rows(const unsigned char* __restrict__ cache, T* __restrict__ out, long long req_stride, long long token_stride, long long head_stride,
                                          const Place& at, Divider by_tokens, const int* __restrict__ ends, const int* __restrict__ which, const float* __restrict__ factors,
                                          int tokens, int hkv, int unit) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x % LANES;
    const int first = unit * READ_ROWS * (THREADS / LANES) + threadIdx.x / LANES;
    int token[READ_ROWS], head[READ_ROWS], pos[READ_ROWS], slot[READ_ROWS];
#pragma unroll
    for (int i = 0; i < READ_ROWS; ++i) {
        const int row = first + i * (THREADS / LANES);
        token[i] = -1;
        if (row >= tokens * hkv) continue;
        if (ends) {                  // neighbouring rows of a head lie side by side
            head[i] = by_tokens(row); token[i] = row - head[i] * tokens;
            const int req = which ? which[blockIdx.y] : blockIdx.y;
            slot[i] = at.req_slot[req]; pos[i] = token[i] < ends[req] ? token[i] : -1;
        } else {
            token[i] = at.by_heads(row); head[i] = row - token[i] * hkv;
            slot[i] = at.req_slot[at.token_req[token[i]]]; pos[i] = at.positions[token[i]];
        }
    }
    long long block[READ_ROWS];
#pragma unroll
    for (int i = 0; i < READ_ROWS; ++i) block[i] = token[i] < 0 ? -1 : int4_block_at(at.pages, slot[i], pos[i], head[i]);
    struct alignas(16) Part { uint32_t w[NG]; };
    Part code[READ_ROWS], held[READ_ROWS];                          // held: steps, of keys the row's (the first half), of values two rows' side by side
#pragma unroll
    for (int i = 0; i < READ_ROWS; ++i) {
        if (block[i] < 0) continue;
        const unsigned char* from = cache + block[i] * int4_block_bytes(D);
        const int r = pos[i] & (INT4_BLOCK - 1);
        if (VALUES) {
            const int at_slot = int4_value_slot(r);
            copy_share<4 * NG>(&code[i], from + at_slot * (D / 2) + (lane ^ int4_value_turn<D>(at_slot) / 2) * 4 * NG);
            copy_share<4 * NG>(&held[i], from + 4 * D + (r >> 1) * 4 * NG);
        } else {
            copy_share<4 * NG>(&code[i], from + r * (D / 2) + lane * 4 * NG);
            copy_share<2 * NG>(&held[i], from + 4 * D + r * 2 * NG);
        }
    }
#pragma unroll
    for (int i = 0; i < READ_ROWS; ++i) {
        if (token[i] < 0) continue;
        T* to = out + (ends ? blockIdx.y * req_stride : 0) + token[i] * token_stride + head[i] * head_stride;
        if (VALUES) from_value_order<NG>(code[i].w);
        float inverse = 1.f;
        if constexpr (std::is_same<T, __half>::value) inverse = __uint_as_float((254u << 23) - __float_as_uint(factors[((size_t)blockIdx.y * hkv + head[i]) * 2 + VALUES]));      // (a power of two)
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t two = VALUES ? held[i].w[j] : held[i].w[j / 2];
            const float step = __half2float(__ushort_as_half((unsigned short)((VALUES ? pos[i] & 1 : j & 1) ? two >> 16 : two & 0xffff))) * inverse;
            float x[PER];            // 2^23 + n as a float, less 2^23 + 8
#pragma unroll
            for (int e = 0; e < PER; ++e)
                x[e] = block[i] < 0 ? 0.f : (__uint_as_float(0x4b000000u | ((code[i].w[j] >> (4 * e)) & 15)) - 8388616.f) * step;
            store8(to + 32 * j + PER * lane, x);
        }
    }
}

// A prompt's queries [rows][D] as float16, each row times a power of two that brings its largest to 2^14 .. 2^15, which its factor takes back, and with
// the sign of the scale (the softmax behind takes its maximum before it scales, so its scale is positive).
struct Queries { const uint4* q; uint4* half; float* factor; long long rows; float scale; };
template <int D> __device__ __forceinline__ void convert_queries(const Queries& a, long long block) {
    constexpr int PARTS = D / 8;                                    // threads that share a row
    const long long at = block * blockDim.x + threadIdx.x, row = at / PARTS;
    const bool there = row < a.rows;
    const uint4 v = there ? a.q[at] : make_uint4(0, 0, 0, 0);
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = largest<8>(x);
#pragma unroll
    for (int o = 1; o < PARTS; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int exponent = min(14 - ((int)(top >> 23) - 127), 120);
    const float up = copysignf(__uint_as_float((uint32_t)(exponent + 127) << 23), a.scale);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 two = __floats2half2_rn(widened(x, 2 * i) * up, widened(x, 2 * i + 1) * up);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    if (there) a.half[at] = make_uint4(w[0], w[1], w[2], w[3]);
    if (there && at % PARTS == 0) a.factor[row] = __uint_as_float((uint32_t)(127 - exponent) << 23);
}

// What a prompt's attention with float16 operands needs before its rows are written out: a power of two for each request's key head, keys
// and values apart, to the same end (a thread block reads all its steps, 1/9 of what is held; NaN is left out, and stays NaN), and
// its queries, which the thread blocks behind those take meanwhile.  2 requests of 3500 rows, 8 heads, and 2000 queries of 32 heads of 128: 8.6 us (with one
// thread block to an SM, for its registers, 12).
constexpr int TOP_THREADS = 1024;
template <int D>
__global__ void __launch_bounds__(TOP_THREADS, 2) int4_top_kernel(const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache,
                                                               const int* __restrict__ req_slot, Pages pages, const int* __restrict__ ends, const int* __restrict__ which,
                                                               float* __restrict__ factors, int* __restrict__ pages_out, int n_req, int rows, int* __restrict__ error,
                                                               Queries queries) {
    constexpr int NG = D / 32, AT_ONCE = 4;
    __shared__ uint32_t of_warp[TOP_THREADS / 32];
    pdl_wait();
    pdl_trigger();
    if ((int)blockIdx.x >= 2 * n_req * pages.hkv) return convert_queries<D>(queries, blockIdx.x - 2 * n_req * pages.hkv);
    const int tid = threadIdx.x, unit = blockIdx.x >> 1, i = unit / pages.hkv, head = unit - i * pages.hkv;
    const bool values = blockIdx.x & 1;
    const int req = which ? which[i] : i, slot = req_slot[req], end = ends[req];
    if (tid == 0 && head == 0 && !values) {
        pages_out[i] = i;                                           // the table of the rows written out: a page each
        if (end > rows) atomicExch(error, 6);                       // more rows than there is room for
    }
    const unsigned char* cache = values ? v_cache : k_cache;
    uint32_t top = 0;
    const int chunks = (end + INT4_BLOCK - 1) / INT4_BLOCK * NG;    // of eight steps
    for (int c0 = tid; c0 < chunks; c0 += AT_ONCE * TOP_THREADS) {
        uint4 v[AT_ONCE];
        long long block[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int c = c0 + u * TOP_THREADS;
            block[u] = c < chunks ? int4_block_at(pages, slot, c / NG * INT4_BLOCK, head) : -1;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            v[u] = block[u] < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(cache + block[u] * int4_block_bytes(D) + 4 * D + 16 * ((c0 + u * TOP_THREADS) % NG));
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int c = c0 + u * TOP_THREADS;
            const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = 8 * (c % NG) + e, row = c / NG * INT4_BLOCK + (values ? at / (2 * NG) * 2 + (at & 1) : at / NG);
                const uint32_t s = e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffff;
                if (row < end && s < 0x7c00u) top = max(top, s);
            }
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (tid % 32 == 0) of_warp[tid / 32] = top;
    __syncthreads();
    if (tid < 32) {
        top = __reduce_max_sync(0xffffffffu, of_warp[tid]);
        const float most = 7.f * __half2float(__ushort_as_half((unsigned short)top));               // 2^-22 .. 2^19
        const int exponent = top ? (int)(__float_as_uint(most) >> 23) - 127 - 14 : 0;
        if (tid == 0) factors[((size_t)i * pages.hkv + head) * 2 + values] = __uint_as_float((uint32_t)(exponent + 127) << 23);
    }
}
static_assert(TOP_THREADS == 1024, "a warp joins 32");

template <int D, typename T>
__global__ void __launch_bounds__(THREADS, 8) int4_read_kernel(const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache, T* __restrict__ k,
                                                            T* __restrict__ v, long long req_stride, long long token_stride, long long head_stride, Place at,
                                                            Divider by_tokens, const int* __restrict__ ends, const int* __restrict__ which, const float* __restrict__ factors,
                                                            int tokens, int hkv) {
    pdl_wait();
    pdl_trigger();
    const long long rows = (long long)tokens * hkv;
    constexpr int EACH = READ_ROWS * (THREADS / LANES);
    const int key_units = (int)((rows + EACH - 1) / EACH);
    if ((int)blockIdx.x < key_units) read_rows<D, T, false>(k_cache, k, req_stride, token_stride, head_stride, at, by_tokens, ends, which, factors, tokens, hkv, blockIdx.x);
    else read_rows<D, T, true>(v_cache, v, req_stride, token_stride, head_stride, at, by_tokens, ends, which, factors, tokens, hkv, blockIdx.x - key_units);
}

// ------------------------------------------------------------------ eviction
// Of a request's `len` rows stay, per key head, the first `first`, the last `recent`, and of those between the `keep - first - recent` with
// the largest sums, equal ones by the lowest place; NaN counts as the largest.  Two kernels: one finds the places and
// lists them in order, the other moves the rows (and their sums) to the request's new pages.
//
// The choice is a search for the smallest sum that stays: the bits of a float, turned so that they order like the numbers, are found eleven,
// eleven and ten at a time, by counting how many of the sums that begin with the bits found so far have which bits next.  Bound by
// instructions, some 220 per 32 sums (load, three passes, two walks for the places): 24 requests of 4096 rows, 8 heads, 16 us.
constexpr int SELECT_THREADS = 1024, SELECT_BITS = 11;              // two counts a thread
constexpr int SELECT_CACHED = 48 * 1024;                            // sums that fit shared memory; those of longer requests are read again in every pass
static_assert(2 * SELECT_THREADS == 1 << SELECT_BITS, "a thread has two counts");

__device__ __forceinline__ uint32_t ordered(float x) {
    if (isnan(x)) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.f);                    // -0 becomes 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(SELECT_THREADS, 2) int4_select_kernel(const float* __restrict__ mass, const int* __restrict__ req_slot, Pages pages,
                                                                     const int* __restrict__ ctx_len, int* __restrict__ kept, int keep, int recent, int first, int cached) {
    extern __shared__ uint32_t sums[];
    __shared__ int count[1 << SELECT_BITS], found[2];               // by the next bits; the ones found, and how many are above them
    __shared__ int of_warp[2][32];
    pdl_wait();
    const int head = blockIdx.x, req = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int* table = pages.table + (size_t)req_slot[req] * pages.width;
    const int page_size = pages.page_blocks * INT4_BLOCK;
    const int len = min(max(ctx_len[req], 0), (int)min((long long)pages.width * page_size, 0x7fffffffll));
    int* out = kept + ((size_t)req * pages.hkv + head) * keep;
    if (len <= keep) {
        for (int i = tid; i < keep; i += SELECT_THREADS) out[i] = i < len ? i : -1;
        return;
    }
    const int begin = first, n = len - recent - first, want = keep - recent - first;       // of n rows from `begin` on, `want` stay; want < n
    const auto fetch = [&](int i) -> uint32_t {
        const int pos = begin + i, logical = pages.by_page(pos), page = table[logical];
        return page < 0 ? 0u : ordered(mass[((size_t)page * pages.hkv + head) * page_size + pos - logical * page_size]);
    };
    const bool in_shared = n <= cached;
    if (in_shared) {
        constexpr int AT_ONCE = 4;                                  // of a thread on their way together
        for (int i0 = tid; i0 < n; i0 += AT_ONCE * SELECT_THREADS) {
            int page[AT_ONCE], inside[AT_ONCE];
            float value[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int pos = begin + min(i0 + u * SELECT_THREADS, n - 1), logical = pages.by_page(pos);
                page[u] = table[logical]; inside[u] = pos - logical * page_size;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) value[u] = page[u] < 0 ? 0.f : mass[((size_t)page[u] * pages.hkv + head) * page_size + inside[u]];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (i0 + u * SELECT_THREADS < n) sums[i0 + u * SELECT_THREADS] = page[u] < 0 ? 0u : ordered(value[u]);
        }
    }
    __syncthreads();
    const auto at = [&](int i) -> uint32_t { return in_shared ? sums[i] : fetch(i); };
    uint32_t floor_ = 0;                                            // the smallest sum that stays
    if (want > 0) {
        int need = want;                                            // of those that begin with the bits found
        for (int shift = 32 - SELECT_BITS, bits = SELECT_BITS; ;) {
            for (int i = tid; i < 1 << SELECT_BITS; i += SELECT_THREADS) count[i] = 0;
            __syncthreads();
            const uint32_t known = shift + bits >= 32 ? 0u : ~0u << (shift + bits);
            for (int i = tid; i < n; i += SELECT_THREADS) {
                const uint32_t s = at(i);
                if ((s & known) == floor_) atomicAdd(&count[(s >> shift) & ((1u << bits) - 1)], 1);
            }
            __syncthreads();
            // from the largest down: a thread has two neighbours, and learns how many lie above them
            const int hi = (1 << SELECT_BITS) - 1 - 2 * tid, c0 = count[hi], c1 = count[hi - 1];
            int above = c0 + c1;
            for (int o = 1; o < 32; o *= 2) {
                const int a = __shfl_up_sync(0xffffffffu, above, o);
                if (lane >= o) above += a;
            }
            if (lane == 31) of_warp[0][warp] = above;
            __syncthreads();
            int before = lane < warp ? of_warp[0][lane] : 0;
            above += __reduce_add_sync(0xffffffffu, before) - c0 - c1;
            if (above < need && above + c0 >= need) { found[0] = hi; found[1] = above; }
            else if (above + c0 < need && above + c0 + c1 >= need) { found[0] = hi - 1; found[1] = above + c0; }
            __syncthreads();
            floor_ |= (uint32_t)found[0] << shift;
            need -= found[1];
            if (shift == 0) break;
            bits = shift < SELECT_BITS ? shift : SELECT_BITS;
            shift -= bits;
        }
    }
    // Places in order: a thread owns a run of neighbours (of odd length, so that runs start in different banks), counts those above the
    // floor and those on it, and learns by a scan over the block how many lie before its run.
    const int per = ((n + SELECT_THREADS - 1) / SELECT_THREADS) | 1, lo = min(n, tid * per), hi = min(n, lo + per);
    int above = 0, equal = 0;
    if (want > 0) {
        for (int i = lo; i < hi; ++i) {
            const uint32_t s = at(i);
            above += s > floor_; equal += s == floor_;
        }
    }
    int above_before = above, equal_before = equal;
    for (int o = 1; o < 32; o *= 2) {
        const int a = __shfl_up_sync(0xffffffffu, above_before, o), e = __shfl_up_sync(0xffffffffu, equal_before, o);
        if (lane >= o) { above_before += a; equal_before += e; }
    }
    if (lane == 31) { of_warp[0][warp] = above_before; of_warp[1][warp] = equal_before; }
    __syncthreads();
    int a_sum = of_warp[0][lane], e_sum = of_warp[1][lane];
    const int a_total = __reduce_add_sync(0xffffffffu, a_sum);
    a_sum = lane < warp ? a_sum : 0; e_sum = lane < warp ? e_sum : 0;
    above_before += __reduce_add_sync(0xffffffffu, a_sum) - above;
    equal_before += __reduce_add_sync(0xffffffffu, e_sum) - equal;
    const int spare = want - a_total;                               // of those on the floor, the first `spare` stay
    if (want > 0) {
        for (int i = lo; i < hi; ++i) {
            const uint32_t s = at(i);
            const bool stays = s > floor_ || (s == floor_ && equal_before < spare);
            if (stays) out[first + above_before + min(equal_before, spare)] = begin + i;
            above_before += s > floor_; equal_before += s == floor_;
        }
    }
    for (int i = tid; i < first; i += SELECT_THREADS) out[i] = i;
    for (int i = tid; i < recent; i += SELECT_THREADS) out[keep - recent + i] = len - recent + i;
}

// A warp moves the rows of a new block of 8: lane (r, c) a quarter of row r of the keys, of the row in slot r of the values, a step of each, and
// (c = 0) the row's sum.  Bound by memory, of which a kept row's neighbours come along, and by three trips to it, one behind another, which
// eight thread blocks of an SM hide (with four blocks of rows to a warp, and so fewer warps, it took 35 us): 2048 of 4096 rows of
// 24 requests, 8 heads of 128, 27 us (17 for the rows alone, 26 with all that is read).
template <int D>
__global__ void __launch_bounds__(THREADS, 8) int4_move_kernel(unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache, float* __restrict__ mass,
                                                               const int* __restrict__ req_slot, Pages pages, Pages to_pages, const int* __restrict__ kept, int keep) {
    constexpr int NG = D / 32;
    pdl_wait();
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, head = blockIdx.y, req = blockIdx.z, slot = req_slot[req];
    const int* places = kept + ((size_t)req * pages.hkv + head) * keep;
    const int slot_row = 2 * (r & 3) + (r >> 2);                    // the row in slot r of the values
    const int row = (blockIdx.x * (THREADS / 32) + threadIdx.x / 32) * INT4_BLOCK;
    const int key_pos = row + r < keep ? places[row + r] : -1, value_pos = row + slot_row < keep ? places[row + slot_row] : -1;
    const long long to = row < keep ? int4_block_at(to_pages, req, row, head) : -1;
    const long long key_at = to < 0 ? -1 : int4_block_at(pages, slot, key_pos, head), value_at = to < 0 ? -1 : int4_block_at(pages, slot, value_pos, head);
    struct alignas(16) Part { uint32_t w[NG]; };
    Part k, v;
    __half k_step, v_step;
    float sum;
    if (key_at >= 0) {
        const unsigned char* from = k_cache + key_at * int4_block_bytes(D);
        const int from_r = key_pos % INT4_BLOCK;
        copy_share<4 * NG>(&k, from + from_r * (D / 2) + c * 4 * NG);
        if (c < NG) k_step = reinterpret_cast<const __half*>(from + 4 * D)[from_r * NG + c];
        if (c == 0) sum = mass[key_at * INT4_BLOCK + from_r];
    }
    if (value_at >= 0) {
        const unsigned char* from = v_cache + value_at * int4_block_bytes(D);
        const int from_r = value_pos % INT4_BLOCK, from_slot = int4_value_slot(from_r);
        const int turned = int4_value_turn<D>(r) != int4_value_turn<D>(from_slot) ? 2 : 0;      // eighths exchanged four by four: quarters two by two
        copy_share<4 * NG>(&v, from + from_slot * (D / 2) + (c ^ turned) * 4 * NG);
        if (c < NG) v_step = reinterpret_cast<const __half*>(from + 4 * D)[((from_r >> 1) * NG + c) * 2 + (from_r & 1)];
    }
    if (key_at >= 0) {
        unsigned char* dest = k_cache + to * int4_block_bytes(D);
        copy_share<4 * NG>(dest + r * (D / 2) + c * 4 * NG, &k);
        if (c < NG) reinterpret_cast<__half*>(dest + 4 * D)[r * NG + c] = k_step;
        if (c == 0) mass[to * INT4_BLOCK + r] = sum;
    }
    if (value_at >= 0) {
        unsigned char* dest = v_cache + to * int4_block_bytes(D);
        copy_share<4 * NG>(dest + r * (D / 2) + c * 4 * NG, &v);
        if (c < NG) reinterpret_cast<__half*>(dest + 4 * D)[((slot_row >> 1) * NG + c) * 2 + (slot_row & 1)] = v_step;
    }
}

bool g_pdl = false;

Pages pages_of(const int* table, int width, int page_size, int hkv) { return Pages{table, width, page_size / INT4_BLOCK, hkv, Divider((uint32_t)page_size)}; }

template <typename F> int by_head_size(int dim, F f) {
    switch (dim) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 96: return f(std::integral_constant<int, 96>());
        case 128: return f(std::integral_constant<int, 128>());
        default: return -2;
    }
}
// Thread blocks for a launch over `rows` rows of keys and as many of values, `each` a block.
long long units(long long rows, int each) { return 2 * ((rows + each - 1) / each); }
}  // namespace

CISR_EXPORT void cisr_int4_rows_set_pdl(int on) { g_pdl = on != 0; }

// Calls' arguments, packed by the host in this order (as one address they are a third of the time in the interpreter).
struct Int4StoreCall {
    const void *k, *v; void *k_cache, *v_cache; float* mass; const int *token_req, *positions, *req_slot, *block_table; void* stream;
    long long k_token, k_head, v_token, v_head;
    int dtype, width, page_size, tokens, hkv, dim;
};
struct Int4ReadCall {
    const void *k_cache, *v_cache; void *k, *v; const int *token_req, *positions, *req_slot, *block_table, *ends, *which; void* stream;
    long long req_stride, token_stride, head_stride;
    int dtype, width, page_size, n_req, tokens, hkv, dim;
};
struct Int4EvictCall {
    void *k_cache, *v_cache; float* mass; const int *req_slot, *block_table, *ctx_len; int* kept; const int* to_table; void* stream;
    int width, to_width, n_req, hkv, dim, page_size, keep, recent, first, longest;
};

// k, v [tokens][hkv][dim] with strides in values; codes go to place positions[t] of request token_req[t], whose number in `mass` (if any) becomes 0.
CISR_EXPORT int cisr_int4_store(const Int4StoreCall* call) {
    const Int4StoreCall& c = *call;
    if (c.tokens <= 0) return 0;
    if (c.hkv <= 0 || c.page_size <= 0 || c.page_size % INT4_BLOCK || ((uintptr_t)c.k_cache | (uintptr_t)c.v_cache) & 15) return -2;
    if ((long long)c.tokens * c.hkv >= 1ll << 30) return -2;
    const long long blocks = units((long long)c.tokens * c.hkv, THREADS / LANES);
    const int per16 = c.dtype == CISR_F32 ? 4 : 8;
    const int wide = (((uintptr_t)c.k & 15) == 0 && c.k_token % per16 == 0 && c.k_head % per16 == 0 ? 1 : 0) |
                     (((uintptr_t)c.v & 15) == 0 && c.v_token % per16 == 0 && c.v_head % per16 == 0 ? 2 : 0);
    const Place at{c.token_req, c.positions, c.req_slot, pages_of(c.block_table, c.width, c.page_size, c.hkv), Divider((uint32_t)c.hkv)};
    return by_head_size(c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const auto run = [&](auto* kernel, auto* k, auto* v) {
            return launch_kernel(kernel, dim3((unsigned)blocks), dim3(THREADS), 0, (cudaStream_t)c.stream, g_pdl, k, v, c.k_token, c.k_head, c.v_token, c.v_head,
                                 (unsigned char*)c.k_cache, (unsigned char*)c.v_cache, c.mass, at, c.tokens, c.hkv, wide);
        };
        return c.dtype == CISR_F32 ? run(int4_store_kernel<D, float>, (const float*)c.k, (const float*)c.v)
                                   : run(int4_store_kernel<D, __nv_bfloat16>, (const __nv_bfloat16*)c.k, (const __nv_bfloat16*)c.v);
    });
}

// The reverse: rows (token_req[t], positions[t]) into k, v [tokens][hkv][dim]; or, with `ends`, places 0 .. tokens - 1 of each of n_req
// requests (request which[i], or i without a list) into [n_req][..] with the strides given; places from ends[request] on give zeros.
CISR_EXPORT int cisr_int4_read(const Int4ReadCall* call) {
    const Int4ReadCall& c = *call;
    if (c.tokens <= 0 || c.n_req <= 0) return 0;
    if (c.hkv <= 0 || c.page_size <= 0 || c.page_size % INT4_BLOCK || c.n_req > 65535) return -2;
    if (((uintptr_t)c.k_cache | (uintptr_t)c.v_cache | (uintptr_t)c.k | (uintptr_t)c.v) & 15 || c.token_stride % 8 || c.head_stride % 8 || c.req_stride % 8) return -2;
    if ((long long)c.tokens * c.hkv >= 1ll << 30) return -2;
    const long long blocks = units((long long)c.tokens * c.hkv, READ_ROWS * (THREADS / LANES));
    const Place at{c.token_req, c.positions, c.req_slot, pages_of(c.block_table, c.width, c.page_size, c.hkv), Divider((uint32_t)c.hkv)};
    const dim3 grid((unsigned)blocks, (unsigned)c.n_req);
    return by_head_size(c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const auto run = [&](auto* kernel, auto* k, auto* v) {
            return launch_kernel(kernel, grid, dim3(THREADS), 0, (cudaStream_t)c.stream, g_pdl, (const unsigned char*)c.k_cache, (const unsigned char*)c.v_cache, k, v, c.req_stride,
                                 c.token_stride, c.head_stride, at, Divider((uint32_t)c.tokens), c.ends, c.which, (const float*)nullptr, c.tokens, c.hkv);
        };
        return c.dtype == CISR_F32 ? run(int4_read_kernel<D, float>, (float*)c.k, (float*)c.v) : run(int4_read_kernel<D, __nv_bfloat16>, (__nv_bfloat16*)c.k, (__nv_bfloat16*)c.v);
    });
}

// For a prompt's attention with float16 operands (head sizes 64 and 128): places 0 .. rows - 1 of n_req requests (request which[i], or i without a list) into
// k, v float16 [n_req][hkv][rows][dim] over `factors` [n_req][hkv][2] (pages_out becomes 0, 1, .. n_req - 1), and queries bfloat16 [q_rows][dim] into q_half over q_factor [q_rows],
// with the sign of `scale`.
// A request with more rows sets the error flag.
CISR_EXPORT int cisr_int4_prompt(const void* k_cache, const void* v_cache, void* k, void* v, float* factors, int* pages_out, const void* q, void* q_half, float* q_factor, long long q_rows,
                                 const int* req_slot, const int* block_table, int width, int page_size, const int* ends, const int* which, int n_req, int rows, int hkv, int dim,
                                 float scale, int* error, void* stream) {
    if (!isfinite(scale)) return -2;
    if (rows <= 0 || n_req <= 0) return 0;
    if (hkv <= 0 || page_size <= 0 || page_size % INT4_BLOCK || n_req > 65535 || (long long)rows * hkv >= 1ll << 30) return -2;
    if (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_half) & 15) return -2;
    const Pages pages = pages_of(block_table, width, page_size, hkv);
    const Place at{nullptr, nullptr, req_slot, pages, Divider((uint32_t)hkv)};
    const dim3 grid((unsigned)units((long long)rows * hkv, READ_ROWS * (THREADS / LANES)), (unsigned)n_req);
    const Queries queries{(const uint4*)q, (uint4*)q_half, q_factor, q_rows, scale};
    const long long blocks = 2ll * n_req * hkv + (q_rows * (dim / 8) + TOP_THREADS - 1) / TOP_THREADS;
    if (blocks >= 1ll << 31) return -2;
    const auto run = [&](auto d) {
        constexpr int D = decltype(d)::value;
        const int status = launch_kernel(int4_top_kernel<D>, dim3((unsigned)blocks), dim3(TOP_THREADS), 0, (cudaStream_t)stream, g_pdl, (const unsigned char*)k_cache,
                                         (const unsigned char*)v_cache, req_slot, pages, ends, which, factors, pages_out, n_req, rows, error, queries);
        if (status) return status;
        return launch_kernel(int4_read_kernel<D, __half>, grid, dim3(THREADS), 0, (cudaStream_t)stream, true, (const unsigned char*)k_cache, (const unsigned char*)v_cache, (__half*)k,
                             (__half*)v, (long long)hkv * rows * D, (long long)D, (long long)rows * D, at, Divider((uint32_t)rows), ends, which, (const float*)factors, rows, hkv);
    };
    return dim == 64 ? run(std::integral_constant<int, 64>()) : dim == 128 ? run(std::integral_constant<int, 128>()) : -2;
}

// Places that stay into kept [n_req][hkv][keep] (-1 behind the last), their rows and sums to the pages of to_table [n_req][to_width].
// `longest`: no request has more rows.
CISR_EXPORT int cisr_int4_evict(const Int4EvictCall* call) {
    const Int4EvictCall& c = *call;
    if (c.n_req <= 0 || c.keep <= 0) return 0;
    if (c.hkv <= 0 || c.hkv > 65535 || c.n_req > 65535 || c.page_size <= 0 || c.page_size % INT4_BLOCK || c.recent < 0 || c.first < 0 || c.recent > c.keep ||
        c.first > c.keep - c.recent) return -2;
    if (((uintptr_t)c.k_cache | (uintptr_t)c.v_cache) & 15) return -2;
    const Pages pages = pages_of(c.block_table, c.width, c.page_size, c.hkv);
    const int between = c.longest - c.recent - c.first;
    const int cached = between < 0 ? 0 : between < SELECT_CACHED ? between : SELECT_CACHED;
    const size_t smem = sizeof(uint32_t) * (size_t)cached;
    if (smem > 32 * 1024) {          // with the counts more than the 48 KB that need no leave
        const cudaError_t e = cudaFuncSetAttribute(int4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(uint32_t) * SELECT_CACHED));
        if (e != cudaSuccess) return (int)e;
    }
    const cudaStream_t s = (cudaStream_t)c.stream;
    const int status = launch_kernel(int4_select_kernel, dim3(c.hkv, c.n_req), dim3(SELECT_THREADS), smem, s, g_pdl, (const float*)c.mass, c.req_slot, pages, c.ctx_len, c.kept,
                                     c.keep, c.recent, c.first, cached);
    if (status) return status;
    constexpr int rows = INT4_BLOCK * (THREADS / 32);
    const dim3 grid((unsigned)((c.keep + rows - 1) / rows), c.hkv, c.n_req);
    return by_head_size(c.dim, [&](auto d) {
        return launch_kernel(int4_move_kernel<decltype(d)::value>, grid, dim3(THREADS), 0, s, true, (unsigned char*)c.k_cache, (unsigned char*)c.v_cache, c.mass, c.req_slot, pages,
                             pages_of(c.to_table, c.to_width, c.page_size, c.hkv), (const int*)c.kept, c.keep);
    });
}
