// The form of a key or value cache held in 4 bits, shared by the kernels that write it, read it and attend over it.
//
// 32 neighbours along the head are a group.  Its step is s = float16(max |x| * 1/7, in float), at most 65504 (NaN where the group holds an
// infinity or a NaN); a value is held as the whole number c nearest to x / s (ties to even), -7 <= c <= 7, and stands for c s.  That is
// 4.5 bits a value.  The step is float16 and not bfloat16 because it is a factor of every value: 11 bits of it leave the code's half
// step as the only error that counts.
//
// A page of one key head is page_size / 8 blocks of 8 rows, 9 D / 2 bytes each: eight rows of codes (c + 8 in 4 bits), then the
// steps.  The order inside a block is the one in which the attention kernel's lanes use it, so that a lane reads its share of
// a row by one load and feeds it to the matrix instructions by masks and one shift:
//   keys    row r's word c * (D / 32) + j (32 bits) holds dimensions 32 j + 8 c + 0 .. 7, lowest half byte first; steps [r][j]
//   values  rows 0, 2, 4, 6, 1, 3, 5, 7 in this order; half word g * (D / 32) + u (16 bits) holds dimensions 32 u + 4 g + 0 .. 3, where at
//           D = 128 the eighths g and g ^ 4 of the second and fourth pair of rows are exchanged (else lanes that read four rows
//           at a time would meet in the same shared memory banks); steps [r / 2][u][r % 2]
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace {
constexpr int INT4_GROUP = 32, INT4_BLOCK = 8;

__host__ __device__ constexpr int int4_block_bytes(int dim) { return INT4_BLOCK * (dim / 2 + 2 * dim / INT4_GROUP); }

__device__ __forceinline__ int int4_value_slot(int r) { return (r >> 1) + 4 * (r & 1); }          // where a block keeps row r of the values
template <int D> __device__ __forceinline__ int int4_value_turn(int slot) { return D == 128 ? ((slot >> 1) & 1) << 2 : 0; }

// n / d for n below 2^31 by one multiplication (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divider {
    uint32_t m, shift;               // m 0: divided by one
    __host__ __device__ Divider() : m(0), shift(0) {}
    explicit Divider(uint32_t d) : m(0), shift(0) {
        if (d < 2) return;
        while ((1u << shift) < d) ++shift;
        m = (uint32_t)((1ull << (31 + shift)) / d + 1);
        --shift;
    }
    __device__ __forceinline__ int operator()(int n) const { return m ? (int)(__umulhi((uint32_t)n, m) >> shift) : n; }
};

// Where the block of place `pos` of a sequence is, in blocks from the start of the cache, or -1 where there is no page.  `by_page` divides by
// the page size, `page_blocks` is the page size over 8.
struct Pages { const int* table; int width, page_blocks, hkv; Divider by_page; };
__device__ __forceinline__ long long int4_block_at(const Pages& p, int slot, int pos, int head) {
    const int logical = p.by_page(max(pos, 0));
    const int page = pos >= 0 && logical < p.width ? p.table[(size_t)slot * p.width + logical] : -1;
    if (page < 0) return -1;
    return (long long)((size_t)page * p.hkv + head) * p.page_blocks + ((pos / INT4_BLOCK) - logical * p.page_blocks);
}
}  // namespace
