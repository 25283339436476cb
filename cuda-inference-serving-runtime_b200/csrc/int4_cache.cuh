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

__host__ __device__ constexpr int int4_row_bytes(int dim) { return dim / 2; }
__host__ __device__ constexpr int int4_block_bytes(int dim) { return 9 * dim / 2; }

__device__ __forceinline__ int int4_value_slot(int r) { return (r >> 1) + 4 * (r & 1); }          // where a block keeps row r of the values
template <int D> __device__ __forceinline__ int int4_value_turn(int slot) { return D == 128 ? ((slot >> 1) & 1) << 2 : 0; }

// Byte offset of the block that holds place `pos` of a sequence, from the start of the cache, or -1 where there is no page.
__device__ __forceinline__ long long int4_block_at(const int* __restrict__ table, int width, int pos, int page_size, int hkv, int head, int dim) {
    const int logical = pos / page_size;
    if (pos < 0 || logical >= width) return -1;
    const int page = table[logical];
    if (page < 0) return -1;
    return (((long long)page * hkv + head) * (page_size / INT4_BLOCK) + (pos - logical * page_size) / INT4_BLOCK) * int4_block_bytes(dim);
}
}  // namespace
