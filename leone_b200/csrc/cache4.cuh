// Pages that hold keys and values in 4 bits.
//
// The d elements of a head's row are cut into groups(d) groups of equal size, at most 64 elements each.  A group has a scale s and an
// offset z, both bfloat16: z is the largest bfloat16 not above the group's minimum, s the smallest one not below (max - z) / 15 (0
// where that is no normal number).  An element's code is rint((x - z) / s), 0 .. 15, and stands for z + s * code; it is off by
// at most half of s.  A group that holds a NaN or an infinity, or whose s or z would be one, has s = z = NaN: what reads it sees
// NaN.  A pool is [pages, cached heads, page_tokens, row_bytes(d)] bytes, page_tokens a multiple of 16.
//
// Inside a page the rows of one head lie in units of 16 tokens: 16 rows of d / 2 bytes of codes, then 16 rows of groups(d) words (s in
// the low half, z in the high half), so that a unit of keys or values is one piece of 16 * row_bytes(d) bytes (a multiple of
// 16): 1,152 for 128 elements, where bfloat16 has 4,096.  How the words of codes lie in a unit follows the tensor cores' operands:
//   * word w of a row holds elements 8 w .. 8 w + 7, element 2 j in nibble j and element 2 j + 1 in nibble j + 4: (word >> 4 j) &
//     0x000f000f is the pair 2 j, 2 j + 1 in the two halves of a register.  As bit patterns codes are numbers already (c 2^-133 in
//     bfloat16, c 2^-24 in fp16, 16 times that in bits 4-7), so that one AND makes an operand of a tensor core.
//   * keys: a thread of an mma.sync operand needs, of the key of its row, a quarter of every group: with groups of 64 word (g, i)
//     of a row stands at (i / 2) * 2 G + 2 g + i % 2, so that a thread's words are side by side (16 bytes with 128 elements).
//   * values: a thread needs the same 8 elements of every group of four tokens: word (g, i) stands at i * G + g.  Of the tokens
//     that the four threads of a quad read together (2 t + c for t = 0 .. 3) the rows stand side by side (value_row), and with two groups
//     the 8-byte pieces of every other pair of rows are swapped by halves, so that these reads touch every bank once.
// With groups of another size words stand in their own order.
#pragma once
#include "common.cuh"

namespace leone {
namespace cache4 {

constexpr int kUnit = 16;           // tokens of a unit
constexpr int kMaxDim = 512;

__host__ __device__ constexpr int groups(int d) { return (d + 63) / 64; }
__host__ __device__ constexpr int row_bytes(int d) { return d / 2 + 4 * groups(d); }
__host__ __device__ constexpr bool dim_ok(int d) { return d > 0 && d <= kMaxDim && d % (8 * groups(d)) == 0; }

// Where the unit of tokens slot .. slot + 15 of (page, head) starts, in bytes; slot: a multiple of 16.
__host__ __device__ __forceinline__ long long unit_at(long long page, int n_kv, int kvh, int page_tokens, int slot, int d) {
  return ((page * n_kv + kvh) * page_tokens + slot) * row_bytes(d);
}
// Byte offsets inside a unit, of token t (0 .. 15).
__host__ __device__ __forceinline__ int key_word_at(int t, int w, int d) {
  const int G = groups(d);
  if (d == 64 * G) w = ((w & 7) >> 1) * 2 * G + 2 * (w >> 3) + (w & 1);
  return t * (d / 2) + 4 * w;
}
__host__ __device__ __forceinline__ int value_row(int t) { return (t & 8) | ((t & 7) >> 1) | ((t & 1) << 2); }
__host__ __device__ __forceinline__ int value_word_at(int t, int w, int d) {
  const int G = groups(d), row = value_row(t);
  if (d == 64 * G) {
    w = (w & 7) * G + (w >> 3);
    if (G == 2) w ^= ((row >> 1) & 1) << 3;
  }
  return row * (d / 2) + 4 * w;
}
__host__ __device__ __forceinline__ int scale_at(int t, int g, int d) { return kUnit * (d / 2) + 4 * (t * groups(d) + g); }

// Element e (0 .. 7) of a word.
__device__ __forceinline__ int code_of(uint32_t word, int e) { return (word >> (4 * (e >> 1) + 16 * (e & 1))) & 15; }
__device__ __forceinline__ float scale_of(uint32_t sz) { return __uint_as_float(sz << 16); }
__device__ __forceinline__ float offset_of(uint32_t sz) { return __uint_as_float(sz & 0xffff0000u); }

}  // namespace cache4
}  // namespace leone
