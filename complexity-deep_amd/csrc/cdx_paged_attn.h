// Lane helpers of attention over pages with v_mfma_f32_16x16x32_bf16 (rows are slots, columns queries).
#pragma once

#include "cdx_paged.h"

namespace cdx {

constexpr float kLog2e = 1.4426950408889634f;

// Both values that lanes l and l ^ 16 (l ^ 32) hold, reduced.
__device__ __forceinline__ float max_over_groups(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// The low (high) halves of two words, side by side.
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// Both bf16 of a word, Inf and NaN as the largest finite value of their sign: as signed integers the
// positive ones lie above it, as unsigned integers the negative ones.
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
  typedef __attribute__((ext_vector_type(2))) short i16x2;
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  const i16x2 i = __builtin_elementwise_min(__builtin_bit_cast(i16x2, x), i16x2{0x7f7f, 0x7f7f});
  const u16x2 u = __builtin_elementwise_min(__builtin_bit_cast(u16x2, i), u16x2{0xff7f, 0xff7f});
  return __builtin_bit_cast(uint32_t, u);
}

template <int DPL>
struct Piece;
template <>
struct Piece<4> {
  typedef uint2 type;
};
template <>
struct Piece<8> {
  typedef uint4 type;
};

constexpr int kPagedTile = 32;   // slots of a wave's step
constexpr int kPagedWaves = 8;   // of a block
constexpr int kPagedMaxSplits = 256;
// Blocks that the slots of one block's queries are split over.
int paged_splits(int64_t blocks, int64_t cap);

}  // namespace cdx
