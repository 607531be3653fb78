// The paged KV cache as the kernels see it, and the lane helpers of passes over heads.
#pragma once

#include "cdx_common.h"

namespace cdx {

// Pages [num_pages][nkv][page size][D]; sequence b's slot t lies in row t % page size of page
// table[b][t / page size].  A table entry outside the pool stands for a page that is not there:
// its slots are neither read nor written, and attention over one is NaN.
struct PagedTable {
  const int32_t* table;
  int64_t ld;         // row stride of the table
  int32_t width;      // pages of a sequence
  int32_t num_pages;  // pages of the pool
  int32_t log2_page;

  __device__ __forceinline__ int32_t capacity() const { return width << log2_page; }
  // Row index in the pool of slot t of (sequence b, head h), or -1.  (0 <= t < capacity)
  __device__ __forceinline__ int64_t row(int64_t b, int h, int nkv, int32_t t) const {
    const int32_t page = table[b * ld + (t >> log2_page)];
    if ((uint32_t)page >= (uint32_t)num_pages) return -1;
    return (((int64_t)page * nkv + h) << log2_page) + (t & ((1 << log2_page) - 1));
  }
};

// Checks of the arguments that every paged entry point shares; fills *t.
int paged_table(const char* name, const int32_t* table, int64_t table_ld, int64_t width, int64_t num_pages,
                int32_t page_size, int64_t B, int32_t nkv, int32_t hd, PagedTable* t);

// Sum over each row of 16 lanes, returned to all of them.
__device__ __forceinline__ float head16_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, false));
  return v;
}

// Four consecutive values of a row, as floats.
__device__ __forceinline__ void head_load4(const float* p, float* f) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}
__device__ __forceinline__ void head_load4(const uint16_t* p, float* f) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void head_store4(uint16_t* p, const float* f) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
}

}  // namespace cdx
