// Sums over a wave without LDS round trips.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cdx {

typedef unsigned long long u64;

// Sum over the lanes up to this one (DPP; every lane of the wave takes part).  The last lane has the wave's.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp(u64 v) {
  return (u64)(uint32_t)dpp<CTRL, ROWS>((int)(v >> 32)) << 32 | (uint32_t)dpp<CTRL, ROWS>((int)v);
}
template <typename T>
__device__ __forceinline__ T wave_inclusive(T v) {
  v += dpp<0x111, 0xf>(v);  // from 1, 2, 4 and 8 lanes below in the row of 16
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // the row before's last lane, then the first half's
  v += dpp<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ int read_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ u64 read_lane(u64 v, int lane) {
  return (u64)(uint32_t)read_lane((int)(v >> 32), lane) << 32 | (uint32_t)read_lane((int)v, lane);
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  return read_lane(wave_inclusive(v), 63);
}

}  // namespace cdx
