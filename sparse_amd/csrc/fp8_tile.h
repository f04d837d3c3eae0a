// What the two 8-bit kernels of many rows share: arguments, which tile a workgroup has, counted waits.
#pragma once

#include "fp8.h"
#include "prefill_tiles.h"

namespace sparse {

constexpr int tl_wait(int vmcnt) { return 0x0F70 | (vmcnt & 15) | ((vmcnt >> 4) << 14); }
static_assert(tl_wait(20) == kWaitVmcnt20, "the encoding of the 16-bit kernels");

template <typename T>
__device__ __forceinline__ T* uniform_ptr(T* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<T*>((static_cast<uint64_t>(hi) << 32) | lo);
}

// A power of two from 2^kLow to 2^kHigh: its exponent is all there is to it.
template <int kLow, int kHigh>
__device__ __forceinline__ bool tl_is_exponent(float v) {
  constexpr uint32_t lo = static_cast<uint32_t>(127 + kLow) << 23, hi = static_cast<uint32_t>(127 + kHigh) << 23;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x807fffffu) == 0 && b - lo <= hi - lo;
}

struct TileArgs {
  F8Product p;
  const PfTile* map;       // NULL: dense operands only, the tile comes from the block number
  const int32_t* qhdr;
  uint32_t topk_magic;     // ceil(2^32 / topk); 0 for topk == 1
  int32_t mt, nt, rows;    // row and column tiles when map is NULL, rows per tile
  // gate/up: where the quantised rows go
  uint8_t *q_r, *qs_r, *q_s, *qs_s;
};

// The queue entry of this workgroup, wavefront-uniform; false: none (the grid is sized for the longest possible queue).
__device__ __forceinline__ bool tl_queued(const TileArgs& a, int& slot, int& r0, int& M, int& bn) {
  const int xcd = blockIdx.x % kPfXcds, rank = blockIdx.x / kPfXcds;
  if (rank >= a.qhdr[kPfXcds + xcd]) return false;
  const PfTile tile = a.map[a.qhdr[xcd] + rank];
  slot = __builtin_amdgcn_readfirstlane(tile.slot);
  r0 = __builtin_amdgcn_readfirstlane(tile.r0);
  M = __builtin_amdgcn_readfirstlane(tile.rows);
  bn = __builtin_amdgcn_readfirstlane(tile.bn);
  return M > 0;
}

inline int64_t tl_queue_grid(int cap) { return (static_cast<int64_t>(cap - 1) / kPfXcds + 2) * kPfXcds; }
inline uint32_t tl_magic(int topk) { return topk == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + topk - 1) / topk); }

}  // namespace sparse
