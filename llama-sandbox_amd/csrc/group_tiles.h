// group_tiles.h -- grouped rows (offsets of experts, or of adapters) cut into tiles.
#pragma once

#include "device_common.h"

// The rows of one tile: expert e (-1: none left), rows [r0, r0 + n); only: the expert has no others.
struct row_tile {
  int e, r0, n, only;
};

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8: within rows of 16 lanes
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);  // row_bcast15: the last lane of rows 0 and 2 to rows 1 and 3
  v = dpp_add<0x143, 0xC>(v);  // row_bcast31: lane 31 to rows 2 and 3
  return v;
}

// Tile `item` of the grouped rows cut into tiles of at most BM: expert e has
// ceil(c_e / BM) of them, in expert order.  Every wave finds it for itself: lane
// l counts the tiles of E / 64 experts side by side (all offsets are asked for
// at once), a scan over the lanes finds the lane that holds the item.  Offsets are
// held to [0, M].  PER: experts a lane, at least E / 64.
template <int PER>
__device__ __forceinline__ row_tile row_tile_search(const int32_t *offsets, int E, int M, int item, int BM) {
  const int lane = threadIdx.x & 63;
  int o[PER + 1];
#pragma unroll
  for (int i = 0; i <= PER; i++) o[i] = offsets[min(PER * lane + i, E)];  // (past the end: equal, no rows)
  int c[PER], sum = 0;
#pragma unroll
  for (int i = 0; i <= PER; i++) o[i] = min(max(o[i], 0), M);
#pragma unroll
  for (int i = 0; i < PER; i++) {
    c[i] = o[i + 1] > o[i] ? (o[i + 1] - o[i] - 1) / BM + 1 : 0;
    sum += c[i];
  }
  int at = wave_scan(sum) - sum;
  const uint64_t here = __ballot(at <= item && item < at + sum);
  if (!here) return {-1, 0, 0, 0};
  row_tile t = {-1, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < PER; i++) {
    if (at <= item && item < at + c[i]) {
      const int r0 = o[i] + (item - at) * BM;
      t = {PER * lane + i, r0, o[i + 1] - r0 < BM ? o[i + 1] - r0 : BM, c[i] == 1};
    }
    at += c[i];
  }
  const int owner = __ffsll((unsigned long long)here) - 1;
  return {__builtin_amdgcn_readlane(t.e, owner), __builtin_amdgcn_readlane(t.r0, owner), __builtin_amdgcn_readlane(t.n, owner),
          __builtin_amdgcn_readlane(t.only, owner)};
}
__device__ __forceinline__ row_tile find_row_tile(const int32_t *offsets, int E, int M, int item, int BM) {
  if (E <= 64) return row_tile_search<1>(offsets, E, M, item, BM);
  if (E <= 256) return row_tile_search<4>(offsets, E, M, item, BM);
  return row_tile_search<16>(offsets, E, M, item, BM);
}
