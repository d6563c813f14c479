// Packed rows of several requests: finding a request from the row numbers on the device.
#pragma once

#include "common.hpp"

namespace dlt {

// Row number i of `starts`, inside the tensor whatever it holds.
__device__ __forceinline__ int packed_start(const int32_t* starts, int i, int total) {
  return min(max(starts[i], 0), total);
}

// One tile of a request's rows: rows [row0, row0 + rows) of the tensor belong to the request, the
// tile is its tile-th. req == n: rows of no request (before the first or behind the last); req < 0:
// no such item.
struct PackedItem {
  int req, tile, row0, rows;
};

// The rows of lane i's request (of n, from `first` on; n and n + 1 the rows of none, with `rest`).
__device__ __forceinline__ void packed_rows(const int32_t* starts, int n, int total, bool rest,
                                            int i, int& r0, int& len) {
  r0 = 0, len = 0;
  if (i < n) {
    r0 = packed_start(starts, i, total);
    len = max(packed_start(starts, i + 1, total) - r0, 0);
  } else if (rest && i == n) {
    len = packed_start(starts, 0, total);
  } else if (rest && i == n + 1) {
    r0 = packed_start(starts, n, total);
    len = total - r0;
  }
}

// Inclusive prefix sum over the lanes.
__device__ __forceinline__ int wave_prefix(int v) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

// Item `item` of the tiles of `block` (row, head) pairs, `group` heads a row, over n requests and,
// with `rest`, over the rows of none. A wavefront looks 64 requests up at a time: there are about
// as many dependent loads as n / 64, not a search's log n.
__device__ __forceinline__ PackedItem packed_item(const int32_t* starts, int n, int total,
                                                  int group, int block, bool rest, int item) {
  const int lane = threadIdx.x & (kWave - 1);
  int before = 0;
  for (int c = 0; c < n + 2; c += kWave) {
    int r0, len;
    packed_rows(starts, n, total, rest, c + lane, r0, len);
    const int count = (len * group + block - 1) / block;
    const int upto = wave_prefix(count);
    const uint64_t past = __ballot(before + upto > item);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      PackedItem it;
      it.req = min(c + l, n);
      it.tile = item - before - __builtin_amdgcn_readlane(upto, l) +
                __builtin_amdgcn_readlane(count, l);
      it.row0 = __builtin_amdgcn_readlane(r0, l);
      it.rows = __builtin_amdgcn_readlane(len, l);
      return it;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return PackedItem{-1, 0, 0, 0};
}

}  // namespace dlt
