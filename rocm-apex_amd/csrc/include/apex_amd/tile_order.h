// Order in which a GEMM's workgroups take its tiles.
#pragma once
#include "apex_amd/device.h"

namespace apex_amd {

// XCD-aware, bijective remap of the linear workgroup id (each XCD gets a contiguous band), then
// GROUP_M-grouped tile order; nwg = tiles_m * tiles_n
__device__ __forceinline__ void tile_coords(int nwg, int tiles_m, int tiles_n, int& bm, int& bn) {
  const int orig = blockIdx.x;
  const int xcd = orig % 8, q = nwg / 8, r = nwg % 8;
  const int wgid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig / 8;
  constexpr int GROUP_M = 8;
  const int group = wgid / (GROUP_M * tiles_n);
  const int first_m = group * GROUP_M;
  const int gm = min(tiles_m - first_m, GROUP_M);
  bm = first_m + (wgid % (GROUP_M * tiles_n)) % gm;
  bn = (wgid % (GROUP_M * tiles_n)) / gm;
}

}  // namespace apex_amd
