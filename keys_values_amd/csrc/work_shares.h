// Work of which only the device knows how much there is, dealt out to a fixed number of workgroups (paged_decode.hip, paged_select.hip).
#pragma once
#include "kvx_common.h"

namespace kvx {
namespace {

// Inclusive sum over the lanes of a wavefront, on the vector ALU.
__device__ __forceinline__ int scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to the odd rows
  return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to the upper half
}

// The shares of `total` units: workgroup w begins with unit first(w).
struct Shares {
  int workgroups, each, rest;
  __device__ __forceinline__ Shares(int total, int n) : workgroups(n), each(total / n), rest(total - each * n) {}
  __device__ __forceinline__ int first(int w) const { return min(w, workgroups) * each + min(w, rest); }
  __device__ __forceinline__ int owner(int unit) const {
    const int big = rest * (each + 1);
    return unit < big ? unit / (each + 1) : rest + (unit - big) / each;
  }
};

}  // namespace
}  // namespace kvx
