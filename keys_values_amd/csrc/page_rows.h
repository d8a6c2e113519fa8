// What the kernels of a pool's pages share: rows of K and V to codes, and the choice of a kernel by head size and store.
#pragma once
#include <type_traits>

#include "row_write.h"

namespace kvx {
namespace {

// Codes (bytes) of the lane's 8 values of a K and a V row, as the row quantiser forms them. Even lanes work out the scale and zero point of the K row, odd
// ones of the V row, and each fetches 1 / scale and the zero point of the other from its neighbour; (scale, zp): the lane's own row's.
template <int LPR, int BITS, bool F16>
__device__ __forceinline__ void quantize_kv(const u32x4_t& k, const u32x4_t& v, u32x2_t& kc, u32x2_t& vc, float& scale, int32_t& zp) {
  float xk[8], xv[8], mnk, mxk, mnv, mxv;
  row_extremes<LPR, F16>(k, xk, mnk, mxk);
  row_extremes<LPR, F16>(v, xv, mnv, mxv);
  const bool odd = __lane_id() & 1u;
  quant_params(odd ? mnv : mnk, odd ? mxv : mxk, scale, zp, BITS == 8 ? 255.0f : 15.0f);
  const int inv = __builtin_bit_cast(int, 1.0f / scale), zf = __builtin_bit_cast(int, (float)zp);
  auto of_k = [](int x) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(x, 0xA0, 0xf, 0xf, true)); };  // quad_perm [0,0,2,2]
  auto of_v = [](int x) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(x, 0xF5, 0xf, 0xf, true)); };  // quad_perm [1,1,3,3]
  const float ik = of_k(inv), zk = of_k(zf), iv = of_v(inv), zv = of_v(zf);
  if constexpr (BITS == 8) {
    kc = u32x2_t{codes4_u8(xk[0], xk[1], xk[2], xk[3], ik, zk), codes4_u8(xk[4], xk[5], xk[6], xk[7], ik, zk)};
    vc = u32x2_t{codes4_u8(xv[0], xv[1], xv[2], xv[3], iv, zv), codes4_u8(xv[4], xv[5], xv[6], xv[7], iv, zv)};
  } else {
    kc = u32x2_t{codes4_u4(xk[0], xk[1], xk[2], xk[3], ik, zk), codes4_u4(xk[4], xk[5], xk[6], xk[7], ik, zk)};
    vc = u32x2_t{codes4_u4(xv[0], xv[1], xv[2], xv[3], iv, zv), codes4_u4(xv[4], xv[5], xv[6], xv[7], iv, zv)};
  }
}

// f(head size, store) for the pages' kernels
template <typename F>
void by_store(const kvx_pages& p, F f) {
  auto with_d = [&](auto d) {
    switch (p.kv_dtype) {
#define KVX_PAGES_CASE(KV) case KV: f(d, std::integral_constant<int, KV>{}); break;
      KVX_PAGES_CASE(KVX_KV_BF16)
      KVX_PAGES_CASE(KVX_KV_F16)
      KVX_PAGES_CASE(KVX_KV_U8)
      KVX_PAGES_CASE(KVX_KV_U4)
      KVX_PAGES_CASE(KVX_KV_U8_F16)
      KVX_PAGES_CASE(KVX_KV_U4_F16)
#undef KVX_PAGES_CASE
    }
  };
  if (p.D == 256) with_d(std::integral_constant<int, 256>{});
  else if (p.D == 128) with_d(std::integral_constant<int, 128>{});
  else with_d(std::integral_constant<int, 64>{});
}

}  // namespace
}  // namespace kvx
