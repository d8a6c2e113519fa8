// Rotary position encoding of a ragged batch for gfx950 (HBM-bound, one pass, in place): every token has a position of its own, the pairs of a head are
// its halves' or interleaved, and may cover its first part alone; the head is normalised first where weights are given.
//   y = x / (|x|_2 / sqrt(D) + eps) * w;   (a, b) -> (a cos - b sin, b cos + a sin),   in fp32, rounded once.
#include <type_traits>

#include "kvx_common.h"

namespace kvx {
namespace {

constexpr int NT = 256;

template <int LPR>
__device__ __forceinline__ float sum_over_row(float v) {
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// A workgroup a token; LPR = D / 8 lanes a head, which hold 8 values each: pairs never leave a lane. Interleaved pairs lie side by side, and a lane holds a stretch of 8;
// pairs of halves: four values of either half of the rotated part. Lanes behind that part hold stretches.
template <int D, bool F16, bool INTERLEAVED>
__global__ __launch_bounds__(NT) void rotary_kernel(const kvx_rotary_args a, const float factor) {
  constexpr int LPR = D / 8;
  const int t = blockIdx.x, pos = a.positions[t];
  if (pos < 0 || pos >= a.table_rows) return;
  const int col = threadIdx.x % LPR, heads = a.Hq + a.Hkv, half = a.rotary_dim / 2;
  const bool turns = 8 * col < a.rotary_dim, split = !INTERLEAVED && turns;
  const int lo = split ? 4 * col : 8 * col, hi = split ? half + 4 * col : lo + 4;
  f32x4_t cv = {1.0f, 1.0f, 1.0f, 1.0f}, sv = {0.0f, 0.0f, 0.0f, 0.0f};
  if (turns) {
    cv = *(const f32x4_t*)(a.cos + (int64_t)pos * half + 4 * col);
    sv = *(const f32x4_t*)(a.sin + (int64_t)pos * half + 4 * col);
  }
  uint16_t* token = (uint16_t*)a.qkv + t * a.stride_t;
  for (int first = 0; first < heads; first += NT / LPR) {  // all lanes stay: heads are reduced across them
    const int head = first + (int)threadIdx.x / LPR, h = min(head, heads - 1);
    uint16_t* p = token + h * D;
    const u32x2_t x0 = *(const u32x2_t*)(p + lo), x1 = *(const u32x2_t*)(p + hi);
    float y[8] = {elem_lo<F16>(x0[0]), elem_hi<F16>(x0[0]), elem_lo<F16>(x0[1]), elem_hi<F16>(x0[1]),
                  elem_lo<F16>(x1[0]), elem_hi<F16>(x1[0]), elem_lo<F16>(x1[1]), elem_hi<F16>(x1[1])};
    if (a.q_weight) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
      const float n = sqrtf(sum_over_row<LPR>(ss)) * factor + a.eps;
      const float* w = h < a.Hq ? a.q_weight : a.k_weight;
      const f32x4_t w0 = *(const f32x4_t*)(w + lo), w1 = *(const f32x4_t*)(w + hi);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] / n * (e < 4 ? w0[e] : w1[e - 4]);
    }
    float z[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = INTERLEAVED ? 2 * e : e, j = INTERLEAVED ? 2 * e + 1 : e + 4;
      z[i] = y[i] * cv[e] - y[j] * sv[e];
      z[j] = y[j] * cv[e] + y[i] * sv[e];
    }
    if (!turns)
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = y[e];
    if (head < heads) {
      *(u32x2_t*)(p + lo) = u32x2_t{pack_pair<F16>(z[0], z[1]), pack_pair<F16>(z[2], z[3])};
      *(u32x2_t*)(p + hi) = u32x2_t{pack_pair<F16>(z[4], z[5]), pack_pair<F16>(z[6], z[7])};
    }
  }
}

template <int D>
void launch_head(const kvx_rotary_args& a, hipStream_t st) {
  const float factor = 1.0f / sqrtf((float)D);
  auto go = [&](auto f16, auto interleaved) {
    hipLaunchKernelGGL((rotary_kernel<D, decltype(f16)::value, decltype(interleaved)::value>), dim3((unsigned)a.tokens), dim3(NT), 0, st, a, factor);
  };
  if (a.elem_dtype == KVX_KV_F16) {
    if (a.interleaved) go(std::true_type{}, std::true_type{});
    else go(std::true_type{}, std::false_type{});
  } else {
    if (a.interleaved) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
  }
}

}  // namespace

int launch_rotary(const kvx_rotary_args& a, hipStream_t st) {
  if (a.D == 256) launch_head<256>(a, st);
  else if (a.D == 128) launch_head<128>(a, st);
  else launch_head<64>(a, st);
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
