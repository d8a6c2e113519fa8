// Attention of one new token a sequence over the pages of a pool, for gfx950.
//   o = softmax(sm_scale q K^T) V over the sequence's first lens[b] rows, in one pass with a running maximum and sum.
#include <type_traits>

#include "kvx_common.h"

namespace kvx {
namespace {

constexpr int NT = 256;

// 8 values of a row in fp32: the lane's share
template <int D, int KV>
__device__ __forceinline__ void row_values(const uint8_t* row, int col, float scale, int zp, float (&x)[8]) {
  if constexpr (kv_is_plain(KV)) {
    const u32x4_t w = *(const u32x4_t*)(row + 16 * col);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = elem_lo<kv_elem_f16(KV)>(w[e]);
      x[2 * e + 1] = elem_hi<kv_elem_f16(KV)>(w[e]);
    }
  } else {
    u32x2_t c = *(const u32x2_t*)(row + (kv_is_u4(KV) ? u4_byte_off<D>(col) : 8 * col));
    if constexpr (kv_is_u4(KV)) c = u4_codes(c, u4_shift<D>(col));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)((int)((c[e >> 2] >> (8 * (e & 3))) & 0xff) - zp) * scale;
  }
}

// A workgroup for each (sequence, query head): D / 8 lanes hold a row, every group of lanes has a running maximum and sum of its own.
template <int D, int KV>
__global__ __launch_bounds__(NT) void paged_decode_kernel(const kvx_paged_decode_args a, const int shift, const float c) {
  constexpr bool PLAIN = kv_is_plain(KV), F16 = kv_elem_f16(KV);
  constexpr int LPR = D / 8, ES = PLAIN ? 2 : 1, GROUPS = NT / LPR;
  __shared__ float out[GROUPS][D], top[GROUPS], sum[GROUPS];
  const kvx_pages& p = a.pages;
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / (a.Hq / p.Hkv), col = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int n = min(max(a.lens[b], 0), a.max_pages << shift);
  float q[8], acc[8], m = -INFINITY, l = 0.0f;
  row_values<D, F16 ? KVX_KV_F16 : KVX_KV_BF16>((const uint8_t*)((const uint16_t*)a.q + b * a.q_stride_b + hq * a.q_stride_h), col, 0.0f, 0, q);
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
  for (int t = group; t < n; t += GROUPS) {
    const int page = a.block_table[b * a.bt_stride_b + (t >> shift)], place = t & (p.page_size - 1);
    if (page < 0 || page >= p.num_pages) continue;  // the same for all lanes of a row
    const int64_t s = (int64_t)page * p.qs_stride_page + h * p.qs_stride_h + place;
    float x[8], dot = 0.0f;
    row_values<D, KV>((const uint8_t*)p.k + ((int64_t)page * p.k_stride_page + h * p.k_stride_h + (int64_t)place * p.k_stride_t) * ES, col, PLAIN ? 0.0f : p.k_scale[s],
                      PLAIN ? 0 : p.k_zp[s], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) dot = fmaf(x[e], q[e], dot);
#pragma unroll
    for (int off = 1; off < LPR; off <<= 1) dot += __shfl_xor(dot, off, 64);
    dot *= c;
    const float mn = fmaxf(m, dot), al = fast_exp2(m - mn), w = fast_exp2(dot - mn);
    m = mn;
    l = l * al + w;
    row_values<D, KV>((const uint8_t*)p.v + ((int64_t)page * p.v_stride_page + h * p.v_stride_h + (int64_t)place * p.v_stride_t) * ES, col, PLAIN ? 0.0f : p.v_scale[s],
                      PLAIN ? 0 : p.v_zp[s], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, x[e], acc[e] * al);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) out[group][8 * col + e] = acc[e];
  if (col == 0) {
    top[group] = m;
    sum[group] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.0f;
  for (int g = 0; g < GROUPS; ++g) M = fmaxf(M, top[g]);
  for (int g = 0; g < GROUPS; ++g) L += M > -INFINITY ? sum[g] * fast_exp2(top[g] - M) : sum[g];  // a NaN goes on
  for (int d = 2 * threadIdx.x; d < D; d += 2 * NT) {
    float o0 = 0.0f, o1 = 0.0f;
    for (int g = 0; g < GROUPS; ++g) {
      const float w = M > -INFINITY ? fast_exp2(top[g] - M) : 1.0f;
      o0 += out[g][d] * w;
      o1 += out[g][d + 1] * w;
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *(uint32_t*)((uint16_t*)a.o + b * a.o_stride_b + hq * a.o_stride_h + d) = pack_pair<F16>(o0 * inv, o1 * inv);
  }
  if (a.lse && threadIdx.x == 0) a.lse[(int64_t)b * a.Hq + hq] = L == 0.0f ? -INFINITY : M + fast_log2(L);
}

template <int D>
void launch_head(const kvx_paged_decode_args& a, hipStream_t st) {
  const float c = a.sm_scale * kLog2e;
  auto go = [&](auto kv) {
    hipLaunchKernelGGL((paged_decode_kernel<D, decltype(kv)::value>), dim3(a.Hq, a.B), dim3(NT), 0, st, a, __builtin_ctz(a.pages.page_size), c);
  };
  switch (a.pages.kv_dtype) {
#define KVX_PAGES_CASE(KV) case KV: go(std::integral_constant<int, KV>{}); break;
    KVX_PAGES_CASE(KVX_KV_BF16)
    KVX_PAGES_CASE(KVX_KV_F16)
    KVX_PAGES_CASE(KVX_KV_U8)
    KVX_PAGES_CASE(KVX_KV_U4)
    KVX_PAGES_CASE(KVX_KV_U8_F16)
    KVX_PAGES_CASE(KVX_KV_U4_F16)
#undef KVX_PAGES_CASE
  }
}

}  // namespace

size_t paged_decode_workspace(const kvx_paged_decode_args& a) { return 0; }

int launch_paged_decode(const kvx_paged_decode_args& a, hipStream_t st) {
  if (a.pages.D == 256) launch_head<256>(a, st);
  else if (a.pages.D == 128) launch_head<128>(a, st);
  else launch_head<64>(a, st);
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
