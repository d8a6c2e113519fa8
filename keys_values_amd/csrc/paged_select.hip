// Which pages of a sequence a query attends to, for gfx950: bounds of a page's keys, and the choice by what they allow.
//   low, high = min, max over the page's keys, value by value (rows of codes: of the rows that they stand for, rounded to 16 bits);
//   score = max over the query heads of a KV head of sum_d max(q_d low_d, q_d high_d) = sum_d (q+_d high_d + q-_d low_d), which no logit of the page exceeds.
#include <type_traits>

#include "page_rows.h"

namespace kvx {
namespace {

// Minimum and maximum that hand on a NaN (llvm.minimum: v_minimum3_f32)
__device__ __forceinline__ float lowest(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float highest(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A wavefront a (page, KV head) or, for larger pages, several; D / 8 lanes a row. Block: W wavefronts.
template <int D, int KV, int W>
__global__ __launch_bounds__(64 * W) void paged_bounds_kernel(const kvx_paged_bounds_args a, const int shift, const int most) {
  constexpr bool PLAIN = kv_is_plain(KV), U4 = kv_is_u4(KV), F16 = kv_elem_f16(KV);
  constexpr int LPR = D / 8, ROWS = 64 * W / LPR, ES = PLAIN ? 2 : 1;
  const kvx_pages& p = a.pages;
  const int64_t item = blockIdx.x;
  const int h = (int)(item % p.Hkv), j = (int)(item / p.Hkv % most), b = (int)(item / p.Hkv / most);
  const int cap = a.max_pages << shift, len = min(max(a.lens[b], 0), cap);
  const int i = ((len + p.page_size - 1) >> shift) - 1 - j;  // the sequence's page, from the last one back
  if (i < 0 || (int64_t)(i + 1) * p.page_size <= (int64_t)len - a.tokens) return;
  const int page = a.block_table[b * a.bt_stride_b + i];
  if ((uint32_t)page >= (uint32_t)p.num_pages) return;
  const int rows = min(len - (i << shift), p.page_size), col = threadIdx.x % LPR, first = threadIdx.x / LPR;
  const uint8_t* k = (const uint8_t*)p.k + ((int64_t)page * p.k_stride_page + h * p.k_stride_h) * ES;
  const int64_t q = (int64_t)page * p.qs_stride_page + h * p.qs_stride_h;
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
  for (int r = first; r < rows; r += ROWS) {
    const uint8_t* at = k + (int64_t)r * p.k_stride_t * ES;
    float x[8];
    if constexpr (PLAIN) {
      const u32x4_t w = *(const u32x4_t*)(at + 16 * col);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = elem_lo<F16>(w[e]);
        x[2 * e + 1] = elem_hi<F16>(w[e]);
      }
    } else {
      u32x2_t c = *(const u32x2_t*)(at + (U4 ? (int)u4_byte_off<D>(col) : 8 * col));
      if constexpr (U4) c = u4_codes(c, u4_shift<D>(col));
      const float scale = p.k_scale[q + r];
      const int32_t zp = p.k_zp[q + r];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)((int32_t)((c[e >> 2] >> (8 * (e & 3))) & 0xff) - zp) * scale;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = lowest(lo[e], x[e]);
      hi[e] = highest(hi[e], x[e]);
    }
  }
#pragma unroll
  for (int step = LPR; step < 64; step *= 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = lowest(lo[e], __shfl_xor(lo[e], step, 64));
      hi[e] = highest(hi[e], __shfl_xor(hi[e], step, 64));
    }
  }
  if constexpr (W > 1) {
    __shared__ float joined[W][2][D];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < LPR) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        joined[wave][0][8 * col + e] = lo[e];
        joined[wave][1][8 * col + e] = hi[e];
      }
    }
    __syncthreads();
    if (threadIdx.x >= LPR) return;
    for (int w = 1; w < W; ++w) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = lowest(lo[e], joined[w][0][8 * col + e]);
        hi[e] = highest(hi[e], joined[w][1][8 * col + e]);
      }
    }
  }
  if (threadIdx.x >= LPR) return;
  uint16_t* to = (uint16_t*)a.bounds + (int64_t)page * a.b_stride_page + h * a.b_stride_h + 8 * col;
  *(u32x4_t*)to = u32x4_t{pack_pair<F16>(lo[0], lo[1]), pack_pair<F16>(lo[2], lo[3]), pack_pair<F16>(lo[4], lo[5]), pack_pair<F16>(lo[6], lo[7])};
  *(u32x4_t*)(to + a.b_stride_side) = u32x4_t{pack_pair<F16>(hi[0], hi[1]), pack_pair<F16>(hi[2], hi[3]), pack_pair<F16>(hi[4], hi[5]), pack_pair<F16>(hi[6], hi[7])};
}

// ---- the choice ------------------------------------------------------------------------------------------------------------------

constexpr uint32_t kNever = 0u, kInfinite = 0xfffffffeu, kAlways = 0xffffffffu;

// Keys of scores: unsigned numbers in their order, between kNever and kInfinite. What is not finite counts as infinite.
__device__ __forceinline__ uint32_t key_of(double sum) {
  const float s = (float)sum + 0.0f;  // no -0
  const uint32_t bits = __float_as_uint(s);
  if (!(fabsf(s) < INFINITY)) return kInfinite;
  return (bits >> 31) ? ~bits : bits | 0x80000000u;
}

struct SelectParams {
  kvx_paged_select_args a;
  uint32_t* keys;  // (B, Hkv, max_pages)
  int parts;       // workgroups of a (sequence, KV head)
};
__device__ __forceinline__ int pages_of_sequence(const kvx_paged_select_args& a, int b) {
  const int len = max(a.lens[b], 0);
  return (int)min(((int64_t)len + a.page_size - 1) / a.page_size, (int64_t)a.max_pages);
}

constexpr int SCORED = 64;  // pages of a workgroup

// D / 8 lanes a page. Products of 16-bit values are exact in 32 bits, and their sums, in 64, differ with the order by less than what the rounding to 32 sees.
template <int D, bool F16>
__global__ __launch_bounds__(NTHREADS) void select_score_kernel(const SelectParams p) {
  constexpr int LPR = D / 8, ROWS = NTHREADS / LPR;
  const kvx_paged_select_args& a = p.a;
  const int pair = blockIdx.x / p.parts, part = blockIdx.x - pair * p.parts, b = pair / a.Hkv, h = pair - b * a.Hkv, n = pages_of_sequence(a, b), G = a.Hq / a.Hkv;
  const int col = threadIdx.x % LPR;
  for (int i = part * SCORED + threadIdx.x / LPR; i < min((part + 1) * SCORED, n); i += ROWS) {
    const int page = a.block_table[b * a.bt_stride_b + i];
    uint32_t key = kNever;
    if ((uint32_t)page < (uint32_t)a.num_pages) {
      const uint16_t* at = (const uint16_t*)a.bounds + (int64_t)page * a.b_stride_page + h * a.b_stride_h + 8 * col;
      const u32x4_t lo = *(const u32x4_t*)at, hi = *(const u32x4_t*)(at + a.b_stride_side);
      for (int g = 0; g < G; ++g) {
        const u32x4_t q = *(const u32x4_t*)((const uint16_t*)a.q + b * a.q_stride_b + (int64_t)(h * G + g) * a.q_stride_h + 8 * col);
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = e & 1 ? elem_hi<F16>(q[e >> 1]) : elem_lo<F16>(q[e >> 1]);
          const float l = e & 1 ? elem_hi<F16>(lo[e >> 1]) : elem_lo<F16>(lo[e >> 1]), u = e & 1 ? elem_hi<F16>(hi[e >> 1]) : elem_lo<F16>(hi[e >> 1]);
          sum += (double)(x > 0.0f ? x : 0.0f) * (double)u + (double)(x > 0.0f ? 0.0f : x) * (double)l;
        }
#pragma unroll
        for (int step = 1; step < LPR; step *= 2) sum += __shfl_xor(sum, step, 64);
        key = max(key, key_of(sum));
      }
      if (i < a.first || i >= n - a.last) key = kAlways;
    }
    if (col == 0) p.keys[(int64_t)pair * a.max_pages + i] = key;
  }
}

// The `count` largest keys of a (sequence, KV head), of equal ones the first, in order of their pages: the last key that is taken is found from its upper bits
// down, by counting.
constexpr int CHOOSERS = 1024;
__global__ __launch_bounds__(CHOOSERS) void select_choose_kernel(const SelectParams p) {
  const kvx_paged_select_args& a = p.a;
  const int pair = blockIdx.x, b = pair / a.Hkv, n = pages_of_sequence(a, b), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int WAVES = CHOOSERS / 64, BINS = 2048;
  __shared__ int counts[BINS], sums[WAVES], at_bin, at_rest;
  const uint32_t* keys = p.keys + (int64_t)pair * a.max_pages;
  int32_t* out = a.chosen + (int64_t)pair * a.count;
  // ---- the key of rank `count`: `rest` of those equal to it are taken
  uint32_t prefix = 0u;
  int rest = a.count, bits = 0;
  for (const int width : {11, 11, 10}) {
    const int shift = 32 - bits - width;
    for (int i = tid; i < BINS; i += CHOOSERS) counts[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += CHOOSERS) {
      const uint32_t key = keys[i];
      if (bits == 0 || key >> (32 - bits) == prefix) atomicAdd(&counts[(key >> shift) & ((1u << width) - 1)], 1);
    }
    __syncthreads();
    // from the largest bin down: a thread has two
    const int c1 = counts[BINS - 1 - 2 * tid], c0 = counts[BINS - 2 - 2 * tid];
    int upto = c0 + c1;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int x = __shfl_up(upto, step, 64);
      if (lane >= step) upto += x;
    }
    if (lane == 63) sums[wave] = upto;
    if (tid == 0) at_bin = -1;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += sums[w];
    const int before = upto - c0 - c1;
    if (before < rest && rest <= upto) {
      const bool second = before + c1 < rest;
      at_bin = BINS - 1 - 2 * tid - (second ? 1 : 0);
      at_rest = rest - before - (second ? c1 : 0);
    }
    __syncthreads();
    if (at_bin < 0) break;  // fewer pages than are asked for, in the first pass: all of them
    prefix = prefix << width | (uint32_t)at_bin;
    rest = at_rest;
    bits += width;
    __syncthreads();
  }
  const bool all = bits == 0;
  // ---- what is taken, in order
  int taken = 0, equal = 0;  // so far, by the workgroup
  for (int begin = 0; begin < n; begin += CHOOSERS) {
    const int i = begin + tid;
    const uint32_t key = i < n ? keys[i] : kNever;
    const bool tie = !all && key == prefix && key != kNever, above = key != kNever && (all || key > prefix);
    const unsigned long long ties = __ballot(tie);
    __syncthreads();
    if (lane == 0) sums[wave] = __popcll(ties);
    __syncthreads();
    int ties_before = equal + __popcll(ties & ((1ull << lane) - 1)), ties_here = 0;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) ties_before += sums[w];
      ties_here += sums[w];
    }
    equal += ties_here;
    const bool take = above || (tie && ties_before < rest);
    const unsigned long long takes = __ballot(take);
    __syncthreads();
    if (lane == 0) sums[wave] = __popcll(takes);
    __syncthreads();
    int to = taken + __popcll(takes & ((1ull << lane) - 1)), here = 0;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) to += sums[w];
      here += sums[w];
    }
    taken += here;
    if (take && to < a.count) out[to] = i;
  }
  for (int i = taken + tid; i < a.count; i += CHOOSERS) out[i] = -1;
}

}  // namespace

int launch_paged_bounds(const kvx_paged_bounds_args& a, hipStream_t st) {
  const kvx_pages& p = a.pages;
  const int64_t lie_in = ((int64_t)a.tokens + 2 * p.page_size - 2) / p.page_size;  // pages that so many tokens lie in, at most
  const int most = (int)(lie_in < a.max_pages ? lie_in : a.max_pages);
  const int64_t items = (int64_t)a.B * most * p.Hkv;
  KVX_REQUIRE(items < (1 << 22), KVX_ERR_UNSUPPORTED, "kvx_paged_bounds: %d sequences of up to %d pages, %d KV heads in one call", a.B, most, p.Hkv);
  by_store(p, [&](auto d, auto kv) {
    auto go = [&](auto w) {
      hipLaunchKernelGGL((paged_bounds_kernel<decltype(d)::value, decltype(kv)::value, decltype(w)::value>), dim3((unsigned)items), dim3(64 * decltype(w)::value), 0, st, a,
                         __builtin_ctz(p.page_size), most);
    };
    if (p.page_size <= 32) go(std::integral_constant<int, 1>{});
    else if (p.page_size <= 128) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 16>{});
  });
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

size_t paged_select_workspace(const kvx_paged_select_args& a) { return (size_t)4 * a.B * a.Hkv * a.max_pages; }

int launch_paged_select(const kvx_paged_select_args& a, hipStream_t st) {
  const SelectParams p = {a, (uint32_t*)a.workspace, (a.max_pages + SCORED - 1) / SCORED};
  const int64_t blocks = (int64_t)a.B * a.Hkv * p.parts;
  KVX_REQUIRE(blocks < (1 << 23) && (int64_t)a.B * a.Hkv < (1 << 21), KVX_ERR_UNSUPPORTED, "kvx_paged_select: %d sequences of up to %d pages, %d KV heads in one call", a.B,
              a.max_pages, a.Hkv);
  const dim3 grid((unsigned)blocks);
  auto go = [&](auto d) {
    if (a.elem_dtype == KVX_KV_F16) hipLaunchKernelGGL((select_score_kernel<decltype(d)::value, true>), grid, dim3(NTHREADS), 0, st, p);
    else hipLaunchKernelGGL((select_score_kernel<decltype(d)::value, false>), grid, dim3(NTHREADS), 0, st, p);
  };
  if (a.D == 256) go(std::integral_constant<int, 256>{});
  else if (a.D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  hipLaunchKernelGGL(select_choose_kernel, dim3((unsigned)(a.B * a.Hkv)), dim3(CHOOSERS), 0, st, p);
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
