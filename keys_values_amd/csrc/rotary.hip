// Rotary position encoding of a ragged batch for gfx950 (HBM-bound, one pass, in place): every token has a position of its own, the pairs of a head are
// its halves' or interleaved, and may cover its first part alone; the head is normalised first where weights are given.
//   y = x / (|x|_2 / sqrt(D) + eps) * w;   (a, b) -> (a cos - b sin, b cos + a sin),   in fp32, rounded once.
#include "rotary_heads.h"

namespace kvx {
namespace {

constexpr int NT = 256;

// A workgroup a token, or several (grid y); LPR = D / 8 lanes a head, which hold 8 values each: pairs never leave a lane. Interleaved pairs lie side by side, and a lane
// holds a stretch of 8; pairs of halves: four values of either half of the rotated part. Lanes behind that part hold stretches. `rows` heads of a workgroup at a
// time, U of them a lane, every `stride` heads; a lane's angles and weights are the same for all of them.
template <int D, bool F16, bool INTERLEAVED, int U, bool PAST>  // PAST: loads and stores past the caches
__global__ __launch_bounds__(512) void rotary_kernel(const kvx_rotary_args a, const float factor, const int rows, const int stride) {
  constexpr int LPR = D / 8;
  const int t = blockIdx.x, pos = a.positions[t];
  const int col = threadIdx.x % LPR, mine = threadIdx.x / LPR, heads = a.Hq + a.Hkv, half = a.rotary_dim / 2;
  const bool turns = 8 * col < a.rotary_dim, split = !INTERLEAVED && turns;
  const int lo = split ? 4 * col : 8 * col, hi = split ? half + 4 * col : lo + 4;
  uint16_t* token = (uint16_t*)a.qkv + t * a.stride_t;
  auto get = [](const u32x2_t* p) {
    if constexpr (PAST) return __builtin_nontemporal_load(p);
    else return *p;
  };
  auto put = [](u32x2_t v, u32x2_t* p) {
    if constexpr (PAST) __builtin_nontemporal_store(v, p);
    else *p = v;
  };
  u32x2_t x0[U], x1[U];
  auto load = [&](int begin) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint16_t* p = token + min(begin + i * rows + mine, heads - 1) * D;
      x0[i] = get((const u32x2_t*)(p + lo));
      x1[i] = get((const u32x2_t*)(p + hi));
    }
  };
  int begin = blockIdx.y * U * rows;
  load(begin);  // does not wait for the position
  if (pos < 0 || pos >= a.table_rows) return;
  f32x4_t cv = {1.0f, 1.0f, 1.0f, 1.0f}, sv = {0.0f, 0.0f, 0.0f, 0.0f};
  if (turns) {
    cv = *(const f32x4_t*)(a.cos + (int64_t)pos * half + 4 * col);
    sv = *(const f32x4_t*)(a.sin + (int64_t)pos * half + 4 * col);
  }
  for (;;) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int head = begin + i * rows + mine;
      u32x2_t z0, z1;
      turn<D, F16, INTERLEAVED>(x0[i], x1[i], a.q_weight != nullptr, head < a.Hq ? a.q_weight : a.k_weight, lo, hi, turns, cv, sv, factor, a.eps, z0, z1);
      if (head < heads) {
        uint16_t* p = token + head * D;
        put(z0, (u32x2_t*)(p + lo));
        put(z1, (u32x2_t*)(p + hi));
      }
    }
    begin += stride;
    if (begin >= heads) break;
    load(begin);
  }
}

template <int D>
void launch_head(const kvx_rotary_args& a, hipStream_t st) {
  const float factor = 1.0f / sqrtf((float)D);
  constexpr int LPR = D / 8;
  const int64_t lanes = (int64_t)(a.Hq + a.Hkv) * LPR;
  // A token's heads over several workgroups where few tokens leave units idle or its heads are many; over one, two heads a lane, where up to 640 lanes of many
  // tokens would read the angles again.
  const int parts = lanes > 2 * NT + 128 || a.tokens <= 2 * num_cus() ? (int)min((lanes + NT - 1) / NT, (int64_t)65535) : 1;
  const int each = parts > 1 || lanes <= NT ? 1 : 2;
  const int threads = parts > 1 ? NT : (int)(lanes / each + 63) / 64 * 64, rows = threads / LPR;
  // More than 64 MB goes past the caches; less was just written and may be found in the one that the dies share. us, through / past them: 16384 tokens of 40 heads of 128
  // 69.0 / 63.4 (5.4 TB/s), of 32 heads of 128, half of each, 51.8 / 44.8; 4096 of 40, read from memory, 22.2 / 19.0, but 5001 of 32 in turn with two other batches
  // 13.7 / 15.4, 16384 of 10 heads of 64, 21 MB, 10.0 / 11.0.
  const bool past = a.tokens * (a.Hq + a.Hkv) * D * 2 > (64ll << 20);
  const int64_t at_once = (1ll << 32) / threads / parts - 1;  // tokens whose threads a grid can count
  for (int64_t done = 0; done < a.tokens; done += at_once) {
    kvx_rotary_args part = a;
    part.qkv = (uint16_t*)a.qkv + done * a.stride_t;
    part.positions = a.positions + done;
    const dim3 grid((unsigned)min(at_once, a.tokens - done), (unsigned)parts);
    auto go = [&](auto f16, auto interleaved, auto u) {
      constexpr bool F16 = decltype(f16)::value, IL = decltype(interleaved)::value;
      constexpr int U = decltype(u)::value;
      if (past) hipLaunchKernelGGL((rotary_kernel<D, F16, IL, U, true>), grid, dim3(threads), 0, st, part, factor, rows, parts * each * rows);
      else hipLaunchKernelGGL((rotary_kernel<D, F16, IL, U, false>), grid, dim3(threads), 0, st, part, factor, rows, parts * each * rows);
    };
    auto go_u = [&](auto f16, auto interleaved) {
      if (each == 1) go(f16, interleaved, std::integral_constant<int, 1>{});
      else go(f16, interleaved, std::integral_constant<int, 2>{});
    };
    auto go_layout = [&](auto f16) {
      if (a.interleaved) go_u(f16, std::true_type{});
      else go_u(f16, std::false_type{});
    };
    if (a.elem_dtype == KVX_KV_F16) go_layout(std::true_type{});
    else go_layout(std::false_type{});
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
