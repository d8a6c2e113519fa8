// What a layer writes for new tokens, in one launch, for gfx950 (HBM-bound): queries normalised and rotated in place, keys normalised, rotated, rounded to the
// model's type and written to their slots, values written to theirs; quantised on the way where pages hold codes. The arithmetic is that of rotary_kernel
// (rotary_heads.h) and of paged_write_kernel (page_rows.h), to the bit.
#include "page_rows.h"
#include "rotary_heads.h"

namespace kvx {
namespace {

// D / 8 lanes a row: a query head, or the key head and the value head of a KV head. The first `q_blocks` workgroups take query heads, the others KV heads: heads
// first on plain pages, tokens first on pages of codes (as paged_write_kernel, whose comment has the reasons).
template <int D, int KV, bool INTERLEAVED>
__global__ __launch_bounds__(NTHREADS) void paged_append_kernel(const kvx_paged_append_args a, const int shift, const float factor, const int64_t q_blocks, const int64_t groups) {
  constexpr bool PLAIN = kv_is_plain(KV), U4 = kv_is_u4(KV), F16 = kv_elem_f16(KV);
  constexpr int LPR = D / 8, ROWS = NTHREADS / LPR, ES = PLAIN ? 2 : 1;
  const kvx_rotary_args& r = a.rotary;
  const kvx_pages& p = a.pages;
  const int col = threadIdx.x % LPR, row = threadIdx.x / LPR, half = r.rotary_dim / 2;
  const bool turns = 8 * col < r.rotary_dim, split = !INTERLEAVED && turns, queries = blockIdx.x < q_blocks;
  const int lo = split ? 4 * col : 8 * col, hi = split ? half + 4 * col : lo + 4;
  int64_t t;
  int h;
  if (queries || PLAIN) {
    const int heads = queries ? r.Hq : r.Hkv;
    const int64_t i = ((int64_t)blockIdx.x - (queries ? 0 : q_blocks)) * ROWS + row;
    t = i / heads;
    h = (int)(i - t * heads);
  } else {
    const int64_t block = (int64_t)blockIdx.x - q_blocks;
    h = (int)(block / groups);
    t = (block - h * groups) * ROWS + row;
  }
  const bool mine = t < r.tokens;
  t = min(t, r.tokens - 1);  // all lanes stay: rows are reduced across them
  uint16_t* token = (uint16_t*)r.qkv + t * r.stride_t;
  uint16_t* head = token + (int64_t)(queries ? h : r.Hq + h) * D;
  const u32x2_t x0 = *(const u32x2_t*)(head + lo), x1 = *(const u32x2_t*)(head + hi);
  const int pos = r.positions[t];
  const bool there = mine && pos >= 0 && pos < r.table_rows;
  f32x4_t cv = {1.0f, 1.0f, 1.0f, 1.0f}, sv = {0.0f, 0.0f, 0.0f, 0.0f};
  if (turns && there) {
    cv = *(const f32x4_t*)(r.cos + (int64_t)pos * half + 4 * col);
    sv = *(const f32x4_t*)(r.sin + (int64_t)pos * half + 4 * col);
  }
  u32x2_t z0, z1;
  turn<D, F16, INTERLEAVED>(x0, x1, r.q_weight != nullptr, queries ? r.q_weight : r.k_weight, lo, hi, turns, cv, sv, factor, r.eps, z0, z1);
  if (queries) {
    if (there) {
      *(u32x2_t*)(head + lo) = z0;
      *(u32x2_t*)(head + hi) = z1;
    }
    return;
  }
  const u32x4_t vrow = *(const u32x4_t*)(token + (int64_t)(r.Hq + r.Hkv + h) * D + col * 8);
  const int64_t slot = a.slots[t], page = slot >> shift;
  const bool ok = there && slot >= 0 && page < p.num_pages;  // any other is no slot: never written out of bounds
  const int place = (int)(slot & (p.page_size - 1));
  uint8_t* kp = (uint8_t*)p.k + (page * p.k_stride_page + h * p.k_stride_h + (int64_t)place * p.k_stride_t) * ES;
  uint8_t* vp = (uint8_t*)p.v + (page * p.v_stride_page + h * p.v_stride_h + (int64_t)place * p.v_stride_t) * ES;
  if constexpr (PLAIN) {
    if (ok) {
      __builtin_nontemporal_store(z0, (u32x2_t*)(kp + 2 * lo));
      __builtin_nontemporal_store(z1, (u32x2_t*)(kp + 2 * hi));
      __builtin_nontemporal_store(vrow, (u32x4_t*)(vp + 16 * col));
    }
  } else {
    // the lanes of a row, which is one wavefront's, hand each other their pieces: a lane gets 8 values side by side
    __shared__ __align__(16) uint16_t rows[ROWS][D];
    *(u32x2_t*)&rows[row][lo] = z0;
    *(u32x2_t*)&rows[row][hi] = z1;
    __builtin_amdgcn_wave_barrier();
    const u32x4_t krow = *(const u32x4_t*)&rows[row][8 * col];
    u32x2_t kc, vc;
    float scale;
    int32_t zp;
    quantize_kv<LPR, U4 ? 4 : 8, F16>(krow, vrow, kc, vc, scale, zp);
    if constexpr (U4) {  // byte j = code[j] << 4 | code[j + D/2]: the partner lane holds the low nibbles
      kc = u32x2_t{(kc[0] << 4) | (uint32_t)__shfl_xor(kc[0], LPR / 2, 64), (kc[1] << 4) | (uint32_t)__shfl_xor(kc[1], LPR / 2, 64)};
      vc = u32x2_t{(vc[0] << 4) | (uint32_t)__shfl_xor(vc[0], LPR / 2, 64), (vc[1] << 4) | (uint32_t)__shfl_xor(vc[1], LPR / 2, 64)};
    }
    if (ok) {
      if (!U4 || col < LPR / 2) {
        __builtin_nontemporal_store(kc, (u32x2_t*)(kp + 8 * col));
        __builtin_nontemporal_store(vc, (u32x2_t*)(vp + 8 * col));
      }
      const int64_t q = page * p.qs_stride_page + h * p.qs_stride_h + place;
      if (col < 2) {
        (col ? p.v_scale : p.k_scale)[q] = scale;
        (col ? p.v_zp : p.k_zp)[q] = zp;
      }
    }
  }
}

}  // namespace

int launch_paged_append(const kvx_paged_append_args& a, hipStream_t st) {
  const kvx_rotary_args& r = a.rotary;
  const int64_t each = NTHREADS / (r.D / 8), groups = (r.tokens + each - 1) / each, q_blocks = (r.tokens * r.Hq + each - 1) / each;
  const int64_t blocks = q_blocks + (kv_is_plain(a.pages.kv_dtype) ? (r.tokens * r.Hkv + each - 1) / each : groups * r.Hkv);
  KVX_REQUIRE(blocks < (1 << 23), KVX_ERR_UNSUPPORTED, "kvx_paged_append: %lld tokens of %d + 2 * %d heads in one call", (long long)r.tokens, r.Hq, r.Hkv);
  by_store(a.pages, [&](auto d, auto kv) {
    auto go = [&](auto interleaved) {
      hipLaunchKernelGGL((paged_append_kernel<decltype(d)::value, decltype(kv)::value, decltype(interleaved)::value>), dim3((unsigned)blocks), dim3(NTHREADS), 0, st, a,
                         __builtin_ctz(a.pages.page_size), 1.0f / sqrtf((float)decltype(d)::value), q_blocks, groups);
    };
    if (r.interleaved) go(std::true_type{});
    else go(std::false_type{});
  });
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
