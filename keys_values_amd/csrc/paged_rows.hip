// Rows into the pages of a pool and back (HBM-bound): the write of new tokens, quantised on the way where pages hold codes, and whole sequences to dense rows.
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

// D / 8 lanes hold the K and V row of a (token, KV head). HBM-bound. Measured with rows of 128 in 8 heads:
// - Plain rows go heads first, which reads a token's rows as they lie. Codes go tokens first (the head is blockIdx.y): a workgroup's stores, 4 bytes a row of scales
//   and zero points among them, then fill lines of one page instead of leaving parts of them to workgroups on other dies. 37 K tokens: 8-bit 49.3 -> 47.4 us, 4-bit
//   48.9 -> 42.5; plain rows that way 29.2 -> 31.9 for 18 K tokens.
// - Rows are stored past the caches, which they would leave before anybody reads them: plain 29.2 -> 23.3 us (6.6 TB/s), 8-bit 47.4 -> 42.5, 4-bit 42.5 -> 41.4.
// - Two and four rows a lane took as long or longer.
template <int D, int KV>
__global__ __launch_bounds__(NTHREADS) void paged_write_kernel(const kvx_paged_write_args a, const int shift) {
  constexpr bool PLAIN = kv_is_plain(KV), U4 = kv_is_u4(KV);
  constexpr int LPR = D / 8, ROWS = NTHREADS / LPR, ES = PLAIN ? 2 : 1;
  const kvx_pages& p = a.pages;
  const int col = threadIdx.x % LPR, ccol = U4 ? col % (LPR / 2) : col;
  int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  int h = blockIdx.y;
  if constexpr (PLAIN) {
    h = (int)(t % p.Hkv);
    t /= p.Hkv;
  }
  const bool mine = t < a.tokens;
  t = min(t, a.tokens - 1);  // all lanes stay: rows are reduced across them
  const u32x4_t krow = *(const u32x4_t*)((const uint16_t*)a.key + t * a.key_stride_t + h * a.key_stride_h + col * 8);
  const u32x4_t vrow = *(const u32x4_t*)((const uint16_t*)a.value + t * a.value_stride_t + h * a.value_stride_h + col * 8);
  const int64_t slot = a.slots[t], page = slot >> shift;
  const bool ok = mine && slot >= 0 && page < p.num_pages;  // any other is no slot: never written out of bounds
  const int place = (int)(slot & (p.page_size - 1));
  uint8_t* kp = (uint8_t*)p.k + (page * p.k_stride_page + h * p.k_stride_h + (int64_t)place * p.k_stride_t) * ES + ccol * 8 * ES;
  uint8_t* vp = (uint8_t*)p.v + (page * p.v_stride_page + h * p.v_stride_h + (int64_t)place * p.v_stride_t) * ES + ccol * 8 * ES;
  if constexpr (PLAIN) {
    if (ok) {
      __builtin_nontemporal_store(krow, (u32x4_t*)kp);
      __builtin_nontemporal_store(vrow, (u32x4_t*)vp);
    }
  } else {
    u32x2_t kc, vc;
    float scale;
    int32_t zp;
    quantize_kv<LPR, U4 ? 4 : 8, kv_elem_f16(KV)>(krow, vrow, kc, vc, scale, zp);
    if constexpr (U4) {  // byte j = code[j] << 4 | code[j + D/2]: the partner lane holds the low nibbles
      kc = u32x2_t{(kc[0] << 4) | (uint32_t)__shfl_xor(kc[0], LPR / 2, 64), (kc[1] << 4) | (uint32_t)__shfl_xor(kc[1], LPR / 2, 64)};
      vc = u32x2_t{(vc[0] << 4) | (uint32_t)__shfl_xor(vc[0], LPR / 2, 64), (vc[1] << 4) | (uint32_t)__shfl_xor(vc[1], LPR / 2, 64)};
    }
    if (ok) {
      if (!U4 || col < LPR / 2) {
        __builtin_nontemporal_store(kc, (u32x2_t*)kp);
        __builtin_nontemporal_store(vc, (u32x2_t*)vp);
      }
      const int64_t q = page * p.qs_stride_page + h * p.qs_stride_h + place;
      if (col < 2) {
        (col ? p.v_scale : p.k_scale)[q] = scale;
        (col ? p.v_zp : p.k_zp)[q] = zp;
      }
    }
  }
}

// 8 values of a row a lane; grid: blocks of rows, (sequence, KV head) pairs. The rows are stored past the caches: 4 sequences of 4096 to 16384 tokens, 8 heads of 128,
// 8-bit 67.5 -> 49.1 us (7.1 TB/s on what is read and written), 4-bit 63.6 -> 44.2; plain 36.2 -> 34.3 for 18 K tokens padded to 41 K. Two rows a lane took as long,
// eight longer.
template <int D, int KV>
__global__ __launch_bounds__(NTHREADS) void paged_read_kernel(const kvx_paged_read_args a, const int shift) {
  constexpr bool PLAIN = kv_is_plain(KV), U4 = kv_is_u4(KV), F16 = kv_elem_f16(KV);
  constexpr int LPR = D / 8, ES = PLAIN ? 2 : 1;
  const kvx_pages& p = a.pages;
  const int t = blockIdx.x * (NTHREADS / LPR) + threadIdx.x / LPR, col = threadIdx.x % LPR;
  const int b = blockIdx.y / p.Hkv, h = blockIdx.y - b * p.Hkv;
  if (t >= a.length) return;
  u32x4_t k = {0u, 0u, 0u, 0u}, v = k;
  if (t < a.lens[b] && (t >> shift) < a.max_pages) {
    const int page = a.block_table[b * a.bt_stride_b + (t >> shift)];
    if (page >= 0 && page < p.num_pages) {
      const int place = t & (p.page_size - 1);
      const uint8_t* kp = (const uint8_t*)p.k + ((int64_t)page * p.k_stride_page + h * p.k_stride_h + (int64_t)place * p.k_stride_t) * ES;
      const uint8_t* vp = (const uint8_t*)p.v + ((int64_t)page * p.v_stride_page + h * p.v_stride_h + (int64_t)place * p.v_stride_t) * ES;
      if constexpr (PLAIN) {
        k = *(const u32x4_t*)(kp + col * 16);
        v = *(const u32x4_t*)(vp + col * 16);
      } else {
        const int64_t q = (int64_t)page * p.qs_stride_page + h * p.qs_stride_h + place;
        const int off = U4 ? (int)u4_byte_off<D>(col) : col * 8;
        u32x2_t kc = *(const u32x2_t*)(kp + off), vc = *(const u32x2_t*)(vp + off);
        if constexpr (U4) {
          kc = u4_codes(kc, u4_shift<D>(col));
          vc = u4_codes(vc, u4_shift<D>(col));
        }
        k = dequant_words<F16>(kc[0], kc[1], p.k_zp[q], p.k_scale[q]);
        v = dequant_words<F16>(vc[0], vc[1], p.v_zp[q], p.v_scale[q]);
      }
    }
  }
  __builtin_nontemporal_store(k, (u32x4_t*)((uint16_t*)a.key + b * a.key_stride_b + h * a.key_stride_h + t * a.key_stride_t + col * 8));
  __builtin_nontemporal_store(v, (u32x4_t*)((uint16_t*)a.value + b * a.value_stride_b + h * a.value_stride_h + t * a.value_stride_t + col * 8));
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

int launch_paged_write(const kvx_paged_write_args& a, hipStream_t st) {
  const bool plain = kv_is_plain(a.pages.kv_dtype);
  const int64_t each = NTHREADS / (a.pages.D / 8), grid = ((plain ? a.tokens * a.pages.Hkv : a.tokens) + each - 1) / each;
  const dim3 blocks((unsigned)grid, plain ? 1 : a.pages.Hkv);
  KVX_REQUIRE(grid * blocks.y < (1 << 23), KVX_ERR_UNSUPPORTED, "kvx_paged_write: %lld tokens of %d heads in one call", (long long)a.tokens, a.pages.Hkv);
  by_store(a.pages, [&](auto d, auto kv) {
    hipLaunchKernelGGL((paged_write_kernel<decltype(d)::value, decltype(kv)::value>), blocks, dim3(NTHREADS), 0, st, a, __builtin_ctz(a.pages.page_size));
  });
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

int launch_paged_read(const kvx_paged_read_args& a, hipStream_t st) {
  const int64_t each = NTHREADS / (a.pages.D / 8), grid = (a.length + each - 1) / each, pairs = (int64_t)a.B * a.pages.Hkv;
  KVX_REQUIRE(grid * pairs < (1 << 23), KVX_ERR_UNSUPPORTED, "kvx_paged_read: %lld (sequence, head) pairs of %d tokens in one call", (long long)pairs, a.length);
  const int most = 65535 / a.pages.Hkv;  // sequences of a launch: a grid's y counts to 65535
  for (int done = 0; done < a.B; done += most) {
    kvx_paged_read_args part = a;
    part.B = min(most, a.B - done);
    part.block_table += done * a.bt_stride_b;
    part.lens += done;
    part.key = (uint16_t*)a.key + done * a.key_stride_b;
    part.value = (uint16_t*)a.value + done * a.value_stride_b;
    by_store(a.pages, [&](auto d, auto kv) {
      hipLaunchKernelGGL((paged_read_kernel<decltype(d)::value, decltype(kv)::value>), dim3((unsigned)grid, (unsigned)(part.B * a.pages.Hkv)), dim3(NTHREADS), 0, st, part,
                         __builtin_ctz(a.pages.page_size));
    });
  }
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
