// What a layer writes for new tokens, in one launch, for gfx950: queries normalised and rotated in place, keys normalised, rotated, rounded to the
// model's type and written to their slots, values written to theirs; quantised on the way where pages hold codes. The arithmetic is that of rotary_kernel
// (rotary_heads.h) and of paged_write_kernel (page_rows.h), to the bit.
//   y = x / (|x|_2 / sqrt(D) + eps) * w;   (a, b) -> (a cos - b sin, b cos + a sin);   of codes: scale and zero point of a row from its extremes
// HBM-bound: every row is read once and written once. 18705 tokens of 32 + 16 heads of 128 into plain pages (469 MB): 82 us, 5.7 TB/s, which is more than a large copy reaches
// (5.4); 5036 tokens of 28 + 8 heads of 128 into 4-bit pages: 18 us. 32 tokens, 3.5 us, are latency: rows, angles, stores.
#include "page_rows.h"
#include "rotary_heads.h"

namespace kvx {
namespace {

// D / 8 lanes a row. Plain pages: a workgroup a token, or several a token where tokens are few; U rows a lane (query, key and value heads), every `stride` rows, so that a token's
// angles are read once: the 18705 tokens with two rows a lane 92 us, three 82, four or six 84; loads through the caches 86, stores to pages through them 90, of queries 89. Pages of codes: the first token_blocks workgroups take a token's query heads so, the others ROWS tokens of a KV head, a lane its share of the
// key's and of the value's row (tokens first, as paged_write_kernel, whose comment has the reasons).
template <int D, int KV, bool INTERLEAVED, int U, bool PAST>  // PAST: queries past the caches; rows of pages always go past them
__global__ __launch_bounds__(512) void paged_append_kernel(const kvx_paged_append_args a, const int shift, const float factor, const int parts, const int stride,
                                                           const int64_t token_blocks, const int groups) {
  constexpr bool PLAIN = kv_is_plain(KV), U4 = kv_is_u4(KV), F16 = kv_elem_f16(KV);
  constexpr int LPR = D / 8, ROWS = NTHREADS / LPR;
  const kvx_rotary_args& r = a.rotary;
  const kvx_pages& p = a.pages;
  const int col = threadIdx.x % LPR, mine = threadIdx.x / LPR, half = r.rotary_dim / 2, Hq = r.Hq, Hkv = r.Hkv;
  const bool turns = 8 * col < r.rotary_dim, split = !INTERLEAVED && turns;
  const int lo = split ? 4 * col : 8 * col, hi = split ? half + 4 * col : lo + 4;
  f32x4_t cv = {1.0f, 1.0f, 1.0f, 1.0f}, sv = {0.0f, 0.0f, 0.0f, 0.0f};
  auto angles = [&](int pos) {
    if (turns) {
      cv = *(const f32x4_t*)(r.cos + (int64_t)pos * half + 4 * col);
      sv = *(const f32x4_t*)(r.sin + (int64_t)pos * half + 4 * col);
    }
  };
  auto place_of = [&](int64_t slot, int64_t& page, int& place) {  // whether it is one of the pool's: any other is no slot, never written out of bounds
    page = slot >> shift;
    place = (int)(slot & (p.page_size - 1));
    return slot >= 0 && page < p.num_pages;
  };

  if (PLAIN || blockIdx.x < token_blocks) {
    const int t = blockIdx.x / parts, part = blockIdx.x - t * parts, heads = PLAIN ? Hq + 2 * Hkv : Hq, rows = blockDim.x / LPR;
    uint16_t* token = (uint16_t*)r.qkv + t * r.stride_t;
    u32x2_t x0[U], x1[U];
    auto get = [](const uint16_t* p) {
      if constexpr (PAST) return __builtin_nontemporal_load((const u32x2_t*)p);
      else return *(const u32x2_t*)p;
    };
    auto load = [&](int begin) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const uint16_t* at = token + min(begin + i * rows + mine, heads - 1) * D;
        x0[i] = get(at + lo);
        x1[i] = get(at + hi);
      }
    };
    int begin = part * U * rows;
    load(begin);  // waits for nothing
    const int pos = r.positions[t];
    int64_t page = 0;
    int place = 0;
    const bool ok = PLAIN && place_of(a.slots[t], page, place);
    if (pos < 0 || pos >= r.table_rows) return;
    angles(pos);
    for (;;) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int head = begin + i * rows + mine;
        u32x2_t z0 = x0[i], z1 = x1[i];
        if (head < Hq + Hkv) turn<D, F16, INTERLEAVED>(x0[i], x1[i], r.q_weight != nullptr, head < Hq ? r.q_weight : r.k_weight, lo, hi, turns, cv, sv, factor, r.eps, z0, z1);
        if (head < Hq) {
          uint16_t* to = token + head * D;
          if constexpr (PAST) {
            __builtin_nontemporal_store(z0, (u32x2_t*)(to + lo));
            __builtin_nontemporal_store(z1, (u32x2_t*)(to + hi));
          } else {
            *(u32x2_t*)(to + lo) = z0;
            *(u32x2_t*)(to + hi) = z1;
          }
        } else if (ok && head < heads) {
          const bool value = head >= Hq + Hkv;
          const int h = head - Hq - (value ? Hkv : 0);
          uint16_t* to = value ? (uint16_t*)p.v + page * p.v_stride_page + h * p.v_stride_h + (int64_t)place * p.v_stride_t
                               : (uint16_t*)p.k + page * p.k_stride_page + h * p.k_stride_h + (int64_t)place * p.k_stride_t;
          __builtin_nontemporal_store(z0, (u32x2_t*)(to + lo));
          __builtin_nontemporal_store(z1, (u32x2_t*)(to + hi));
        }
      }
      begin += stride;
      if (begin >= heads) break;
      load(begin);
    }
  } else if constexpr (!PLAIN) {
    const int64_t block = (int64_t)blockIdx.x - token_blocks;
    const int h = (int)(block / groups);
    int64_t t = (block - (int64_t)h * groups) * ROWS + mine;
    const bool is = t < r.tokens;
    t = min(t, r.tokens - 1);  // all lanes stay: rows are reduced across them
    const uint16_t* token = (const uint16_t*)r.qkv + t * r.stride_t;
    const uint16_t* head = token + (int64_t)(Hq + h) * D;
    const u32x2_t x0 = *(const u32x2_t*)(head + lo), x1 = *(const u32x2_t*)(head + hi);
    const u32x4_t vrow = *(const u32x4_t*)(token + (int64_t)(Hq + Hkv + h) * D + col * 8);
    const int pos = r.positions[t];
    int64_t page;
    int place;
    const bool there = is && pos >= 0 && pos < r.table_rows, ok = place_of(a.slots[t], page, place) && there;
    if (there) angles(pos);
    u32x2_t z0, z1;
    turn<D, F16, INTERLEAVED>(x0, x1, r.q_weight != nullptr, r.k_weight, lo, hi, turns, cv, sv, factor, r.eps, z0, z1);
    // the lanes of a row, which is one wavefront's, hand each other their pieces: a lane gets 8 values side by side
    __shared__ __align__(16) uint16_t rows[ROWS][D];
    *(u32x2_t*)&rows[mine][lo] = z0;
    *(u32x2_t*)&rows[mine][hi] = z1;
    __builtin_amdgcn_wave_barrier();
    const u32x4_t krow = *(const u32x4_t*)&rows[mine][8 * col];
    u32x2_t kc, vc;
    float scale;
    int32_t zp;
    quantize_kv<LPR, U4 ? 4 : 8, F16>(krow, vrow, kc, vc, scale, zp);
    if constexpr (U4) {  // byte j = code[j] << 4 | code[j + D/2]: the partner lane holds the low nibbles
      kc = u32x2_t{(kc[0] << 4) | (uint32_t)__shfl_xor(kc[0], LPR / 2, 64), (kc[1] << 4) | (uint32_t)__shfl_xor(kc[1], LPR / 2, 64)};
      vc = u32x2_t{(vc[0] << 4) | (uint32_t)__shfl_xor(vc[0], LPR / 2, 64), (vc[1] << 4) | (uint32_t)__shfl_xor(vc[1], LPR / 2, 64)};
    }
    if (ok) {
      uint8_t* kp = (uint8_t*)p.k + page * p.k_stride_page + h * p.k_stride_h + (int64_t)place * p.k_stride_t;
      uint8_t* vp = (uint8_t*)p.v + page * p.v_stride_page + h * p.v_stride_h + (int64_t)place * p.v_stride_t;
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
  const bool plain = kv_is_plain(a.pages.kv_dtype);
  const int lpr = r.D / 8, heads = plain ? r.Hq + 2 * r.Hkv : r.Hq;
  const int64_t each = NTHREADS / lpr, groups = (r.tokens + each - 1) / each, lanes = (int64_t)heads * lpr;
  // A token's rows over several workgroups where few tokens leave units idle; over one, up to three a lane, where more tokens would read the angles again.
  const int parts = r.tokens <= 2 * num_cus() ? (int)((lanes + NTHREADS - 1) / NTHREADS) : 1;
  // Lanes of a token are few hundreds; 18705 tokens of plain rows of 128, us with one, two and three rows a lane: 8 / 2 heads (192 lanes) 21.8, 26.3, 25.3; 16 / 4 (384) 52.4, 43.9, 44.1; 32 / 8
  // (768) 98, 88, 81. In between, 28 / 4 (576) 83, 69, 62 and 24 / 8 (640) 86, 73, 68, three would do better than the two that they take; queries of pages of codes (32 / 8, 512) 89, 87, 93.
  const int u = parts > 1 || lanes <= NTHREADS ? 1 : lanes <= 640 ? 2 : 3;
  const int threads = parts > 1 || !plain ? NTHREADS : (int)min((lanes + 64 * u - 1) / (64 * u) * 64, (int64_t)512), stride = parts * u * (threads / lpr);
  const bool past = r.tokens * lanes * 16 > (64ll << 20);
  const int64_t token_blocks = r.tokens * parts, blocks = token_blocks + (plain ? 0 : groups * r.Hkv);
  KVX_REQUIRE(blocks < (1 << 23), KVX_ERR_UNSUPPORTED, "kvx_paged_append: %lld tokens of %d + 2 * %d heads in one call", (long long)r.tokens, r.Hq, r.Hkv);
  by_store(a.pages, [&](auto d, auto kv) {
    auto go = [&](auto interleaved, auto rows, auto past) {
      hipLaunchKernelGGL((paged_append_kernel<decltype(d)::value, decltype(kv)::value, decltype(interleaved)::value, decltype(rows)::value, decltype(past)::value>),
                         dim3((unsigned)blocks), dim3(threads), 0, st, a, __builtin_ctz(a.pages.page_size), 1.0f / sqrtf((float)decltype(d)::value), parts, stride, token_blocks,
                         (int)groups);
    };
    auto go_past = [&](auto interleaved, auto rows) {
      if (past) go(interleaved, rows, std::true_type{});
      else go(interleaved, rows, std::false_type{});
    };
    auto go_rows = [&](auto interleaved) {
      if (u == 1) go_past(interleaved, std::integral_constant<int, 1>{});
      else if (u == 2) go_past(interleaved, std::integral_constant<int, 2>{});
      else go_past(interleaved, std::integral_constant<int, 3>{});
    };
    if (r.interleaved) go_rows(std::true_type{});
    else go_rows(std::false_type{});
  });
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
