// Attention of one new token a sequence over the pages of a pool, for gfx950 (HBM-bound).
//   o = softmax(sm_scale q K^T) V over the sequence's first lens[b] rows, in one pass with a running maximum and sum.
//
// Work. Sequences of one batch may have one token or hundreds of thousands, and only the device knows. The rows of all (sequence, KV head) pairs are cut into
// units of 128 keys and dealt out to a fixed number of workgroups, each a stretch of neighbouring units that may end and begin within a pair's rows:
// every workgroup has the same number of units, or one more, whatever the lengths. What a workgroup does of a pair that it does not have to itself it leaves as a
// partial (maximum, sum, outputs); a second launch joins the partials of a pair. A workgroup has at most two: that of the pair it begins in the middle of, and
// that of the pair it leaves off in.
//
// Arithmetic. All query heads of a KV head share its rows: up to 16 of them are the columns of v_mfma_f32_16x16x32, S^T = K Q^T for 16 keys and O^T += V^T P^T
// for 32. The operands are rows as they come from memory (key_blocks.h describes the layouts): the accumulator of S^T becomes the second product's B operand
// without an exchange. A wavefront takes 32 keys at a time; while it forms their weights the next K rows are on their way, and while it forms the next
// logits the next V rows are. No barrier until a stretch ends.
//
// Codes. (code - zp) * scale is linear in the code, so the codes themselves are the operands, and scale and zero point are applied to a key's 16 logits and weights
// instead of its 2 D values: 16-bit integers below 1024 are what fp16 calls subnormal numbers, code * 2^-24, which the matrix cores multiply exactly,
// so one byte permute makes two operand values of 8-bit codes, and one mask, for 4-bit ones, the codes of the high halves as 16 times theirs.
//   logit = scale_k (S - zp_k sum q),        S = sum code q,      q in fp16 times a power of two that brings the head's largest below 2^15 (exact)
//   o     = (sum w code - sum w zp_v) / l,   w = p scale_v,       in units of a power of two above the largest scale_v so far
// w is rounded to fp16 for the product: w'. What that costs is bounded by a row's span, if the middle code c is taken out of the zero point:
//   sum w code - sum w zp = sum w' code - c sum w' - sum w (zp - c) + sum (w - w') (code - c).
#include <type_traits>

#include "key_blocks.h"

namespace kvx {
namespace {

constexpr int NT = 256, WAVES = 4, UNIT = 128;  // keys of a unit: a block of 32 a wavefront
constexpr float kLowest = -3.4028235e38f;       // running maximum before the first key
typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

struct PagedParams {
  kvx_paged_decode_args a;
  float c;          // sm_scale * log2(e)
  int shift;        // log2 of the page size
  int cap;          // tokens of a table's pages
  int Gr;           // query heads per KV head
  int workgroups;
  float* part_o;    // (2 workgroups, Gr, D)
  float* part_ml;   // (2 workgroups, Gr, 2): maximum and sum
  int* part_of;     // (workgroups, 2): the pair whose first partial the workgroup left, and how many the pair has
};

__device__ __forceinline__ int units_of(int len, int cap) { return max(1, (min(max(len, 0), cap) + UNIT - 1) / UNIT); }

// Inclusive sum over the lanes of a wavefront.
__device__ __forceinline__ int scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

// The shares of `total` units: workgroup w begins with unit first(w).
struct Shares {
  int each, rest;
  __device__ __forceinline__ Shares(int total, int workgroups) : each(total / workgroups), rest(total - each * workgroups) {}
  __device__ __forceinline__ int first(int w) const { return w * each + min(w, rest); }
  __device__ __forceinline__ int owner(int unit) const {
    const int big = rest * (each + 1);
    return unit < big ? unit / (each + 1) : rest + (unit - big) / each;
  }
};

template <int D, int KV>
struct Rows {
  static constexpr bool F16 = kv_elem_f16(KV), CODES = !kv_is_plain(KV), U4 = kv_is_u4(KV);
  static constexpr int KJ = D / 32, DPL = D / 16, ES = CODES ? 1 : 2;
  static constexpr int NL4 = D >= 128 ? D / 128 : 1;
  static constexpr int KR = U4 ? NL4 : (CODES ? D / 64 : KJ);                         // 16-byte loads per key of K
  static constexpr int VB = U4 ? DPL / 2 : DPL * ES;                                  // bytes per key of V
  static constexpr int VW = (VB + 3) / 4;
  struct K {
    u32x4_t w[2][KR];
    f32x4_t scale[2];
    i32x4_t zp[2];
  };
  struct V {
    uint32_t w[8][VW];
    f32x4_t scale[2];
    i32x4_t zp[2];
  };
  // first d of the 8 that lane group kg supplies to matrix instruction e of the first product
  __device__ __forceinline__ static int kslice(int e, int kg) {
    if constexpr (!CODES) return 8 * (kg + 4 * e);
    else if constexpr (!U4) return 16 * kg + 8 * (e & 1) + 64 * (e >> 1);
    else if constexpr (D == 64) return 8 * kg + 32 * e;
    else return 64 * (e >> 2) + 16 * kg + 8 * ((e >> 1) & 1) + (D / 2) * (e & 1);
  }
  // 4-bit codes: instruction e takes those of the high halves of its bytes, 16 times as large
  __device__ __forceinline__ static bool high(int e) { return U4 && (e & 1) == 0; }
  // A operand e of the first product for tile gi
  __device__ __forceinline__ static u32x4_t k_operand(const K& r, int gi, int e) {
    if constexpr (!CODES) {
      return r.w[gi][e];
    } else if constexpr (!U4) {
      const u32x4_t w = r.w[gi][e >> 1];
      const uint32_t a = w[2 * (e & 1)], b = w[2 * (e & 1) + 1];
      return u32x4_t{__builtin_amdgcn_perm(0u, a, 0x0c010c00u), __builtin_amdgcn_perm(0u, a, 0x0c030c02u), __builtin_amdgcn_perm(0u, b, 0x0c010c00u),
                     __builtin_amdgcn_perm(0u, b, 0x0c030c02u)};
    } else {
      const int x = D == 64 ? 0 : e >> 2, pair = D == 64 ? 0 : (e >> 1) & 1;
      const uint32_t a = r.w[gi][x][2 * pair], b = r.w[gi][x][2 * pair + 1], mask = high(e) ? 0x00f000f0u : 0x000f000fu;
      return u32x4_t{a & mask, (a >> 8) & mask, b & mask, (b >> 8) & mask};  // values 0, 2 | 1, 3 | 4, 6 | 5, 7
    }
  }
  // A operand t of the second product: value t of each of this lane's 8 keys, in key order
  __device__ __forceinline__ static u32x4_t v_operand(const V& r, int t) {
    u32x4_t a;
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const int j0 = 2 * jj, j1 = 2 * jj + 1;
      if constexpr (!CODES) {
        a[jj] = __builtin_amdgcn_perm(r.w[j1][t >> 1], r.w[j0][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
      } else {
        const int byte = U4 && t >= DPL / 2 ? t - DPL / 2 : t;
        a[jj] = __builtin_amdgcn_perm(r.w[j1][byte >> 2], r.w[j0][byte >> 2], 0x0c040c00u + 0x00010001u * (byte & 3));
        if constexpr (U4) a[jj] &= t < DPL / 2 ? 0x00f000f0u : 0x000f000fu;
      }
    }
    return a;
  }
  // d of row `mrow` of matrix instruction t of the second product
  __device__ __forceinline__ static int dmap(int t, int mrow) {
    if constexpr (U4) return t < DPL / 2 ? (DPL / 2) * mrow + t : D / 2 + (DPL / 2) * mrow + (t - DPL / 2);
    else return DPL * mrow + t;
  }
};

template <typename T>
__device__ __forceinline__ T once(const void* p) { return __builtin_nontemporal_load((const T*)p); }

// Wavefronts a SIMD: as many as the registers of a block of keys allow.
template <int D, int KV>
constexpr int waves_per_simd() { return D == 256 && kv_is_plain(KV) ? 1 : D == 256 ? 2 : 3; }

template <int D, int KV>
__global__ __launch_bounds__(NT, (waves_per_simd<D, KV>())) void paged_decode_kernel(const PagedParams p) {
  using R = Rows<D, KV>;
  constexpr bool F16 = R::F16, CODES = R::CODES, U4 = R::U4, P16 = F16 || CODES;  // P16: weights and operands in fp16
  constexpr int KJ = R::KJ, DPL = R::DPL, ES = R::ES;
  // The running maximum moves when a logit exceeds it by kTop. Weights in fp16 are kept below 2^15, and brought to 2^7 when it moves: what is a normal number
  // there goes down to 2^-21 of the largest then, and what is not zero to 2^-32.
  constexpr float kTop = P16 ? 15.0f : 8.0f, kBias = P16 ? 7.0f : 0.0f;
  constexpr int RS = D + 4;  // floats of a head's row in LDS: heads in different banks
  __shared__ __align__(16) float red[WAVES][16][RS];
  __shared__ float red_m[WAVES][16], red_l[WAVES][16], weight[WAVES][16], fin[2][16];

  const kvx_pages& pg = p.a.pages;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, kg = lane >> 4;
  const int B = p.a.B, Hkv = pg.Hkv, w = blockIdx.x, mask = pg.page_size - 1;
  const int* const lens = p.a.lens;

  // ---- this workgroup's units: every wavefront finds them for itself
  int b, begin_b, unit, end;  // sequence, its first unit, the next unit, the end of the share
  Shares shares(0, 1);
  {
    const int per = (B + 63) / 64;
    int mine = 0;
    for (int i = 0; i < per; ++i)
      if (lane * per + i < B) mine += units_of(lens[lane * per + i], p.cap);
    const int upto = scan(mine), total = __builtin_amdgcn_readlane(upto, 63) * Hkv;
    shares = Shares(total, p.workgroups);
    unit = shares.first(w);
    end = shares.first(w + 1);
    const int at = __builtin_ctzll(__ballot(upto * Hkv > unit) | (1ull << 63));
    b = at * per;
    begin_b = __builtin_amdgcn_readlane(upto - mine, at) * Hkv;
    for (; b < B - 1; ++b) {
      const int n = units_of(lens[b], p.cap) * Hkv;
      if (begin_b + n > unit) break;
      begin_b += n;
    }
  }
  if (tid == 0) p.part_of[2 * w + 1] = 0;

  const uint32_t k_rowb = (uint32_t)pg.k_stride_t * ES, v_rowb = (uint32_t)pg.v_stride_t * ES;
  const uint32_t k_lane = (uint32_t)m * k_rowb + (U4 && D == 64 ? 8 : 16) * kg, v_lane = 4 * kg * v_rowb + (uint32_t)m * R::VB;

  while (unit < end) {
    const int len = min(max(lens[b], 0), p.cap), units = units_of(len, p.cap);
    const int h = (unit - begin_b) / units, begin = begin_b + h * units, first = unit - begin, n_units = min(units - first, end - unit);
    const int k_begin = first * UNIT, k_end = min(len, (first + n_units) * UNIT);

    // ---- queries: B operands of the first product, head m (zero beyond the group)
    u32x4_t qb[KJ];
    float qsum = 0.0f, to_logit = p.c;
#pragma unroll
    for (int e = 0; e < KJ; ++e) {
      qb[e] = u32x4_t{0u, 0u, 0u, 0u};
      if (m < p.Gr) qb[e] = *(const u32x4_t*)((const uint16_t*)p.a.q + b * p.a.q_stride_b + (int64_t)(h * p.Gr + m) * p.a.q_stride_h + R::kslice(e, kg));
    }
    if constexpr (CODES) {
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < KJ; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(elem_lo<F16>(qb[e][i])), fabsf(elem_hi<F16>(qb[e][i]))));
      top = max_halves(max_row_pairs(top));
      // 2^x that brings the largest to [2^14, 2^15); zeros, infinities and NaN stay
      const int ex = (int)(__float_as_uint(top) >> 23), up = ex == 0 || ex == 255 ? 127 : min(268 - ex, 253);
      const float by = __uint_as_float((uint32_t)up << 23);
      to_logit = __uint_as_float((uint32_t)(254 - up) << 23) * p.c;
#pragma unroll
      for (int e = 0; e < KJ; ++e) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = elem_lo<F16>(qb[e][i]) * by;
          x[2 * i + 1] = elem_hi<F16>(qb[e][i]) * by;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) qsum += x[i];
        if constexpr (U4) {
          const float f = R::high(e) ? 0.0625f : 1.0f;
          qb[e] = u32x4_t{pack_pair<true>(x[0] * f, x[2] * f), pack_pair<true>(x[1] * f, x[3] * f), pack_pair<true>(x[4] * f, x[6] * f), pack_pair<true>(x[5] * f, x[7] * f)};
        } else {
          qb[e] = u32x4_t{pack_pair<true>(x[0], x[1]), pack_pair<true>(x[2], x[3]), pack_pair<true>(x[4], x[5]), pack_pair<true>(x[6], x[7])};
        }
      }
      qsum = sum_halves([](float v) {
        const u32pair_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
      }(qsum));
    }

    f32x4_t acc[DPL];
#pragma unroll
    for (int t = 0; t < DPL; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kLowest, l_run = 0.0f;
    float corr = 0.0f, unit_v = 0x1p-126f, per_v = 0x1p126f;  // codes: sum of c w' + w (zp - c); the unit of the scales, and its inverse

    // ---- rows of a block of 32 keys. The pages of its two halves come by scalar loads; a page that the pool does not have is read as page 0, and its keys are
    // masked behind. Keys behind the end lie in the same pages, or masked ones.
    struct Tiles {
      int page[2];
    };
    const auto table = (const int __attribute__((address_space(4)))*)(uintptr_t)(p.a.block_table + b * p.a.bt_stride_b);
    auto pages = [&](int chunk) {
      Tiles t;
#pragma unroll
      for (int gi = 0; gi < 2; ++gi) t.page[gi] = table[min((chunk + 16 * gi) >> p.shift, p.a.max_pages - 1)];
      return t;
    };
    auto there = [&](int page) { return (uint32_t)page < (uint32_t)pg.num_pages; };
    auto load_k = [&](typename R::K& r, int chunk, const Tiles& t) {
#pragma unroll
      for (int gi = 0; gi < 2; ++gi) {
        const int64_t page = there(t.page[gi]) ? t.page[gi] : 0;
        const uint8_t* base = (const uint8_t*)pg.k + (page * pg.k_stride_page + h * pg.k_stride_h) * ES;
        const int place = (chunk + 16 * gi) & mask;
        const uint32_t off = (uint32_t)place * k_rowb + k_lane;
#pragma unroll
        for (int x = 0; x < R::KR; ++x) {
          if constexpr (U4 && D == 64) {
            const u32x2_t y = once<u32x2_t>(base + off);
            r.w[gi][x] = u32x4_t{y[0], y[1], 0u, 0u};
          } else {
            r.w[gi][x] = once<u32x4_t>(base + off + 64 * x);
          }
        }
        if constexpr (CODES) {
          const int64_t q = page * pg.qs_stride_page + h * pg.qs_stride_h + place;
          r.scale[gi] = once<f32x4_t>((const char*)(pg.k_scale + q) + 16 * kg);
          r.zp[gi] = once<i32x4_t>((const char*)(pg.k_zp + q) + 16 * kg);
        }
      }
    };
    auto load_v = [&](typename R::V& r, int chunk, const Tiles& t) {
#pragma unroll
      for (int gi = 0; gi < 2; ++gi) {
        const int64_t page = there(t.page[gi]) ? t.page[gi] : 0;
        const uint8_t* base = (const uint8_t*)pg.v + (page * pg.v_stride_page + h * pg.v_stride_h) * ES;
        const int place = (chunk + 16 * gi) & mask;
        const uint32_t off = (uint32_t)place * v_rowb + v_lane;
        if constexpr (CODES) {
          const int64_t q = page * pg.qs_stride_page + h * pg.qs_stride_h + place;
          r.scale[gi] = once<f32x4_t>((const char*)(pg.v_scale + q) + 16 * kg);
          r.zp[gi] = once<i32x4_t>((const char*)(pg.v_zp + q) + 16 * kg);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* row = base + (off + (uint32_t)i * v_rowb);
          uint32_t(&x)[R::VW] = r.w[4 * gi + i];
          if constexpr (R::VB >= 16) {
#pragma unroll
            for (int y = 0; y < R::VB / 16; ++y) {
              const u32x4_t z = once<u32x4_t>(row + 16 * y);
              x[4 * y] = z[0]; x[4 * y + 1] = z[1]; x[4 * y + 2] = z[2]; x[4 * y + 3] = z[3];
            }
          } else if constexpr (R::VB == 8) {
            const u32x2_t z = once<u32x2_t>(row);
            x[0] = z[0]; x[1] = z[1];
          } else if constexpr (R::VB == 4) {
            x[0] = once<uint32_t>(row);
          } else {
            x[0] = (uint32_t)once<uint16_t>(row);
          }
        }
      }
    };
    auto whole = [&](int chunk, const Tiles& t) { return chunk + 32 <= k_end && there(t.page[0]) && there(t.page[1]); };
    // key 4 kg + i of tile gi, this lane's, is one of the sequence's
    auto live = [&](int chunk, const Tiles& t, int gi, int i) { return there(t.page[gi]) && chunk + 16 * gi + 4 * kg + i < k_end; };
    // logits in log2 units: head m, keys 4 kg + i of the two tiles
    auto logits = [&](const typename R::K& r, int chunk, const Tiles& t, float (&s)[8]) {
      f32x4_t x[2];
#pragma unroll
      for (int gi = 0; gi < 2; ++gi) {
        x[gi] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < KJ; ++e) x[gi] = mfma_16x16x32<P16>(R::k_operand(r, gi, e), qb[e], x[gi]);
      }
#pragma unroll
      for (int gi = 0; gi < 2; ++gi)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (CODES) s[4 * gi + i] = fmaf(-(float)r.zp[gi][i], qsum, x[gi][i] * 0x1p24f) * (r.scale[gi][i] * to_logit);
          else s[4 * gi + i] = x[gi][i] * to_logit;
        }
      if (!whole(chunk, t)) {
#pragma unroll
        for (int gi = 0; gi < 2; ++gi)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!live(chunk, t, gi, i)) s[4 * gi + i] = -INFINITY;
      }
    };
    auto weights = [&](float (&s)[8]) {
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
      if (__any(top > m_run + kTop)) {
        top = max_halves(max_row_pairs(top));  // of the head, over the four lane groups
        const bool moves = top > m_run + kTop;
        const float to = moves ? top - kBias : m_run, al = moves ? fast_exp2(m_run - to) : 1.0f;
        m_run = to;
        l_run *= al;
        corr *= al;
#pragma unroll
        for (int t = 0; t < DPL; ++t) acc[t] *= al;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] = fast_exp2(s[i] - m_run);
        l_run += s[i];
      }
    };
    auto outputs = [&](typename R::V& r, int chunk, const Tiles& t, float (&s)[8]) {
      if (!whole(chunk, t)) {  // what lies in masked places may be infinite or NaN
#pragma unroll
        for (int gi = 0; gi < 2; ++gi)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!live(chunk, t, gi, i)) {
              if constexpr (CODES) {
                r.scale[gi][i] = 0.0f;
                r.zp[gi][i] = 0;
              } else {
#pragma unroll
                for (int y = 0; y < R::VW; ++y) r.w[4 * gi + i][y] = 0u;
              }
            }
      }
      if constexpr (CODES) {
        float top = r.scale[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, r.scale[i >> 2][i & 3]);
        if (__any(top > unit_v)) {
          top = max_halves(max_row_pairs(top));
          if (top > unit_v) {
            const int ex = min((int)(__float_as_uint(top) >> 23) + 1, 253);
            const float to = __uint_as_float((uint32_t)ex << 23), al = unit_v * __uint_as_float((uint32_t)(254 - ex) << 23);
            unit_v = to;
            per_v = __uint_as_float((uint32_t)(254 - ex) << 23);
            corr *= al;
#pragma unroll
            for (int t = 0; t < DPL; ++t) acc[t] *= al;
          }
        }
        constexpr int MID = U4 ? 8 : 128;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[i] *= r.scale[i >> 2][i & 3] * per_v;
          corr = fmaf(s[i], (float)(r.zp[i >> 2][i & 3] - MID), corr);
        }
      }
      const u32x4_t pb = {pack_pair<P16>(s[0], s[1]), pack_pair<P16>(s[2], s[3]), pack_pair<P16>(s[4], s[5]), pack_pair<P16>(s[6], s[7])};
      if constexpr (CODES) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += elem_lo<true>(pb[i]) + elem_hi<true>(pb[i]);
        corr = fmaf(sum, U4 ? 8.0f : 128.0f, corr);
      }
#pragma unroll
      for (int t = 0; t < DPL; ++t) acc[t] = mfma_16x16x32<P16>(R::v_operand(r, t), pb, acc[t]);
    };

    int chunk = k_begin + 32 * wave;
    if (chunk < k_end) {
      Tiles now = pages(chunk), next = pages(chunk + UNIT);
      typename R::K k;
      typename R::V v;
      float s[8];
      load_k(k, chunk, now);
      load_v(v, chunk, now);
      for (; chunk + UNIT < k_end; chunk += UNIT) {
        const Tiles then = pages(chunk + 2 * UNIT);
        logits(k, chunk, now, s);
        __builtin_amdgcn_sched_barrier(0);  // the loads below reuse the registers consumed above
        load_k(k, chunk + UNIT, next);
        __builtin_amdgcn_sched_barrier(0);
        weights(s);
        outputs(v, chunk, now, s);
        __builtin_amdgcn_sched_barrier(0);
        load_v(v, chunk + UNIT, next);
        __builtin_amdgcn_sched_barrier(0);
        now = next;
        next = then;
      }
      logits(k, chunk, now, s);
      weights(s);
      outputs(v, chunk, now, s);
    }

    // ---- the four wavefronts' results, joined
    auto over_groups = [](float x) {
      const u32pair_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    };
    const float l = over_groups(l_run);
    if constexpr (CODES) {
      corr = over_groups(corr);
#pragma unroll
      for (int t = 0; t < DPL; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = (acc[t][i] * (U4 && t < DPL / 2 ? 0x1p20f : 0x1p24f) - corr) * unit_v;
    }
    if (m < p.Gr) {
#pragma unroll
      for (int t = 0; t < DPL; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][m][R::dmap(t, 4 * kg + i)] = acc[t][i];
      if (kg == 0) {
        red_m[wave][m] = m_run;
        red_l[wave][m] = l;
      }
    }
    __syncthreads();
    const bool alone = first == 0 && n_units == units;  // the pair is this workgroup's alone
    const int slot = 2 * w + (first == 0 ? 1 : 0);
    if (tid < p.Gr) {
      float top = red_m[0][tid], sum = 0.0f;
#pragma unroll
      for (int i = 1; i < WAVES; ++i) top = fmaxf(top, red_m[i][tid]);
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const float f = fast_exp2(red_m[i][tid] - top);
        weight[i][tid] = f;
        sum += red_l[i][tid] * f;
      }
      fin[0][tid] = alone ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
      if (alone) {
        if (p.a.lse) p.a.lse[(int64_t)b * p.a.Hq + h * p.Gr + tid] = sum == 0.0f ? -INFINITY : top + fast_log2(sum);
      } else {
        *(f32x2_t*)(p.part_ml + ((int64_t)slot * p.Gr + tid) * 2) = f32x2_t{top, sum};
      }
    }
    __syncthreads();
    for (int i = tid; i < p.Gr * (D / 4); i += NT) {
      const int g = i / (D / 4), d = 4 * (i % (D / 4));
      f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < WAVES; ++j) x += *(const f32x4_t*)&red[j][g][d] * weight[j][g];
      if (alone) {
        x *= fin[0][g];
        *(u32x2_t*)((uint16_t*)p.a.o + b * p.a.o_stride_b + (int64_t)(h * p.Gr + g) * p.a.o_stride_h + d) = u32x2_t{pack_pair<F16>(x[0], x[1]), pack_pair<F16>(x[2], x[3])};
      } else {
        *(f32x4_t*)(p.part_o + ((int64_t)slot * p.Gr + g) * D + d) = x;
      }
    }
    if (tid == 0 && first == 0 && !alone) {
      p.part_of[2 * w] = b * Hkv + h;
      p.part_of[2 * w + 1] = shares.owner(begin + units - 1) - w + 1;
    }
    __syncthreads();  // LDS is free again

    unit += n_units;
    if (unit == begin_b + units * Hkv) {
      begin_b = unit;
      ++b;
    }
  }
}

// The partials of the pair that workgroup blockIdx.x of the launch above left off in: 256 values of its outputs, four a lane; the wavefronts share the partials.
template <int D, bool F16>
__global__ __launch_bounds__(NT) void paged_join_kernel(const PagedParams p) {
  const int w = blockIdx.x, n = p.part_of[2 * w + 1];
  if (n == 0) return;
  __shared__ __align__(16) float red[WAVES][64][4];
  __shared__ float red_m[WAVES][64], red_l[WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.y * 256 + 4 * lane, g = min(i / D, p.Gr - 1), d = i % D;
  const int pair = p.part_of[2 * w], b = pair / p.a.pages.Hkv, h = pair - b * p.a.pages.Hkv;
  float top = kLowest, sum = 0.0f;
  f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = wave; s < n; s += WAVES) {
    const int64_t slot = s == 0 ? 2 * w + 1 : 2 * (w + s);
    const f32x2_t ml = *(const f32x2_t*)(p.part_ml + (slot * p.Gr + g) * 2);
    const f32x4_t y = *(const f32x4_t*)(p.part_o + (slot * p.Gr + g) * D + d);
    const float to = fmaxf(top, ml[0]), al = fast_exp2(top - to), be = fast_exp2(ml[0] - to);
    top = to;
    sum = sum * al + ml[1] * be;
    x = x * al + y * be;
  }
  *(f32x4_t*)red[wave][lane] = x;
  red_m[wave][lane] = top;
  red_l[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || i >= p.Gr * D) return;
  float all = red_m[0][lane];
#pragma unroll
  for (int j = 1; j < WAVES; ++j) all = fmaxf(all, red_m[j][lane]);
  sum = 0.0f;
  x = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < WAVES; ++j) {
    const float f = fast_exp2(red_m[j][lane] - all);
    sum += red_l[j][lane] * f;
    x += *(const f32x4_t*)red[j][lane] * f;
  }
  x *= sum == 0.0f ? 0.0f : 1.0f / sum;
  *(u32x2_t*)((uint16_t*)p.a.o + b * p.a.o_stride_b + (int64_t)(h * p.Gr + g) * p.a.o_stride_h + d) = u32x2_t{pack_pair<F16>(x[0], x[1]), pack_pair<F16>(x[2], x[3])};
  if (p.a.lse && d == 0) p.a.lse[(int64_t)b * p.a.Hq + h * p.Gr + g] = sum == 0.0f ? -INFINITY : all + fast_log2(sum);
}

PagedParams params_of(const kvx_paged_decode_args& a) {
  PagedParams p{};
  p.a = a;
  p.c = a.sm_scale * kLog2e;
  p.shift = __builtin_ctz(a.pages.page_size);
  p.cap = a.max_pages << p.shift;
  p.Gr = a.Hq / a.pages.Hkv;
  const int per_cu = a.pages.D == 256 ? (kv_is_plain(a.pages.kv_dtype) ? 1 : 2) : 3;
  const int64_t units = (int64_t)a.B * a.pages.Hkv * ((p.cap + UNIT - 1) / UNIT), most = (int64_t)per_cu * num_cus();
  p.workgroups = (int)(units < most ? units : most);
  return p;
}
bool splits(const PagedParams& p) { return p.cap > UNIT; }

template <int D>
void launch_head(const PagedParams& p, hipStream_t st) {
  switch (p.a.pages.kv_dtype) {
#define KVX_PAGES_CASE(KV) case KV: hipLaunchKernelGGL((paged_decode_kernel<D, KV>), dim3(p.workgroups), dim3(NT), 0, st, p); break;
    KVX_PAGES_CASE(KVX_KV_BF16)
    KVX_PAGES_CASE(KVX_KV_F16)
    KVX_PAGES_CASE(KVX_KV_U8)
    KVX_PAGES_CASE(KVX_KV_U4)
    KVX_PAGES_CASE(KVX_KV_U8_F16)
    KVX_PAGES_CASE(KVX_KV_U4_F16)
#undef KVX_PAGES_CASE
  }
  if (!splits(p)) return;
  const dim3 grid(p.workgroups, (p.Gr * D + 255) / 256);
  if (kv_elem_f16(p.a.pages.kv_dtype)) hipLaunchKernelGGL((paged_join_kernel<D, true>), grid, dim3(NT), 0, st, p);
  else hipLaunchKernelGGL((paged_join_kernel<D, false>), grid, dim3(NT), 0, st, p);
}

size_t part_floats(const PagedParams& p) { return (size_t)2 * p.workgroups * p.Gr * p.a.pages.D; }

}  // namespace

size_t paged_decode_workspace(const kvx_paged_decode_args& a) {
  const PagedParams p = params_of(a);
  return 4 * (part_floats(p) + (size_t)4 * p.workgroups * p.Gr + 2 * p.workgroups);
}

int launch_paged_decode(const kvx_paged_decode_args& a, hipStream_t st) {
  PagedParams p = params_of(a);
  p.part_o = (float*)a.workspace;
  p.part_ml = p.part_o + part_floats(p);
  p.part_of = (int*)(p.part_ml + (size_t)4 * p.workgroups * p.Gr);
  if (a.pages.D == 256) launch_head<256>(p, st);
  else if (a.pages.D == 128) launch_head<128>(p, st);
  else launch_head<64>(p, st);
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
