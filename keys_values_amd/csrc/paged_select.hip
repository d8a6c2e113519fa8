// Which pages of a sequence a query attends to, for gfx950: bounds of a page's keys, and the choice by what they allow.
//   low, high = min, max over the page's keys, value by value (rows of codes: of the rows that they stand for, rounded to 16 bits);
//   score = max over the query heads of a KV head of sum_d max(q_d low_d, q_d high_d) = sum_d (q+_d high_d + q-_d low_d),
// which no product of the queries with the page's keys exceeds, codes' keys being those that are rounded (to nearest: bounds are what paged_read gives). Attention over codes takes them unrounded, and a
// product there may be larger by 2^-8 (bf16; fp16 2^-11) of its sum of |q_d k_d|; in pages of one token about every second one is.
#include <type_traits>

#include "page_rows.h"
#include "work_shares.h"

namespace kvx {
namespace {

// Minimum and maximum that hand on a NaN (llvm.minimum: v_minimum3_f32)
__device__ __forceinline__ float lowest(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float highest(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// min / max over the halves of a wavefront, then over the rows of 16 of a half, of two registers at a time: lanes trade the half (or row) of one register for that of the
// other, so that a result has both. x[] shrinks by half with every step.
template <int N, typename F>
__device__ __forceinline__ void fold_halves(float (&x)[N], F best) {
#pragma unroll
  for (int e = 0; e < N / 2; ++e) {
    const u32pair_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[e]), __float_as_uint(x[e + N / 2]), false, false);
    x[e] = best(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
}
template <int N, typename F>
__device__ __forceinline__ void fold_rows(float (&x)[N], F best) {  // of x[0 .. N / 2)
#pragma unroll
  for (int e = 0; e < N / 4; ++e) {
    const u32pair_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(x[e + N / 4]), false, false);
    x[e] = best(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
}

// W wavefronts a (page, KV head); D / 8 lanes a row, U rows a lane at a time. HBM-bound. The pages of all sequences are dealt out to a fixed number of workgroups, a stretch of
// neighbouring (page, head) each, and a wavefront has the first rows of its next one on their way while it folds one. A page's last rows are looked at again in place of those that it does
// not have: all loads of a step are on their way before the first is waited for.
// 142000 tokens in pages of 16, 8 heads of 128 (290 MB of keys, 37 of bounds): 64 us, with loads through the caches 71. A grid of all pages that the tables have room for takes 63
// there, but longer the emptier the tables are.
// W goes by the page's size, 1 up to 32, 4 up to 128, 16 above (same tokens, us with 1, 4 and 16): pages of 32 60, 68, 291; 64 63, 61, 154; 128 60, 61, 86; 256 60 with any; 1024 66, 60, 62.
// Of the newest page of 32 sequences alone: 64 3.8, 3.4, 5.1; 256 6.3, 5.5, 5.2; 1024 38.9, 14.3, 13.0. Pages of codes, which have less to load, would take fewer: 8-bit
// pages of 64 40.5, 45.7, 186; of 256 35.3, 34.2, 54.
template <int D, int KV, int W>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void paged_bounds_kernel(const kvx_paged_bounds_args a, const int shift) {
  constexpr bool PLAIN = kv_is_plain(KV), U4 = kv_is_u4(KV), F16 = kv_elem_f16(KV);
  constexpr int LPR = D / 8, ROWS = 64 / LPR, ES = PLAIN ? 2 : 1, U = 4, NT = W == 16 ? 1024 : 256, AT_ONCE = NT / 64 / W;
  const kvx_pages& p = a.pages;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, B = a.B, Hkv = p.Hkv, cap = a.max_pages << shift;

  // ---- this workgroup's share: every wavefront finds it for itself, 64 sequences at a time
  const int windows = (B + 63) / 64;
  auto window = [&](int i) { return 64 * i + lane < B ? min(max(a.lens[64 * i + lane], 0), cap) : 0; };
  auto begin_of = [&](int len) { return max(len - a.tokens, 0) >> shift; };  // the first page that is looked at
  auto pages_in = [&](int len) { return ((len + p.page_size - 1) >> shift) - begin_of(len); };
  int lane_len = 0, mine = 0;  // lane_len: of sequence (b & ~63) + lane
  for (int i = 0; i < windows; ++i) {
    lane_len = window(i);
    mine += pages_in(lane_len);
  }
  const Shares shares(__builtin_amdgcn_readlane(scan(mine), 63) * Hkv, gridDim.x);
  int unit = shares.first(blockIdx.x) + wave / W;
  const int end = shares.first(blockIdx.x + 1);
  if (unit >= end) return;  // all wavefronts of a (page, head), which are all of the workgroup where they wait for each other
  int b = 0, begin_b = 0;   // the unit's sequence, and the sequence's first unit
  for (int i = 0, before = 0;; ++i) {
    if (windows > 1) lane_len = window(i);
    mine = pages_in(lane_len);
    const int upto = before + scan(mine);
    const unsigned long long behind = __ballot(upto * Hkv > unit);
    if (behind) {
      const int at = __builtin_ctzll(behind);
      b = 64 * i + at;
      begin_b = __builtin_amdgcn_readlane(upto - mine, at) * Hkv;
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }

  const int col = lane % LPR;
  struct Item {
    int entry, h, rows;  // of the table; rows that hold tokens
  };
  auto item_of = [&](int unit) {  // units come in rising order
    for (;;) {
      const int len = __builtin_amdgcn_readlane(lane_len, b & 63), units = pages_in(len) * Hkv;
      if (unit < begin_b + units) {
        const int i = (unit - begin_b) / Hkv, page = begin_of(len) + i;
        return Item{a.block_table[b * a.bt_stride_b + page], unit - begin_b - i * Hkv, min(len - (page << shift), p.page_size)};
      }
      begin_b += units;
      ++b;
      if ((b & 63) == 0) lane_len = window(b >> 6);
    }
  };
  struct Step {
    u32x4_t w[U];
    float scale[U];
    int32_t zp[U];
  };
  auto load = [&](Step& s, const Item& t, int r0) {
    const int64_t page = (uint32_t)t.entry < (uint32_t)p.num_pages ? t.entry : 0;  // of a page that the pool does not have nothing is kept
    const uint8_t* k = (const uint8_t*)p.k + (page * p.k_stride_page + t.h * p.k_stride_h) * ES + (PLAIN ? 16 * col : U4 ? (int)u4_byte_off<D>(col) : 8 * col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = min(r0 + u * ROWS + lane / LPR, t.rows - 1);
      const uint8_t* at = k + (uint32_t)r * (uint32_t)(p.k_stride_t * ES);
      if constexpr (PLAIN) {
        s.w[u] = __builtin_nontemporal_load((const u32x4_t*)at);
      } else {
        const u32x2_t c = __builtin_nontemporal_load((const u32x2_t*)at);
        s.w[u] = u32x4_t{c[0], c[1], 0u, 0u};
        const int64_t q = page * p.qs_stride_page + t.h * p.qs_stride_h + r;
        s.scale[u] = p.k_scale[q];
        s.zp[u] = p.k_zp[q];
      }
    }
  };
  float lo[8], hi[8];
  auto take = [&](const Step& s) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8];
      if constexpr (PLAIN) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = elem_lo<F16>(s.w[u][e]);
          x[2 * e + 1] = elem_hi<F16>(s.w[u][e]);
        }
      } else {
        u32x2_t c = {s.w[u][0], s.w[u][1]};
        if constexpr (U4) c = u4_codes(c, u4_shift<D>(col));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)((int32_t)((c[e >> 2] >> (8 * (e & 3))) & 0xff) - s.zp[u]) * s.scale[u];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = lowest(lo[e], x[e]);
        hi[e] = highest(hi[e], x[e]);
      }
    }
  };
  // over the lanes of a value: a lane keeps VALUES of its 8, from `first` on
  constexpr int VALUES = D == 256 ? 4 : 2;
  auto fold = [&](float (&x)[8], auto best) {
    fold_halves(x, best);
    if constexpr (D <= 128) fold_rows(x, best);
    if constexpr (D == 64)
#pragma unroll
      for (int e = 0; e < VALUES; ++e) x[e] = best(x[e], __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x[e]), 0x128, 0xf, 0xf, true)));  // row_ror:8
  };
  const int first = 8 * col + (D == 256 ? lane >> 5 << 2 : lane >> 4 << 1);
  auto bounds_of = [&](const Item& t, Step& s) {  // s: the first rows
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = INFINITY;
      hi[e] = -INFINITY;
    }
    for (int r0 = wave % W * ROWS * U;;) {
      take(s);
      r0 += W * ROWS * U;
      if (r0 >= t.rows) break;
      load(s, t, r0);
    }
    fold(lo, lowest);
    fold(hi, highest);
    if constexpr (W > 1) {
      __shared__ __align__(16) float joined[NT / 64][2][D];
#pragma unroll
      for (int e = 0; e < VALUES; ++e) {
        joined[wave][0][first + e] = lo[e];
        joined[wave][1][first + e] = hi[e];
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll 3
        for (int w = 1; w < W; ++w)
#pragma unroll
          for (int e = 0; e < VALUES; ++e) {
            lo[e] = lowest(lo[e], joined[w][0][first + e]);
            hi[e] = highest(hi[e], joined[w][1][first + e]);
          }
      }
      __syncthreads();
      if (wave != 0) return;
    }
    if ((uint32_t)t.entry >= (uint32_t)p.num_pages || (D == 64 && (lane & 8))) return;
    uint16_t* to = (uint16_t*)a.bounds + (int64_t)t.entry * a.b_stride_page + t.h * a.b_stride_h + first;
#pragma unroll
    for (int e = 0; e < VALUES; e += 2) {
      *(uint32_t*)(to + e) = pack_pair<F16>(lo[e], lo[e + 1]);
      *(uint32_t*)(to + a.b_stride_side + e) = pack_pair<F16>(hi[e], hi[e + 1]);
    }
  };
  Step one, two;
  Item now = item_of(unit), next = now, then = now;  // behind the last, the last one is read again
  if (unit + AT_ONCE < end) next = then = item_of(unit + AT_ONCE);
  load(one, now, wave % W * ROWS * U);
  for (;; unit += 2 * AT_ONCE) {
    if (unit + 2 * AT_ONCE < end) then = item_of(unit + 2 * AT_ONCE);
    load(two, next, wave % W * ROWS * U);
    __builtin_amdgcn_sched_barrier(0);
    bounds_of(now, one);
    if (unit + AT_ONCE >= end) break;
    now = then;
    if (unit + 3 * AT_ONCE < end) then = item_of(unit + 3 * AT_ONCE);
    load(one, now, wave % W * ROWS * U);
    __builtin_amdgcn_sched_barrier(0);
    bounds_of(next, two);
    if (unit + 2 * AT_ONCE >= end) break;
    next = then;
  }
}

// ---- the choice ------------------------------------------------------------------------------------------------------------------

constexpr uint32_t kNever = 0u, kInfinite = 0xfffffffdu, kAlways = 0xfffffffeu;

// Keys of scores: unsigned numbers in their order, between kNever and kInfinite. What is not finite counts as infinite.
__device__ __forceinline__ uint32_t key_of(double sum) {
  const float s = (float)sum + 0.0f;  // no -0
  const uint32_t bits = __float_as_uint(s);
  if (!(fabsf(s) < INFINITY)) return kInfinite;
  return (bits >> 31) ? ~bits : bits | 0x80000000u;
}

struct SelectParams {
  kvx_paged_select_args a;
  uint32_t* keys;  // (B, Hkv, stride)
  int stride;      // of tables' pages, in fours
  int shift;       // log2 of the page size
  int all_keys;    // few enough for all that a list has room for to be read, while its length is: 48 sequences of up to 8192 pages, 4 heads, 7.7 us, 8.4 without
  __device__ __forceinline__ int pages(int b) const { return (min(max(a.lens[b], 0), a.max_pages << shift) + a.page_size - 1) >> shift; }  // of a sequence
};

// v_mfma_f64_4x4x4, four blocks of 4 pages, 4 heads and 4 values: lane l has a value of page l % 16 (A), of head l % 4 (B), and gets the sum of page
// 4 (l / 4 % 4) + l / 16 and head l % 4. Products of 16-bit values are exact in 64 bits (bfloat16 ones go beyond the range of 32). The order of a page's sum is the same in every kernel, for every
// split and place, so that the choice does not depend on these, and pages alike tie. In another order it may be off by D * 2^-53 of sum |q_d bound_d|, where the rounding to 32 bits sees 2^-24 of the
// score: where large terms cancel the two orders round differently.
// A wavefront takes 16 pages at a time and has the next 16 on their way meanwhile. Queries wait in LDS as pairs q+, q- of 64 bits, the 16 pairs of an instruction
// side by side. An instruction takes 16 cycles (v_mfma_f64_16x16x4, four times as much work, a hundred).
//
// The pages of all (sequence, KV head) pairs are cut into units and dealt out to a fixed number of workgroups, each a stretch of neighbouring units, as paged_decode does with
// keys. A grid of all units that the table has room for, whatever the lengths: 93 us for 48 sequences of 300 to 131072 tokens in pages of 16, 28 / 4 heads of 128, 42 as it is.
// Bounds of 134 MB (8 sequences of 131072 tokens in pages of 32, 32 / 8 heads of 128) take 31 us, 5 of them before the first ones arrive; with two workgroups a compute
// unit that hold twice as many each 33, with loads past the caches 3 more.
constexpr int UNIT = NTHREADS / 64 * 16;  // pages

// What a wavefront scores 16 pages of one (sequence, KV head) with; `q`: the queries in LDS
template <int D, bool F16, int HEADS /* of the group, in fours */>
struct Scorer {
  typedef double f64x2_t __attribute__((ext_vector_type(2)));
  typedef f64x2_t Queries[HEADS][D / 32][8][4][4];  // value 32 x + 8 kg + j of head 4 f + g at [f][x][j][kg][g]
  struct Tile {
    u32x4_t lo[D / 32], hi[D / 32];
    int page;  // of the pool, of page lane % 16 of the tile; -1: none
  };
  const kvx_paged_select_args& a;
  const Queries& q;
  const int* table;
  const uint16_t* bounds;
  int lane, n, last;  // pages of the sequence, and those that are scored end here

  __device__ __forceinline__ Scorer(const kvx_paged_select_args& a, const Queries& q, int b, int h, int n, int last)
      : a(a), q(q), table(a.block_table + b * a.bt_stride_b), lane(threadIdx.x & 63), n(n), last(last) {
    bounds = (const uint16_t*)a.bounds + h * a.b_stride_h + 8 * (lane >> 4);
  }
  // The queries to LDS, by all lanes of a workgroup of NT: on their way from construction on, so that what a wavefront waits for before `put` is theirs and not the bounds'
  template <int NT>
  struct Fetch {
    static constexpr int ALL = 4 * HEADS * (D / 8), EACH = (ALL + NT - 1) / NT;
    u32x4_t w[EACH];
    __device__ __forceinline__ Fetch(const kvx_paged_select_args& a, int b, int h) {
      const int G = a.Hq / a.Hkv;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = min((int)threadIdx.x + e * NT, ALL - 1), g = i % (4 * HEADS), col = i / (4 * HEADS);
        w[e] = *(const u32x4_t*)((const uint16_t*)a.q + b * a.q_stride_b + (int64_t)(h * G + min(g, G - 1)) * a.q_stride_h + 8 * col);
      }
    }
    __device__ __forceinline__ void put(Queries& q) const {  // heads behind the group's last: copies of it, whose sums nobody looks at
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = threadIdx.x + e * NT, g = i % (4 * HEADS), col = i / (4 * HEADS);
        if (i < ALL) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = j & 1 ? elem_hi<F16>(w[e][j >> 1]) : elem_lo<F16>(w[e][j >> 1]);
            q[g >> 2][col >> 2][j][col & 3][g & 3] = f64x2_t{x > 0.0f ? x : 0.0f, x > 0.0f ? 0.0f : x};  // a NaN is the second's
          }
        }
      }
    }
  };
  __device__ __forceinline__ int entry(int first) const { return table[min(first + (lane & 15), a.max_pages - 1)]; }  // does not wait for n
  __device__ __forceinline__ void load(Tile& r, int entry, int first) const {
    r.page = first + (lane & 15) < last && (uint32_t)entry < (uint32_t)a.num_pages ? entry : -1;
    const uint16_t* at = bounds + (int64_t)max(r.page, 0) * a.b_stride_page;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      r.lo[x] = *(const u32x4_t*)(at + 32 * x);
      r.hi[x] = *(const u32x4_t*)(at + a.b_stride_side + 32 * x);
    }
  }
  __device__ __forceinline__ void score(const Tile& r, int first, uint32_t* keys) const {
    asm volatile("" ::: "memory");  // the queries are read anew, not held in registers, of which there are too few
    const int kg = lane >> 4, G = a.Hq / a.Hkv;
    double up[HEADS], down[HEADS];
#pragma unroll
    for (int f = 0; f < HEADS; ++f) up[f] = down[f] = 0.0;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double l = j & 1 ? elem_hi<F16>(r.lo[x][j >> 1]) : elem_lo<F16>(r.lo[x][j >> 1]), u = j & 1 ? elem_hi<F16>(r.hi[x][j >> 1]) : elem_lo<F16>(r.hi[x][j >> 1]);
#pragma unroll
        for (int f = 0; f < HEADS; ++f) {
          const f64x2_t w = q[f][x][j][kg][lane & 3];
          up[f] = __builtin_amdgcn_mfma_f64_4x4x4f64(u, w[0], up[f], 0, 0, 0);
          down[f] = __builtin_amdgcn_mfma_f64_4x4x4f64(l, w[1], down[f], 0, 0, 0);
        }
      }
    uint32_t key = kNever;
#pragma unroll
    for (int f = 0; f < HEADS; ++f)
      if (4 * f + (lane & 3) < G) key = max(key, key_of(up[f] + down[f]));
    key = max(key, (uint32_t)__builtin_amdgcn_mov_dpp((int)key, 0xB1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
    key = max(key, (uint32_t)__builtin_amdgcn_mov_dpp((int)key, 0x4E, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
    const int mine = (lane & 12) + kg, i = first + mine;  // the page whose sums this lane has
    const unsigned long long pages = __ballot(r.page >= 0);
    if (!((pages >> mine) & 1)) key = kNever;
    else if (i < a.first || i >= n - a.last) key = kAlways;
    if ((lane & 3) == 0 && i < last) keys[i] = key;
  }
  // Pages first, first + each, ... below `last`, 16 at a time, with the next 16 on their way. A tile's entries of the table are read one tile ahead of its bounds, and before those of the
  // tile in between: what waits for them waits for nothing else. Behind the last page, page 0 of the pool is read: loads under a condition would have to be waited for whether they
  // are there or not. `ready`: what has to be done before the queries are read
  template <typename F>
  __device__ __forceinline__ void run(int first, int each, uint32_t* keys, F ready) const {
    int next = entry(first), then = entry(first + each);
    Tile one, two;
    load(one, next, first);
    __builtin_amdgcn_sched_barrier(0);
    ready();
    for (; first < last; first += 2 * each) {
      next = entry(first + 2 * each);
      __builtin_amdgcn_sched_barrier(0);
      load(two, then, first + each);
      __builtin_amdgcn_sched_barrier(0);
      score(one, first, keys);
      if (first + each >= last) break;
      __builtin_amdgcn_sched_barrier(0);
      then = entry(first + 3 * each);
      __builtin_amdgcn_sched_barrier(0);
      load(one, next, first + 2 * each);
      __builtin_amdgcn_sched_barrier(0);
      score(two, first + each, keys);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Workgroups a compute unit. Registers leave room for four with rows of 128, two with rows of 256 and more than four heads a group; elsewhere for more, which would take a little less: rows of 64
// (16 sequences of 131072 in pages of 32, 32 / 8 heads) 34.3 us with six, 35.4 with four; rows of 256 and up to four heads (4 such sequences) 35.3 with three, 36.3 with two.
constexpr int score_workgroups(int D) { return D == 256 ? 2 : 4; }
template <int D, bool F16, int HEADS /* of the group, in fours */>
__global__ __launch_bounds__(NTHREADS, score_workgroups(D)) void select_score_kernel(const SelectParams p) {
  typedef Scorer<D, F16, HEADS> S;
  const kvx_paged_select_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), B = a.B, Hkv = a.Hkv;
  __shared__ __align__(16) typename S::Queries qs;

  // ---- this workgroup's units: every wavefront finds them for itself, 64 sequences at a time
  const int windows = (B + 63) / 64;
  auto window = [&](int i) { return 64 * i + lane < B ? p.pages(64 * i + lane) : 0; };
  auto units_in = [&](int pages) { return (pages + UNIT - 1) / UNIT; };
  int lane_pages = 0, mine = 0;  // lane_pages: of sequence (b & ~63) + lane
  for (int i = 0; i < windows; ++i) {
    lane_pages = window(i);
    mine += units_in(lane_pages);
  }
  const Shares shares(__builtin_amdgcn_readlane(scan(mine), 63) * Hkv, gridDim.x);
  int unit = shares.first(blockIdx.x);
  const int end = shares.first(blockIdx.x + 1);
  if (unit >= end) return;
  int b = 0, begin_b = 0;  // the unit's sequence, and the sequence's first unit
  for (int i = 0, before = 0;; ++i) {
    if (windows > 1) lane_pages = window(i);
    mine = units_in(lane_pages);
    const int upto = before + scan(mine);
    const unsigned long long behind = __ballot(upto * Hkv > unit);
    if (behind) {
      const int at = __builtin_ctzll(behind);
      b = 64 * i + at;
      begin_b = __builtin_amdgcn_readlane(upto - mine, at) * Hkv;
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }

  for (bool again = false;; again = true) {
    const int n = __builtin_amdgcn_readlane(lane_pages, b & 63), units = units_in(n);
    if (units > 0) {
      const int h = (unit - begin_b) / units, from = unit - begin_b - h * units, count = min(units - from, end - unit), pair = b * Hkv + h;
      const typename S::template Fetch<NTHREADS> queries(a, b, h);
      const S s(a, qs, b, h, n, min(n, (from + count) * UNIT));
      s.run(from * UNIT + wave * 16, UNIT, p.keys + (int64_t)pair * p.stride, [&] {
        if (again) __syncthreads();  // the queries before are read
        queries.put(qs);
        __syncthreads();
      });
      unit += count;
      if (unit >= end) break;
    }
    if (unit == begin_b + units * Hkv) {
      begin_b = unit;
      ++b;
      if ((b & 63) == 0 && b < B) lane_pages = window(b >> 6);
    }
  }
}

// Scores and choice in one launch, a workgroup for a (sequence, KV head) of up to 128 pages: 16 a wavefront, whose keys meet in LDS, where each is compared with all others.
// 64 pages, 32 / 8 heads of 128: 1 sequence 6.5 us, in two launches 5.4 and 3.8 and what lies between, 32 sequences 6.7, 5.6 and 4.2, 128 16.0, 12.6 and 5.6. With more pages a
// workgroup that has them alone takes longer: 512 pages, 1 sequence, 13.6, 5.5 and 4.1.
constexpr int FEW = 128;
template <int D, bool F16, int HEADS>
__global__ __launch_bounds__(4 * FEW) void select_few_kernel(const SelectParams p) {
  typedef Scorer<D, F16, HEADS> S;
  const kvx_paged_select_args& a = p.a;
  __shared__ __align__(16) typename S::Queries qs;
  __shared__ __align__(16) uint32_t keys[FEW];
  __shared__ int taken[FEW / 16];
  const int b = blockIdx.y, h = blockIdx.x, pair = b * a.Hkv + h, tid = threadIdx.x, lane = tid & 63;
  const typename S::template Fetch<4 * FEW> queries(a, b, h);
  const int n = p.pages(b);
  if (tid < FEW) keys[tid] = kNever;
  const S s(a, qs, b, h, n, n);
  const int first = 16 * __builtin_amdgcn_readfirstlane(tid >> 6);
  auto ready = [&] {
    queries.put(qs);
    __syncthreads();
  };
  if (first < n) s.run(first, FEW, keys, ready);
  else ready();
  __syncthreads();
  // four lanes a key, each of which compares it with a quarter of the others
  const int i = tid >> 2, part = tid & 3;
  const uint32_t key = keys[i];
  int before = 0;  // keys that come first
#pragma unroll
  for (int j = 0; j < FEW / 4; j += 4) {
    const u32x4_t x = *(const u32x4_t*)(keys + FEW / 4 * part + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) before += x[e] + (FEW / 4 * part + j + e < i) > key;  // of equal ones those in front; no key is the largest of all words
  }
  before += __builtin_amdgcn_mov_dpp(before, 0xB1, 0xf, 0xf, true);  // quad_perm [1,0,3,2]
  before += __builtin_amdgcn_mov_dpp(before, 0x4E, 0xf, 0xf, true);  // quad_perm [2,3,0,1]
  const bool take = key != kNever && before < a.count;
  const unsigned long long m = __ballot(take && part == 0);
  if (lane == 0) taken[tid >> 6] = __popcll(m);
  __syncthreads();
  int to = __popcll(m & ((1ull << lane) - 1)), all = 0;
#pragma unroll
  for (int w = 0; w < FEW / 16; ++w) {
    to += w < tid >> 6 ? taken[w] : 0;
    all += taken[w];
  }
  int32_t* out = a.chosen + (int64_t)pair * a.count;
  if (take && part == 0) out[to] = i;
  for (int j = all + tid; j < a.count; j += 4 * FEW) out[j] = -1;
}

// The `count` largest keys of a (sequence, KV head), of equal ones the first, in order of their pages, for up to R * NT pages: R neighbours a lane, which stay in registers. The last key
// that is taken lies in one of 2048 equal parts of a range of keys, found by counting, then in one of 2048 parts of that, until no more of its part are left over (after three times a part is
// one key). By their upper bits instead, as the long form does, most keys would count in the same few places, one after the other.
// What bounds it is that it runs once: a few workgroups fetch each of its instructions from afar, about 130 cycles for 64 bytes of them, more than the work itself takes. Hence one
// order for all of a lane's keys, sums over wavefronts by lanes and not one after the other, a loop for the few that are taken: 8 lists of 8192 pages, 7.0 KB of code 6.6 us, 3.3 KB 5.1.
// Keys that cannot be among the `count` largest kept from being counted (by the largest of groups of lanes): no gain.
template <int R, int NT>
__global__ __launch_bounds__(NT) void select_choose_kernel(const SelectParams p) {
  constexpr int BINS = 2048, WAVES = NT / 64, EACH = BINS / NT;  // EACH: parts a lane counts up, from the largest down
  const kvx_paged_select_args& a = p.a;
  const int b = blockIdx.y, pair = b * a.Hkv + blockIdx.x, n = p.pages(b), tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), first = R * tid;
  __shared__ int counts[BINS], sums[WAVES], placed[WAVES], at_bin, at_rest, at_count;
  __shared__ __align__(16) u32x4_t ranges[WAVES];
  const uint32_t* keys = p.keys + (int64_t)pair * p.stride;
  int32_t* out = a.chosen + (int64_t)pair * a.count;
  uint32_t key[R];
  constexpr int V = R < 4 ? R : 4;
  typedef uint32_t Keys __attribute__((ext_vector_type(V)));
  Keys x[R / V] = {};
  if (p.all_keys) {  // does not wait for n
#pragma unroll
    for (int v = 0; v < R / V; ++v) x[v] = *(const Keys*)(keys + min(first + V * v, p.stride - V));
  } else {
#pragma unroll
    for (int v = 0; v < R / V; ++v)
      if (first + V * v < n) x[v] = *(const Keys*)(keys + first + V * v);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = x[r / V][r % V];
#pragma unroll
  for (int e = 0; e < EACH; ++e) counts[NT * e + tid] = 0;
  // ---- range of the keys that are neither taken anyway nor left out, and the numbers of those
  uint32_t low = kAlways, high = kNever;
  uint32_t number = 0;  // those that are taken anyway << 16 | the others: of a workgroup at most R * NT in all, which is 32768
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (first + r >= n) key[r] = kNever;
    const bool other = key[r] != kNever && key[r] != kAlways;
    low = other ? min(low, key[r]) : low;
    high = other ? max(high, key[r]) : high;
    number += key[r] == kAlways ? 1u << 16 : other ? 1u : 0u;
  }
  auto fold = [&](auto ctrl, auto rows) {
    auto other = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false); };
    low = min(low, other(low));
    high = max(high, other(high));
    number += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)number, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  const std::integral_constant<int, 0xf> every;
  auto fold_row = [&](int lanes) {
    fold(std::integral_constant<int, 0xB1>{}, every);   // quad_perm [1,0,3,2]
    fold(std::integral_constant<int, 0x4E>{}, every);   // quad_perm [2,3,0,1]
    fold(std::integral_constant<int, 0x141>{}, every);  // row_half_mirror
    if (lanes == 16) fold(std::integral_constant<int, 0x140>{}, every);  // row_mirror
  };
  fold_row(16);
  fold(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15 to the odd rows
  fold(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31 to the upper half: lane 63 has all
  if (lane == 63) ranges[wave] = u32x4_t{low, high, number, 0u};
  __syncthreads();
  const u32x4_t range = ranges[lane % WAVES];
  low = range[0];
  high = range[1];
  number = range[2];
  fold_row(WAVES);
  low = __builtin_amdgcn_readfirstlane(low);
  high = __builtin_amdgcn_readfirstlane(high);
  number = __builtin_amdgcn_readfirstlane(number);
  const int always = (int)(number >> 16), others = (int)(number & 0xffff);
  // what the wavefronts in front of this one have, and all of them
  auto over_waves = [&](const int* sums, uint32_t& all) {
    const int x = lane < WAVES ? sums[lane] : 0, upto = scan(x);
    all = (uint32_t)__builtin_amdgcn_readlane(upto, 63);
    return (uint32_t)__builtin_amdgcn_readlane(upto - x, wave);
  };
  uint32_t all;
  // ---- `from`: the least key that is taken; `rest` of the keys equal to it, where there are more
  int rest = a.count - always;
  uint32_t from = low;
  bool part = false;  // not all of the last keys are taken
  if (rest <= 0) {
    from = kAlways;
  } else if (others > rest) {
    uint32_t span = high - from;                   // keys from .. from + span are looked at
    int shift = max(0, 21 - __builtin_clz(span | 1u));
    for (;;) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (key[r] - from <= span) atomicAdd(&counts[(key[r] - from) >> shift], 1);
      __syncthreads();
      int c[EACH], here = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        c[e] = counts[BINS - 1 - EACH * tid - e];
        here += c[e];
      }
      int upto = scan(here);
      if (lane == 63) sums[wave] = upto;
      __syncthreads();
      upto += (int)over_waves(sums, all);
      if (upto - here < rest && rest <= upto) {
        int before = upto - here;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          if (before < rest && rest <= before + c[e]) {
            at_bin = BINS - 1 - EACH * tid - e;
            at_rest = rest - before;
            at_count = c[e];
          }
          before += c[e];
        }
      }
#pragma unroll
      for (int e = 0; e < EACH; ++e) counts[BINS - 1 - EACH * tid - e] = 0;
      __syncthreads();
      rest = at_rest;
      const uint32_t skipped = (uint32_t)at_bin << shift;
      from += skipped;
      span = min((1u << shift) - 1, span - skipped);
      part = at_count > rest;
      if (!part || shift == 0) break;
      shift = max(0, shift - 11);
    }
  }
  // ---- what is taken, in order: keys above `from`, and the first of those equal to it
  const uint32_t most = part ? rest : R * NT;
  uint32_t above = 0, equal = 0;  // of the lane's keys
#pragma unroll
  for (int r = 0; r < R; ++r) {
    above |= (uint32_t)(key[r] > from) << r;
    equal |= (uint32_t)(key[r] == from) << r;
  }
  const uint32_t mine = __popc(above) | __popc(equal) << 16;  // of a workgroup no more than 32768 together
  uint32_t before = scan((int)mine);
  if (lane == 63) placed[wave] = (int)before;
  __syncthreads();
  before += over_waves(placed, all) - mine;
  uint32_t ties = before >> 16, to = (before & 0xffff) + min(ties, most);
  for (uint32_t left = above | equal; left; left &= left - 1) {
    const int r = __builtin_ctz(left);
    const bool tie = equal >> r & 1;
    if ((!tie || ties < most) && to < (uint32_t)a.count) out[to++] = first + r;
    ties += tie;
  }
  for (int i = (int)((all & 0xffff) + min(all >> 16, most)) + tid; i < a.count; i += NT) out[i] = -1;
}

// The same for any number of pages, whose keys are read again and again: the last key that is taken is found from its upper bits down, by counting. Slow: most keys count in the same few
// places, and each 1024 pages wait four times in the last pass. 65536 pages, one list or eight, 138 us (their scores 12 and 67), 131072 248 and 271; 32768 pages by the kernel above 12.
constexpr int CHOOSERS = 1024;
__global__ __launch_bounds__(CHOOSERS) void select_choose_long_kernel(const SelectParams p) {
  const kvx_paged_select_args& a = p.a;
  const int b = blockIdx.y, pair = b * a.Hkv + blockIdx.x, n = p.pages(b), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int WAVES = CHOOSERS / 64, BINS = 2048;
  __shared__ int counts[BINS], sums[WAVES], at_bin, at_rest;
  const uint32_t* keys = p.keys + (int64_t)pair * p.stride;
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
  KVX_REQUIRE(items < (1 << 30), KVX_ERR_UNSUPPORTED, "kvx_paged_bounds: %d sequences of up to %d pages, %d KV heads in one call", a.B, most, p.Hkv);
  by_store(p, [&](auto d, auto kv) {
    auto go = [&](auto w) {
      constexpr int W = decltype(w)::value, NT = W == 16 ? 1024 : 256;
      constexpr int64_t each = NT / 64 / W;
      const int64_t blocks = min((items + each - 1) / each, (int64_t)(W == 16 ? 1 : 5) * num_cus());  // what registers leave room for
      hipLaunchKernelGGL((paged_bounds_kernel<decltype(d)::value, decltype(kv)::value, W>), dim3((unsigned)blocks), dim3(NT), 0, st, a, __builtin_ctz(p.page_size));
    };
    if (p.page_size <= 32) go(std::integral_constant<int, 1>{});
    else if (p.page_size <= 128) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 16>{});
  });
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

int keys_stride(const kvx_paged_select_args& a) { return (a.max_pages + 3) / 4 * 4; }
size_t paged_select_workspace(const kvx_paged_select_args& a) { return a.max_pages <= FEW ? 0 : (size_t)4 * a.B * a.Hkv * keys_stride(a); }

int launch_paged_select(const kvx_paged_select_args& a, hipStream_t st) {
  const SelectParams p = {a, (uint32_t*)a.workspace, keys_stride(a), __builtin_ctz(a.page_size), (int64_t)a.B * a.Hkv * a.max_pages <= (1 << 21)};
  const int64_t count = (int64_t)a.B * a.Hkv, units = count * ((a.max_pages + UNIT - 1) / UNIT);
  KVX_REQUIRE(count < (1 << 21) && units < (1 << 30), KVX_ERR_UNSUPPORTED, "kvx_paged_select: %d sequences of up to %d pages, %d KV heads in one call", a.B, a.max_pages,
              a.Hkv);
  const unsigned blocks = (unsigned)min(units, (int64_t)score_workgroups(a.D) * num_cus());
  const int group = a.Hq / a.Hkv;
  const bool few = a.max_pages <= FEW;
  const dim3 pairs(a.Hkv, a.B);
  auto go = [&](auto d, auto f16) {
    auto score = [&](auto heads) {
      constexpr int D = decltype(d)::value, HEADS = decltype(heads)::value;
      if (few) hipLaunchKernelGGL((select_few_kernel<D, decltype(f16)::value, HEADS>), pairs, dim3(4 * FEW), 0, st, p);
      else hipLaunchKernelGGL((select_score_kernel<D, decltype(f16)::value, HEADS>), dim3(blocks), dim3(NTHREADS), 0, st, p);
    };
    if (group <= 4) score(std::integral_constant<int, 1>{});
    else if (group <= 8) score(std::integral_constant<int, 2>{});
    else score(std::integral_constant<int, 4>{});
  };
  auto go_type = [&](auto d) {
    if (a.elem_dtype == KVX_KV_F16) go(d, std::true_type{});
    else go(d, std::false_type{});
  };
  if (a.D == 256) go_type(std::integral_constant<int, 256>{});
  else if (a.D == 128) go_type(std::integral_constant<int, 128>{});
  else go_type(std::integral_constant<int, 64>{});
  if (few) {
    KVX_HIP(hipGetLastError());
    return KVX_OK;
  }
  // 512 lanes take less time than 1024 up to 4096 pages and more beyond: 1024 pages 4.2 and 5.0 us (with more code in both), 4096 5.0 and 5.2, 8192 5.4 and 5.2, 48 ragged
  // lists of them 7.4 and 6.5
  auto choose = [&](auto r, auto nt) {
    constexpr int R = decltype(r)::value, NT = decltype(nt)::value;
    hipLaunchKernelGGL((select_choose_kernel<R, NT>), pairs, dim3(NT), 0, st, p);
  };
  const std::integral_constant<int, 512> half;
  const std::integral_constant<int, 1024> whole;
  if (a.max_pages <= 512) choose(std::integral_constant<int, 1>{}, half);
  else if (a.max_pages <= 1024) choose(std::integral_constant<int, 2>{}, half);
  else if (a.max_pages <= 2048) choose(std::integral_constant<int, 4>{}, half);
  else if (a.max_pages <= 4096) choose(std::integral_constant<int, 8>{}, half);
  else if (a.max_pages <= 8192) choose(std::integral_constant<int, 8>{}, whole);
  else if (a.max_pages <= 16384) choose(std::integral_constant<int, 16>{}, whole);
  else if (a.max_pages <= 32768) choose(std::integral_constant<int, 32>{}, whole);
  else hipLaunchKernelGGL(select_choose_long_kernel, pairs, dim3(CHOOSERS), 0, st, p);
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
