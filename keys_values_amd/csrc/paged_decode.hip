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
// Codes. (code - zp) * scale is linear in the code, so whole numbers are the operands, and scale and zero point are applied to a key's 16 logits and weights
// instead of its 2 D values. 16-bit integers below 1024 are what fp16 calls subnormal numbers, code * 2^-24, so one byte permute makes two operand values of
// 8-bit codes, and a mask and a shift those of 4-bit ones, 16 times theirs. Of V one multiply-add more for a pair takes the middle code c away and makes normal numbers.
//   logit = scale_k (S - zp_k sum q),        S = sum code q,      q in fp16 times a power of two that brings the head's largest below 2^15 (exact, but for what
//                                                                 is 2^28 times smaller than it: that is off by 2^-39 of it at most)
//   o     = (sum w (code - c) - sum w (zp_v - c)) / l,   w = p scale_v,       in units of a power of two above the largest scale_v so far
// w is rounded to fp16 for the first of these sums, which costs at most 2^-11 of a row's span / 2.
// What the matrix cores do (measured): eight products at a time, those of a lane group, are brought to the exponent of the largest and cut at 2^-24 of it; the
// four sums are added one after the other and rounded to nearest. A subnormal factor counts with the exponent of 2^-14, so that products of bare codes are cut at 2^-14
// of a code, always towards zero. In K's products that is less than what fp32 rounds (and of the lower halves of 4-bit codes it was not, before they were brought to 16
// times theirs). In V's it was a bias of up to half the rounding of fp16 outputs, and of all keys' sums the middle code had to be taken off again at the end:
// 16 heads of 64 over 3000 to 50000 keys, 4-bit, fp16: 2.20e-4 off in the mean, and 2.04e-4, which is the rounding of the outputs, with the middle code taken off before
// (16 sequences of 16384, 32 / 8 heads, 8-bit and 4-bit codes: rows of 64 +0 and 4 %, of 128 1 and 2 %, of 256 0 and 2 % longer).
//
// Bounds, 16 sequences of 16384 tokens, 32 / 8 heads: plain rows are at HBM (64 values 85 us, 128 158, 256 352: 6.3, 6.8, 6.1 TB/s), 8-bit rows of 128 nearly (91: 6.2). 8-bit
// rows of 64 (53.6: 5.6) and 4-bit ones (64 values 42, 128 55, 256 95: 4.0, 5.5, 6.0) have as much to do in the vector ALU as in memory: per 32 keys of 64 4-bit
// values some 230 vector instructions and 8 loads. Neither a third wavefront a SIMD nor a second block of keys in flight shortens them
// by more than 3 %. A call's fixed part is 5 us of serial loads (lengths, table, rows) and a join of 3 to 5, most of it the launch.
#include <type_traits>

#include "key_blocks.h"

namespace kvx {
namespace {

constexpr int NT = 256, WAVES = 4, UNIT = 128;  // keys of a step: a block of 32 a wavefront
constexpr float kLowest = -3.4028235e38f;       // running maximum before the first key
typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

// The first line is read first: what a workgroup's share follows from.
struct PagedParams {
  const int* lens;
  const int* table;
  int64_t table_sb;
  int B, Hkv, cap /* tokens of a table's pages */, unit /* log2 of the keys of a unit */, cus /* compute units */, workgroups, extra /* units added to a pair */, shift /* log2 of the page size */, max_pages;
  int num_pages, Gr /* query heads per KV head */;

  const uint16_t* q;
  int64_t q_sb, q_sh;
  const uint8_t *k, *v;
  const uint32_t *k_scale, *k_zp, *v_scale, *v_zp;
  uint32_t k_page, v_page, q_page, k_head, v_head, q_head, k_row, v_row;  // bytes from page to page, head to head, row to row of K, V and the quantiser's arrays
  float c;      // sm_scale * log2(e)
  int by_pair;  // part_of goes by pairs, which are fewer, else by workgroups

  uint16_t* o;
  int64_t o_sb, o_sh;
  float* lse;      // or NULL
  float* part_o;   // (2 workgroups, Gr, D)
  float* part_ml;  // (2 workgroups, Gr, 2): maximum and sum
  int* part_of;    // by pairs: the workgroup that left a pair's first partial; by workgroups: the pair; and how many partials the pair has, 0: none. NULL: no partials
};

// Units of a pair of `len` tokens: those with keys, and, behind them, as many without as the change to the pair takes the time of.
__device__ __forceinline__ int units_of(int len, const PagedParams& p, int extra) { return max(1, (min(max(len, 0), p.cap) + (1 << p.unit) - 1) >> p.unit) + extra; }

// Inclusive sum over the lanes of a wavefront, on the vector ALU.
__device__ __forceinline__ int scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to the odd rows
  return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to the upper half
}

// The shares of `total` units: workgroup w begins with unit first(w).
struct Shares {
  int workgroups, each, rest;
  __device__ __forceinline__ Shares(int total, int n) : workgroups(n), each(total / n), rest(total - each * n) {}
  __device__ __forceinline__ int first(int w) const { return min(w, workgroups) * each + min(w, rest); }
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
  // Short pieces of V rows are loaded twice as wide, by the lower eight lanes of a column group from a key and by the upper eight from the next one; then lanes
  // exchange. 4-bit rows of 64: 41.3 -> 39.2 us, of 128 53.5 -> 53.2, 8-bit rows of 64 53.5 -> 52.5 (as below); pieces of 8 bytes gain nothing (8-bit, 128: 89.6, 89.8).
  static constexpr bool PAIRED = CODES && VB <= 4;
  static constexpr int VN = PAIRED ? 4 : 8, VW = PAIRED ? VB / 2 : VB / 4;  // loads, and 32-bit words of one
  // state: lane l has the scale of key l (l < 32) or the zero point of key l - 32
  struct K {
    u32x4_t w[2][KR];
    uint32_t state;
  };
  struct V {
    uint32_t w[VN][VW];
    uint32_t state;
  };
  // What the matrix cores take from V: the words of both keys of a pair, and the bytes of them that a lane takes
  struct Pairs {
    uint32_t own[VN][VW], other[PAIRED ? VN : 1][VW], pick[2];
    __device__ __forceinline__ Pairs(const V& r, int m) {
#pragma unroll
      for (int j = 0; j < VN; ++j)
#pragma unroll
        for (int y = 0; y < VW; ++y) {
          own[j][y] = r.w[j][y];
          if constexpr (PAIRED) other[j][y] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)r.w[j][y], 0x128, 0xf, 0xf, true);  // row_ror:8
        }
      if constexpr (PAIRED) {
        pick[0] = m < 8 ? 0x0c040c00u : 0x0c020c06u;
        pick[1] = pick[0] + 0x00010001u;
      }
    }
  };
  // first d of the 8 that lane group kg supplies to matrix instruction e of the first product
  __device__ __forceinline__ static int kslice(int e, int kg) {
    if constexpr (!CODES) return 8 * (kg + 4 * e);
    else if constexpr (!U4) return 16 * kg + 8 * (e & 1) + 64 * (e >> 1);
    else if constexpr (D == 64) return 8 * kg + 32 * e;
    else return 64 * (e >> 2) + 16 * kg + 8 * ((e >> 1) & 1) + (D / 2) * (e & 1);
  }
  // 4-bit codes: instruction e takes those of the high halves of its bytes
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
      const uint32_t a = r.w[gi][x][2 * pair], b = r.w[gi][x][2 * pair + 1], mask = 0x00f000f0u;  // 16 times the codes
      if (high(e)) return u32x4_t{a & mask, (a >> 8) & mask, b & mask, (b >> 8) & mask};  // values 0, 2 | 1, 3 | 4, 6 | 5, 7
      return u32x4_t{(a << 4) & mask, (a >> 4) & mask, (b << 4) & mask, (b >> 4) & mask};
    }
  }
  // A operand t of the second product: value t of each of this lane's 8 keys, in key order. Of codes: (code - MID) * 2^-9, exact; of 4-bit ones the first half's are whole
  // bytes, 16 high + low: the lower halves' sums are taken off at the end, instead of the lower halves here.
  static constexpr float MID = U4 ? 8.0f : 128.0f;  // the middle code
  __device__ __forceinline__ static u32x4_t v_operand(const Pairs& r, int t) {
    u32x4_t a;
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const int j0 = 2 * jj, j1 = 2 * jj + 1, byte = U4 && t >= DPL / 2 ? t - DPL / 2 : t;
      if constexpr (!CODES) a[jj] = __builtin_amdgcn_perm(r.own[j1][t >> 1], r.own[j0][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
      else if constexpr (PAIRED) a[jj] = __builtin_amdgcn_perm(r.other[jj][byte >> 1], r.own[jj][byte >> 1], r.pick[byte & 1]);
      else a[jj] = __builtin_amdgcn_perm(r.own[j1][byte >> 2], r.own[j0][byte >> 2], 0x0c040c00u + 0x00010001u * (byte & 3));
      if constexpr (U4)
        if (t >= DPL / 2) a[jj] &= 0x000f000fu;
      if constexpr (CODES) {
        const uint32_t codes = a[jj];
        const _Float16 up = (_Float16)0x1p15f, mid = (_Float16)((U4 && t < DPL / 2 ? 17.0f * MID : MID) * -0x1p-9f);
        a[jj] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, codes), f16x2_t{up, up}, f16x2_t{mid, mid}));
      }
    }
    return a;
  }
  // d of row `mrow` of matrix instruction t of the second product
  __device__ __forceinline__ static int dmap(int t, int mrow) {
    const int u = U4 && t >= DPL / 2 ? t - DPL / 2 : t, first = U4 && t >= DPL / 2 ? D / 2 : 0;
    constexpr int EACH = U4 ? DPL / 2 : DPL;  // values of a row's piece, or bytes
    if constexpr (PAIRED) return first + 2 * EACH * (mrow & 7) + 4 * (u >> 1) + 2 * (mrow >> 3) + (u & 1);
    else return first + EACH * mrow + u;
  }
};

// What a block's keys are multiplied by and what is added to them, of a lane's keys: 4 kg + i of either tile. A lane loads the scale or the zero point of one key
// (lanes 0 - 31 and 32 - 63), makes of it what is wanted, and the keys' values change hands through LDS of the wavefront's own. Loaded as they are used, by 16 lanes each,
// they took as many cycles of the address units as 4-bit rows of 128, 32 registers on the way, and their conversions a third of the loop.
struct State {
  f32x4_t scale[2], zp[2];
  __device__ __forceinline__ State(float* lds, float mine, int lane, int kg) {
    lds[lane] = mine;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int gi = 0; gi < 2; ++gi) {
      scale[gi] = *(const f32x4_t*)(lds + 16 * gi + 4 * kg);
      zp[gi] = *(const f32x4_t*)(lds + 32 + 16 * gi + 4 * kg);
    }
    __builtin_amdgcn_wave_barrier();
  }
};

// Maximum over the wavefront, in every lane.
__device__ __forceinline__ float max_lanes(float x) {
  auto step = [](float v, auto ctrl) {
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  x = step(x, std::integral_constant<int, 0x128>{});  // row_ror:8
  x = step(x, std::integral_constant<int, 0x124>{});  // row_ror:4
  x = step(x, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  x = step(x, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  return max_halves(max_row_pairs(x));
}
// Sum over the four lane groups of a column.
__device__ __forceinline__ float sum_groups(float x) {
  const u32pair_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// What `pair`, packed from a and b, drops of them. In fp16: a multiply-add that reads the halves where they are, exact, as the difference is.
template <bool P16>
__device__ __forceinline__ uint32_t dropped(uint32_t pair, float a, float b) {
  if constexpr (P16) {
    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel_hi:[1,0,0]" : "+v"(a) : "v"(pair));
    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(b) : "v"(pair));
    return pack_pair<true>(a, b);
  } else {
    return pack_pair<false>(a - elem_lo<false>(pair), b - elem_hi<false>(pair));
  }
}

template <typename T>
__device__ __forceinline__ T once(const void* p) { return __builtin_nontemporal_load((const T*)p); }

// Wavefronts a SIMD that the registers have to leave room for. Plain rows of 256 values take more than half of them. Plain rows of 128 fit a third wavefront only if
// asked to, which short pairs gain from (256 sequences of 50 to 400 tokens, 32 / 8 heads: 49.1 us with two, 42.8 with three). No bound here spills.
constexpr int waves_per_simd(int D, bool codes) { return D == 256 && !codes ? 1 : D == 128 && !codes ? 3 : 2; }

template <int D, int KV>
__global__ __launch_bounds__(NT, waves_per_simd(D, !kv_is_plain(KV))) void paged_decode_kernel(const PagedParams p) {
  using R = Rows<D, KV>;
  constexpr bool F16 = R::F16, CODES = R::CODES, U4 = R::U4, P16 = F16 || CODES;  // P16: weights and operands in fp16
  constexpr int KJ = R::KJ, DPL = R::DPL, ES = R::ES;
  // The running maximum moves when a logit exceeds it by kTop. Weights in fp16 are kept below 2^15, and brought to 2^7 when it moves: what is a normal number
  // there goes down to 2^-21 of the largest then, and what is not zero to 2^-32.
  constexpr float kTop = P16 ? 15.0f : 8.0f, kBias = P16 ? 7.0f : 0.0f;
  // The part of a weight that its 16 bits drop is a second operand where outputs have as many bits: the rounding of weights would be as large as theirs. It is not
  // seen in the time (16 sequences of 16384, plain rows of 128: 157.9 and 158.1 us).
  constexpr bool FINE = F16 || !CODES;
  constexpr int RS = D + 4;  // floats of a head's row in LDS: heads in different banks
  __shared__ __align__(16) float red[WAVES][16][RS];
  __shared__ __align__(16) float state[WAVES][2][64];
  __shared__ float red_m[WAVES][16], red_l[WAVES][16];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, kg = lane >> 4;
  const int B = p.B, Hkv = p.Hkv, w = blockIdx.x, mask = (1 << p.shift) - 1, extra = CODES ? p.extra : 0;

  // ---- this workgroup's units: every wavefront finds them for itself, 64 sequences at a time
  const int windows = (B + 63) / 64;
  auto window = [&](int i) { return 64 * i + lane < B ? p.lens[64 * i + lane] : -1; };
  auto units_in = [&](int len, int i) { return 64 * i + lane < B ? units_of(len, p, extra) : 0; };
  int lane_len = 0, mine = 0;  // lane_len: of sequence (b & ~63) + lane
  for (int i = 0; i < windows; ++i) {
    lane_len = window(i);
    mine += units_in(lane_len, i);
  }
  const int total = __builtin_amdgcn_readlane(scan(mine), 63) * Hkv;
  // Workgroups that share the units, of the grid's two or three a compute unit: all where pairs are short (of up to four units on average; B256, 32 / 8 heads of 128, 50 to 400
  // tokens: 42.7 us, 44.4 with two a compute unit, 54.2 with one), two elsewhere (64 sequences of 1 to 8192, 28 / 4 heads: 30.9, 33.3 with one, 32.1 with three), and
  // one, whose partials are the fewest, where pairs are long and rows of 128 bytes and more keep enough of them on their way (16 x 16384, plain rows of 128: 158.3, 162.0
  // with two, 165.6 with three; but 4-bit rows of 128: 65.7, 53.7 with two).
  constexpr bool WIDE = D * ES >= (U4 ? 256 : 128);
  const int pairs = B * Hkv, full = total - pairs * extra, sharing = (full + 3) / 4 <= pairs ? p.workgroups : WIDE && full / 64 >= pairs ? p.cus : 2 * p.cus;
  const Shares shares(total, min(sharing, p.workgroups));
  int unit = shares.first(w);  // the next unit
  const int end = shares.first(w + 1);
  if (tid == 0 && p.part_of && !p.by_pair) p.part_of[2 * w + 1] = 0;
  if (unit >= end) return;
  int b, begin_b;  // its sequence, and the sequence's first unit
  for (int i = 0, before = 0;; ++i) {
    if (windows > 1) lane_len = window(i);
    mine = units_in(lane_len, i);
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

  // A stretch of a pair's units. The next one's first rows are on their way while this one's results are joined.
  struct Stretch {
    int b, h, begin, units, first, n, k_begin, k_end;
  };
  auto go_to = [&](int to, int units) {  // to a unit of the same pair, or the next one's first
    unit = to;
    if (unit == begin_b + units * Hkv) {
      begin_b = unit;
      ++b;
      if ((b & 63) == 0 && b < B) lane_len = window(b >> 6);
    }
  };
  if constexpr (CODES) {  // a share does not begin with units without keys
    const int units = units_of(__builtin_amdgcn_readlane(lane_len, b & 63), p, extra), left = units - (unit - begin_b) % units;
    if (left <= extra) go_to(unit + left, units);
    if (unit >= end) return;
  }
  auto take = [&] {
    Stretch s;
    const int len = min(max(__builtin_amdgcn_readlane(lane_len, b & 63), 0), p.cap);
    s.b = b;
    s.units = units_of(len, p, extra);
    s.h = (unit - begin_b) / s.units;
    s.begin = begin_b + s.h * s.units;
    s.first = unit - s.begin;
    s.n = min(s.units - s.first, end - unit);
    s.k_begin = s.first << p.unit;
    s.k_end = min(len, (s.first + s.n) << p.unit);
    go_to(unit + s.n, s.units);
    return s;
  };

  const uint32_t k_lane = (uint32_t)m * p.k_row + (U4 && D == 64 ? 8 : 16) * kg, v_lane = R::PAIRED ? (4 * kg + (m >> 3)) * p.v_row + (m & 7) * 2 * R::VB : 4 * kg * p.v_row + m * R::VB;

  // ---- rows of a block of 32 keys. Lane 2 j + gi holds the page of half gi of the wavefront's block j (of 32 at a time). A page that the pool does not have is
  // read as page 0, and its keys are masked behind. Keys behind the end lie in the same pages, or masked ones.
  struct Tiles {
    int page0, page1;  // no arrays: a lane that picks one of them would send them through memory
    bool ok0, ok1;
    __device__ __forceinline__ int page(bool upper) const {
      const int a = page0, b = page1;
      return upper ? b : a;
    }
    __device__ __forceinline__ bool ok(bool upper) const {
      const bool a = ok0, b = ok1;
      return upper ? b : a;
    }
  };
  Stretch at;       // the stretch whose rows are read
  int lane_page;
  const uint8_t *k_head, *v_head;
  const char *k_state, *v_state;
  auto pages_of = [&](const Stretch& s, int j) {
    return p.table[s.b * p.table_sb + min((s.k_begin + 32 * wave + (j + (lane >> 1)) * UNIT + 16 * (lane & 1)) >> p.shift, p.max_pages - 1)];
  };
  auto tiles = [&](int j) {
    if (j > 0 && (j & 31) == 0) {
      lane_page = pages_of(at, j);
      asm volatile("" : "+v"(lane_page));  // waited for here, not in every pass
    }
    Tiles t;
    const int page0 = __builtin_amdgcn_readlane(lane_page, 2 * (j & 31)), page1 = __builtin_amdgcn_readlane(lane_page, 2 * (j & 31) + 1);
    t.ok0 = (uint32_t)page0 < (uint32_t)p.num_pages;
    t.ok1 = (uint32_t)page1 < (uint32_t)p.num_pages;
    t.page0 = t.ok0 ? page0 : 0;
    t.page1 = t.ok1 ? page1 : 0;
    return t;
  };
  auto load_state = [&](const char* base, int chunk, const Tiles& t) {
    const uint32_t page = t.page(lane & 16), place = (chunk + (lane & 16)) & mask;
    return once<uint32_t>(base + ((uint64_t)page * p.q_page + place * 4u));
  };
  auto load_k = [&](typename R::K& r, int chunk, const Tiles& t) {
#pragma unroll
    for (int gi = 0; gi < 2; ++gi) {
      const uint8_t* base = k_head + (uint64_t)(uint32_t)t.page(gi) * p.k_page;
      const uint32_t off = (uint32_t)((chunk + 16 * gi) & mask) * p.k_row + k_lane;
#pragma unroll
      for (int x = 0; x < R::KR; ++x) {
        if constexpr (U4 && D == 64) {
          const u32x2_t y = once<u32x2_t>(base + off);
          r.w[gi][x] = u32x4_t{y[0], y[1], 0u, 0u};
        } else {
          r.w[gi][x] = once<u32x4_t>(base + off + 64 * x);
        }
      }
    }
    if constexpr (CODES) r.state = load_state(k_state, chunk, t);
  };
  auto load_v = [&](typename R::V& r, int chunk, const Tiles& t) {
    if constexpr (CODES) r.state = load_state(v_state, chunk, t);
#pragma unroll
    for (int gi = 0; gi < 2; ++gi) {
      const uint8_t* base = v_head + (uint64_t)(uint32_t)t.page(gi) * p.v_page;
      const uint32_t off = (uint32_t)((chunk + 16 * gi) & mask) * p.v_row + v_lane;
#pragma unroll
      for (int i = 0; i < R::VN / 2; ++i) {
        const uint8_t* row = base + (off + (uint32_t)(8 / R::VN * i) * p.v_row);
        uint32_t(&x)[R::VW] = r.w[R::VN / 2 * gi + i];
        if constexpr (R::VW >= 4) {
#pragma unroll
          for (int y = 0; y < R::VW / 4; ++y) {
            const u32x4_t z = once<u32x4_t>(row + 16 * y);
            x[4 * y] = z[0]; x[4 * y + 1] = z[1]; x[4 * y + 2] = z[2]; x[4 * y + 3] = z[3];
          }
        } else if constexpr (R::VW == 2) {
          const u32x2_t z = once<u32x2_t>(row);
          x[0] = z[0]; x[1] = z[1];
        } else {
          x[0] = once<uint32_t>(row);
        }
      }
    }
  };
  // Queries, B operands of the first product: head m
  auto load_q = [&](u32x4_t (&q)[KJ], const Stretch& s) {
    const uint16_t* row = p.q + s.b * p.q_sb + (int64_t)(s.h * p.Gr + min(m, p.Gr - 1)) * p.q_sh;
#pragma unroll
    for (int e = 0; e < KJ; ++e) q[e] = *(const u32x4_t*)(row + R::kslice(e, kg));
  };
  typename R::K k;
  typename R::V v;
  u32x4_t qb[KJ];
  Tiles t;
  auto start = [&](const Stretch& s, int page) {
    at = s;
    lane_page = page;
    k_head = p.k + (uint64_t)(uint32_t)s.h * p.k_head;
    v_head = p.v + (uint64_t)(uint32_t)s.h * p.v_head;
    if constexpr (CODES) {
      const uint64_t q = (uint64_t)(uint32_t)s.h * p.q_head + 4 * m;
      k_state = (const char*)(lane < 32 ? p.k_scale : p.k_zp) + q;
      v_state = (const char*)(lane < 32 ? p.v_scale : p.v_zp) + q;
    }
    t = tiles(0);
    load_q(qb, s);
    const int chunk = s.k_begin + 32 * wave;
    if (chunk < s.k_end) {
      load_k(k, chunk, t);
      load_v(v, chunk, t);
    }
  };
  {
    const Stretch s = take();
    start(s, pages_of(s, 0));
  }

  for (bool again = false;; again = true) {
    const Stretch now = at;
    const bool more = unit < end;
    Stretch next = now;
    int next_page = 0;
    if (more) {
      next = take();
      next_page = pages_of(next, 0);
    }

    constexpr float kFromOperand = U4 ? 0x1p20f : 0x1p24f;  // K's codes over the operands that they are
    float qsum = 0.0f, to_logit = 1.0f;  // to_logit: a power of two, of the head's, so that products with it are exact
    // Columns beyond the group are zeros: with copies of the last head there the matrix cores are slower (16 x 16384, 32 / 8 heads of 64, plain: 84.5 us, 90.5)
#pragma unroll
    for (int e = 0; e < KJ; ++e)
      if (m >= p.Gr) qb[e] = u32x4_t{0u, 0u, 0u, 0u};
    if constexpr (CODES) {
      auto largest = [&](bool finite) {  // of the head's values: heads of a group may differ by more than fp16 spans
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < KJ; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x0 = fabsf(elem_lo<F16>(qb[e][i])), x1 = fabsf(elem_hi<F16>(qb[e][i]));
            top = fmaxf(top, finite && !(x0 < INFINITY) ? 0.0f : x0);
            top = fmaxf(top, finite && !(x1 < INFINITY) ? 0.0f : x1);
          }
        return max_halves(max_row_pairs(top));
      };
      float top = largest(false);
      if (__any(!(top < INFINITY))) top = largest(true);
      // 2^x that brings it to [2^14, 2^15)
      const int ex = (int)(__float_as_uint(top) >> 23), up = ex == 0 ? 127 : min(268 - ex, 253);
      const float by = __uint_as_float((uint32_t)up << 23);
      to_logit = __uint_as_float((uint32_t)(254 - up) << 23);
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
          qb[e] = u32x4_t{pack_pair<true>(x[0], x[2]), pack_pair<true>(x[1], x[3]), pack_pair<true>(x[4], x[6]), pack_pair<true>(x[5], x[7])};
        } else {
          qb[e] = u32x4_t{pack_pair<true>(x[0], x[1]), pack_pair<true>(x[2], x[3]), pack_pair<true>(x[4], x[5]), pack_pair<true>(x[6], x[7])};
        }
      }
      qsum = -sum_groups(qsum) / kFromOperand;
    }

    f32x4_t acc[DPL];
#pragma unroll
    for (int t = 0; t < DPL; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kLowest, l_run = 0.0f;
    // codes: sum of w (zp - c), the unit of the scales, and its inverse
    float corr = 0.0f, unit_v = 0x1p-126f, per_v = 0x1p126f;

    auto whole = [&](int chunk) { return chunk + 32 <= now.k_end && t.ok0 && t.ok1; };
    // key `i` of half gi is one of the sequence's
    auto live = [&](int chunk, int gi, int i) { return t.ok(gi) && chunk + 16 * gi + i < now.k_end; };
    // logits: head m, keys 4 kg + i of the two halves; in log2 units, of codes by to_logit, which is the head's
    auto logits = [&](int chunk, float (&s)[8]) {
      f32x4_t x[2];
#pragma unroll
      for (int gi = 0; gi < 2; ++gi) {
        x[gi] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < KJ; ++e) x[gi] = mfma_16x16x32<P16>(R::k_operand(k, gi, e), qb[e], x[gi]);
      }
      if constexpr (CODES) {
        const State st(state[wave][0], lane < 32 ? __uint_as_float(k.state) * (p.c * kFromOperand) : (float)(int32_t)k.state, lane, kg);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = fmaf(st.zp[i >> 2][i & 3], qsum, x[i >> 2][i & 3]) * st.scale[i >> 2][i & 3];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = x[i >> 2][i & 3] * p.c;
      }
      if (!whole(chunk)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!live(chunk, i >> 2, 4 * kg + (i & 3))) s[i] = -INFINITY;
      }
    };
    auto weights = [&](float (&s)[8]) {
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
      if constexpr (CODES) top *= to_logit;
      if (__any(top > m_run + kTop)) {
        top = max_halves(max_row_pairs(top));  // of the head, over the four lane groups
        const bool moves = top > m_run + kTop;
        const float to = moves ? top - kBias : m_run, al = moves ? fast_exp2(m_run - to) : 1.0f;
        m_run = to;
        l_run *= al;
        if constexpr (CODES) corr *= al;
#pragma unroll
        for (int t = 0; t < DPL; ++t) acc[t] *= al;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] = fast_exp2(CODES ? fmaf(s[i], to_logit, -m_run) : s[i] - m_run);
        l_run += s[i];
      }
    };
    auto outputs = [&](int chunk, float (&s)[8]) {
      const bool masked = !whole(chunk);  // what lies in masked places may be infinite or NaN
      if constexpr (!CODES)
        if (masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!live(chunk, i >> 2, 4 * kg + (i & 3))) {
#pragma unroll
              for (int y = 0; y < R::VW; ++y) v.w[i][y] = 0u;
            }
        }
      if constexpr (CODES) {
        float mine = lane < 32 ? __uint_as_float(v.state) : (float)(int32_t)v.state - R::MID;
        if (masked && !live(chunk, (lane >> 4) & 1, m)) mine = 0.0f;
        const float scale = lane < 32 ? fabsf(mine) : 0.0f;
        if (__any(scale > unit_v)) {
          const int ex = min((int)(__float_as_uint(max_lanes(scale)) >> 23) + 1, 253);
          const float per = __uint_as_float((uint32_t)(254 - ex) << 23), al = unit_v * per;
          unit_v = __uint_as_float((uint32_t)ex << 23);
          per_v = per;
          corr *= al;
#pragma unroll
          for (int t = 0; t < DPL; ++t) acc[t] *= al;
        }
        const State st(state[wave][1], lane < 32 ? mine * per_v : mine, lane, kg);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[i] *= st.scale[i >> 2][i & 3];
          corr = fmaf(s[i], st.zp[i >> 2][i & 3], corr);
        }
      }
      const u32x4_t pb = {pack_pair<P16>(s[0], s[1]), pack_pair<P16>(s[2], s[3]), pack_pair<P16>(s[4], s[5]), pack_pair<P16>(s[6], s[7])};
      const typename R::Pairs rows(v, m);
      if constexpr (FINE) {
        u32x4_t pl;
#pragma unroll
        for (int i = 0; i < 4; ++i) pl[i] = dropped<P16>(pb[i], s[2 * i], s[2 * i + 1]);
#pragma unroll
        for (int t = 0; t < DPL; ++t) {
          const u32x4_t x = R::v_operand(rows, t);
          acc[t] = mfma_16x16x32<P16>(x, pl, mfma_16x16x32<P16>(x, pb, acc[t]));
        }
      } else {
#pragma unroll
        for (int t = 0; t < DPL; ++t) acc[t] = mfma_16x16x32<P16>(R::v_operand(rows, t), pb, acc[t]);
      }
    };

    int chunk = now.k_begin + 32 * wave;
    if (chunk < now.k_end) {
      float s[8];
      for (int j = 1; chunk + UNIT < now.k_end; ++j) {
        const Tiles then = tiles(j);
        logits(chunk, s);
        __builtin_amdgcn_sched_barrier(0);  // the loads below reuse the registers consumed above
        load_k(k, chunk + UNIT, then);
        __builtin_amdgcn_sched_barrier(0);
        weights(s);
        outputs(chunk, s);
        __builtin_amdgcn_sched_barrier(0);
        load_v(v, chunk + UNIT, then);
        __builtin_amdgcn_sched_barrier(0);
        t = then;
        chunk += UNIT;
      }
      logits(chunk, s);
      weights(s);
      outputs(chunk, s);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) start(next, next_page);
    __builtin_amdgcn_sched_barrier(0);

    // ---- the four wavefronts' results, joined
    const float l = sum_groups(l_run);
    if constexpr (CODES) {
      corr = sum_groups(corr);
#pragma unroll
      for (int t = 0; t < DPL; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (U4 && t < DPL / 2) acc[t][i] = ((acc[t][i] - acc[t + DPL / 2][i]) * 0x1p5f - corr) * unit_v;
          else acc[t][i] = (acc[t][i] * 0x1p9f - corr) * unit_v;
        }
    }
    if (again) __syncthreads();  // the results before are read
    if (m < p.Gr) {
      constexpr int RUN = R::PAIRED ? 2 : 4;  // values side by side
      typedef float run_t __attribute__((ext_vector_type(RUN)));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < DPL; t += RUN) {
          run_t x;
#pragma unroll
          for (int e = 0; e < RUN; ++e) x[e] = acc[t + e][i];
          *(run_t*)&red[wave][m][R::dmap(t, 4 * kg + i)] = x;
        }
      if (kg == 0) {
        red_m[wave][m] = m_run;
        red_l[wave][m] = l;
      }
    }
    __syncthreads();
    const bool alone = now.first == 0 && now.n >= now.units - extra;  // the pair is this workgroup's alone
    const int slot = 2 * w + (now.first == 0 ? 1 : 0);
    auto sums = [&](int g, float (&f)[WAVES], float& top) {
      top = red_m[0][g];
#pragma unroll
      for (int j = 1; j < WAVES; ++j) top = fmaxf(top, red_m[j][g]);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < WAVES; ++j) {
        f[j] = fast_exp2(red_m[j][g] - top);
        sum += red_l[j][g] * f[j];
      }
      return sum;
    };
    // Infinite values of plain rows make the output infinite, whatever the key's weight, which is positive. Products with a weight that is 0 in 16 bits, or with what the 16
    // bits drop of it (0, or negative), do not: outputs that are NaN get the sum of the infinities and NaNs among their values, if there are any. (Looked for in a second
    // pass over the results, which leaves the registers of the first as they are: 64 sequences of 1 to 8192, 28 / 4 heads of 128, 31.4 us before, 31.5, 31.9 in one pass.
    // It reads V again, a key after the other: 8 sequences of 131072 with a NaN or an infinity in one of them 15 ms, 0.6 without.)
    auto unbounded = [&](f32x4_t& x, int d) {
      f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma clang loop unroll(disable)
      for (int key = now.k_begin; key < now.k_end; ++key) {
        const int page = p.table[now.b * p.table_sb + (key >> p.shift)];
        if ((uint32_t)page >= (uint32_t)p.num_pages) continue;
        const uint8_t* row = p.v + (uint64_t)(uint32_t)now.h * p.v_head + (uint64_t)(uint32_t)page * p.v_page + (uint32_t)(key & mask) * p.v_row;
        const u32x2_t pairs = *(const u32x2_t*)(row + 2 * d);
        const f32x4_t value = {elem_lo<F16>(pairs[0]), elem_hi<F16>(pairs[0]), elem_lo<F16>(pairs[1]), elem_hi<F16>(pairs[1])};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(fabsf(value[e]) < INFINITY)) sum[e] += value[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x[e] != x[e] && sum[e] != 0.0f) x[e] = sum[e];
    };
    bool odd = false;  // some output is NaN though the weights are not
    auto results = [&](auto second) {
      for (int i = tid; i < p.Gr * (D / 4); i += NT) {
        const int g = i / (D / 4), d = 4 * (i % (D / 4));
        float f[WAVES], top;
        const float sum = sums(g, f, top);
        f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < WAVES; ++j) x += *(const f32x4_t*)&red[j][g][d] * f[j];
        if constexpr (!CODES) {
          const float all = x[0] + x[1] + x[2] + x[3];
          const bool nan = all != all && sum == sum;
          if constexpr (decltype(second)::value) {
            if (nan) unbounded(x, d);
          } else {
            odd |= nan;
          }
        }
        if (alone) {
          x *= sum == 0.0f ? 0.0f : 1.0f / sum;
          *(u32x2_t*)(p.o + now.b * p.o_sb + (int64_t)(now.h * p.Gr + g) * p.o_sh + d) = u32x2_t{pack_pair<F16>(x[0], x[1]), pack_pair<F16>(x[2], x[3])};
          if (d == 0 && p.lse) p.lse[((int64_t)now.b * Hkv + now.h) * p.Gr + g] = sum == 0.0f ? -INFINITY : top + fast_log2(sum);
        } else {
          *(f32x4_t*)(p.part_o + ((int64_t)slot * p.Gr + g) * D + d) = x;
          if (d == 0) *(f32x2_t*)(p.part_ml + ((int64_t)slot * p.Gr + g) * 2) = f32x2_t{top, sum};
        }
      }
    };
    results(std::false_type{});
    if constexpr (!CODES)
      if (__builtin_expect(__any(odd), 0)) results(std::true_type{});
    if (tid == 0 && p.part_of && now.first == 0 && (p.by_pair || !alone)) {
      const int pair = now.b * Hkv + now.h, i = 2 * (p.by_pair ? pair : w);
      p.part_of[i] = p.by_pair ? w : pair;
      p.part_of[i + 1] = alone ? 0 : shares.owner(now.begin + now.units - extra - 1) - w + 1;
    }
    if (!more) break;
  }
}

// The partials of a pair, joined: 4 LANES of its outputs a workgroup, four a lane; NT / LANES groups of lanes share the partials.
template <int D, bool F16, int LANES>
__global__ __launch_bounds__(NT) void paged_join_kernel(const PagedParams p) {
  constexpr int GROUPS = NT / LANES, U = 8;  // partials of a group in flight
  const int at = p.part_of[2 * blockIdx.x], n = p.part_of[2 * blockIdx.x + 1];
  if (n == 0) return;
  __shared__ __align__(16) float red[GROUPS][LANES][4];
  __shared__ float red_m[GROUPS][LANES], red_l[GROUPS][LANES];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, i = blockIdx.y * 4 * LANES + 4 * lane, g = min(i / D, p.Gr - 1), d = i % D;
  const int w = p.by_pair ? at : blockIdx.x, pair = p.by_pair ? blockIdx.x : at, b = pair / p.Hkv, h = pair - b * p.Hkv;
  float top = kLowest, sum = 0.0f;
  f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = group; s0 < n; s0 += GROUPS * U) {
    f32x2_t ml[U];
    f32x4_t y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + GROUPS * u, n - 1);
      const int64_t slot = s == 0 ? 2 * w + 1 : 2 * (w + s);
      ml[u] = *(const f32x2_t*)(p.part_ml + (slot * p.Gr + g) * 2);
      y[u] = *(const f32x4_t*)(p.part_o + (slot * p.Gr + g) * D + d);
    }
    float to = top;
#pragma unroll
    for (int u = 0; u < U; ++u) to = fmaxf(to, ml[u][0]);
    const float al = fmaxf(fast_exp2(top - to), 0x1p-126f);  // factors are positive: infinite outputs stay infinite
    sum *= al;
    x *= al;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + GROUPS * u >= n) break;
      const float be = fmaxf(fast_exp2(ml[u][0] - to), 0x1p-126f);
      sum += ml[u][1] * be;
      x += y[u] * be;
    }
    top = to;
  }
  *(f32x4_t*)red[group][lane] = x;
  red_m[group][lane] = top;
  red_l[group][lane] = sum;
  __syncthreads();
  if (group != 0 || i >= p.Gr * D) return;
  float all = red_m[0][lane];
#pragma unroll
  for (int j = 1; j < GROUPS; ++j) all = fmaxf(all, red_m[j][lane]);
  sum = 0.0f;
  x = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const float f = fmaxf(fast_exp2(red_m[j][lane] - all), 0x1p-126f);
    sum += red_l[j][lane] * f;
    x += *(const f32x4_t*)red[j][lane] * f;
  }
  x *= sum == 0.0f ? 0.0f : 1.0f / sum;
  *(u32x2_t*)(p.o + b * p.o_sb + (int64_t)(h * p.Gr + g) * p.o_sh + d) = u32x2_t{pack_pair<F16>(x[0], x[1]), pack_pair<F16>(x[2], x[3])};
  if (p.lse && d == 0) p.lse[(int64_t)pair * p.Gr + g] = sum == 0.0f ? -INFINITY : all + fast_log2(sum);
}

PagedParams params_of(const kvx_paged_decode_args& a) {
  const kvx_pages& g = a.pages;
  const bool plain = kv_is_plain(g.kv_dtype);
  const int es = plain ? 2 : 1;
  PagedParams p{};
  p.lens = a.lens;
  p.table = a.block_table;
  p.table_sb = a.bt_stride_b;
  p.B = a.B;
  p.Hkv = g.Hkv;
  p.shift = __builtin_ctz(g.page_size);
  p.max_pages = a.max_pages;
  p.cap = a.max_pages << p.shift;
  p.num_pages = g.num_pages;
  p.Gr = a.Hq / g.Hkv;
  p.q = (const uint16_t*)a.q;
  p.q_sb = a.q_stride_b;
  p.q_sh = a.q_stride_h;
  p.k = (const uint8_t*)g.k;
  p.v = (const uint8_t*)g.v;
  p.k_scale = (const uint32_t*)g.k_scale;
  p.k_zp = (const uint32_t*)g.k_zp;
  p.v_scale = (const uint32_t*)g.v_scale;
  p.v_zp = (const uint32_t*)g.v_zp;
  p.k_page = (uint32_t)(g.k_stride_page * es);
  p.v_page = (uint32_t)(g.v_stride_page * es);
  p.k_head = (uint32_t)(g.k_stride_h * es);
  p.v_head = (uint32_t)(g.v_stride_h * es);
  p.k_row = (uint32_t)(g.k_stride_t * es);
  p.v_row = (uint32_t)(g.v_stride_t * es);
  if (!plain) {
    p.q_page = (uint32_t)(g.qs_stride_page * 4);
    p.q_head = (uint32_t)(g.qs_stride_h * 4);
  }
  p.c = a.sm_scale * kLog2e;
  p.o = (uint16_t*)a.o;
  p.o_sb = a.o_stride_b;
  p.o_sh = a.o_stride_h;
  p.lse = a.lse;
  // Tables of up to 512 tokens: a pair is a workgroup's, and there is no second launch.
  p.unit = p.cap <= 4 * UNIT ? 9 : 7;
  // Beginning a pair of codes takes the time of one unit of 8-bit rows, or two of 4-bit ones: it counts as such, or the workgroups that get the short pairs come last. 92
  // sequences of lengths even in the logarithm from 15 to 9560, 4-bit rows of 128, 32 / 4 heads: 40.8 us without, 29.6 with one unit, 26.2 with two; 14 from 25 to 35609, 8-bit
  // rows of 256: 76.8 without, 63.1 with one or two. Plain rows, whose units take longer, only lose: 200 of 1 to 3000, 65.8 without, 68.5 with one.
  p.extra = plain || p.unit == 9 ? 0 : kv_is_u4(g.kv_dtype) ? 2 : 1;
  p.cus = num_cus();
  // One workgroup a compute unit for the only pair: the partials of more take longer to join than they save (one of 100000 tokens, 16 heads of 128: 21.7 us, 33.8
  // with three).
  // More of them than registers leave room for would come in a second round: 239 sequences of 1 to 641, 24 / 8 heads of 128, 8-bit: 28.7, 35.7 with three.
  const int64_t per_cu = g.D == 256 ? waves_per_simd(256, !plain) : g.D == 128 && !plain && !kv_is_u4(g.kv_dtype) ? 2 : 3;
  const int64_t pairs = (int64_t)a.B * a.pages.Hkv, units = pairs * ((p.cap + (1 << p.unit) - 1) >> p.unit), most = p.cus * (pairs < per_cu ? pairs : per_cu);
  p.workgroups = (int)(units < most ? units : most);
  p.by_pair = pairs <= p.workgroups;
  return p;
}
bool splits(const PagedParams& p) { return p.cap > (1 << p.unit); }

template <int D>
void launch_head(const PagedParams& p, int kv_dtype, hipStream_t st) {
  switch (kv_dtype) {
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
  const unsigned rows = p.by_pair ? (unsigned)(p.B * p.Hkv) : (unsigned)p.workgroups;
  auto join = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    const dim3 grid(rows, (p.Gr * D + 4 * LANES - 1) / (4 * LANES));
    if (kv_elem_f16(kv_dtype)) hipLaunchKernelGGL((paged_join_kernel<D, true, LANES>), grid, dim3(NT), 0, st, p);
    else hipLaunchKernelGGL((paged_join_kernel<D, false, LANES>), grid, dim3(NT), 0, st, p);
  };
  if (rows <= 64) join(std::integral_constant<int, 16>{});
  else join(std::integral_constant<int, 64>{});
}

size_t part_floats(const PagedParams& p, int D) { return (size_t)2 * p.workgroups * p.Gr * D; }

}  // namespace

size_t paged_decode_workspace(const kvx_paged_decode_args& a) {
  const PagedParams p = params_of(a);
  return splits(p) ? 4 * (part_floats(p, a.pages.D) + (size_t)4 * p.workgroups * p.Gr + 2 * p.workgroups) : 0;
}

int launch_paged_decode(const kvx_paged_decode_args& a, hipStream_t st) {
  PagedParams p = params_of(a);
  if (splits(p)) {
    p.part_o = (float*)a.workspace;
    p.part_ml = p.part_o + part_floats(p, a.pages.D);
    p.part_of = (int*)(p.part_ml + (size_t)4 * p.workgroups * p.Gr);
  }
  if (a.pages.D == 256) launch_head<256>(p, a.pages.kv_dtype, st);
  else if (a.pages.D == 128) launch_head<128>(p, a.pages.kv_dtype, st);
  else launch_head<64>(p, a.pages.kv_dtype, st);
  KVX_HIP(hipGetLastError());
  return KVX_OK;
}

}  // namespace kvx
