// mk_product.h — one tiled bf16 product for three operand orders, with what
// follows it in the epilogue (gfx950):
//   C[m, n] = sum_k A(m, k) B(k, n),  then the epilogue
// An operand is k-contiguous ("KC": A[m * lda + k], B[n * ldb + k]) or k-strided
// ("KS": A[k * lda + m], B[k * ldb + n]).  Forward products are KC x KS, gradients
// of the left operand KC x KC (the weights as they are stored), gradients of the
// right operand KS x KS: nothing is transposed in memory.
//
// Any M, N and K.  Rows are 16-byte aligned, and a KC operand's rows end with a
// 16-byte unit or zeros up to one (mk_capi lays other operands out anew); the
// last K stage of a KC operand asks for no unit behind K, and buffer descriptors
// end at the last valid row, so that what lies behind an operand is read as zeros:
// the zeros of one operand meet zeros of the other, never what a neighbour holds.
//
// Groups (experts): with `counts`, group e owns counts[e] rows behind those of the
// groups before it, of A and C (ragged 1, tiles of rows) or of A and B (ragged 2,
// the sum's length, C of every group whole).  Counts are read on the device; each
// workgroup finds its tile by a scan of them.
//
// A tile's K may be cut into parts, a workgroup each.  Each part writes its fp32
// sums, then takes a ticket; the last to come adds all parts in K order and runs
// the epilogue, so no workgroup waits for another and results do not depend on
// which came last.
//
// Epilogue: each 32-row block of a wave's sums goes through the wave's own LDS
// rows in fp32 and comes back as 8 neighbouring columns a lane, so that every
// load and store of the epilogue covers whole row segments.
#pragma once
#include <type_traits>

#include "mk_device.h"
#include "mk_internal.h"
#include "mk_once.h"
#include "mk_tile.h"

namespace mk {

template <int BM_, int BN_, int WM_, int WN_, int BK_, int S_, bool PP_ = false>
struct PCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, S = S_;
  static constexpr bool PP = PP_;  // two wave groups take turns at the matrix cores
  static constexpr int WAVES = WM * WN, NT = 64 * WAVES;
  static constexpr int WTM = BM / WM, WTN = BN / WN, FM = WTM / 32, FN = WTN / 32;
  static constexpr int KSTEPS = BK / 16;
  static constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int A_INST = A_BYTES / 1024 / WAVES, B_INST = B_BYTES / 1024 / WAVES, LOADS = A_INST + B_INST;
  static constexpr int PITCH = WTN * 4 + 16;  // bytes of an epilogue row
  static constexpr uint32_t EPI_BYTES = WAVES * 32 * PITCH;
  static constexpr uint32_t STATS_BYTES = WN * BM * 8 + BM * 16;  // behind them, of the vocabulary's epilogues
  static constexpr uint32_t LDS_BYTES = S * STAGE > EPI_BYTES + STATS_BYTES ? S * STAGE : EPI_BYTES + STATS_BYTES;
  static constexpr int PER_CU = 160 * 1024 / LDS_BYTES;
  static constexpr int WAVES_PER_SIMD = PER_CU * WAVES / 4 > 0 ? PER_CU * WAVES / 4 : 1;
  static constexpr int UNITS = FM * FN * 4;  // 16-byte units of sums per thread
  // operands of the next stage in registers too, where there are as many
  static constexpr int AHEAD = !PP && WAVES_PER_SIMD <= 2 ? 1 : 0;
  static_assert(WTM % 32 == 0 && WTN % 64 == 0 && A_INST >= 1 && B_INST >= 1, "tile too small for the wave grid");
  static_assert(A_INST * 1024 * WAVES == A_BYTES && B_INST * 1024 * WAVES == B_BYTES, "DMA shares");
  static_assert(LDS_BYTES <= 160 * 1024 && (S - 1) * LOADS < 64 && S <= 7, "ring");
};

// Home of 16-byte unit c of row r (KC: r an operand row of BK elements, KS: a
// k-row of W elements): XORed so that the rows one LDS read touches fall into
// different banks.
template <bool KC, int W, int BK>
__device__ __forceinline__ int unit_home(int r, int c) {
  if constexpr (KC) return BK == 32 ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7);
  else return W == 64 ? c ^ (4 * ((r >> 1) & 1)) : W == 32 ? c : c ^ (4 * (r & 3));
}

// One operand of a tile: where its DMA lanes read and its fragments lie.
template <bool KC, int W, int BK, int INST, int F>
struct Operand {
  static constexpr int UPR = KC ? BK / 8 : W / 8;      // 16-byte units of an LDS row
  static constexpr uint32_t ROW = UPR * 16;
  uint32_t src[INST];   // byte offset of this lane's unit from the stage's base
  uint32_t rd[KC ? BK / 16 : F];
  u32x4_t rsrc;         // KC: the tile's rows; KS: a whole stage's k-rows, the base moves on with every stage
  uint32_t koff;        // KC: byte offset of the next stage
  int64_t ld;
  int cols;             // KS: valid columns of a k-row

  // LDS row and unit of DMA lane l of the wave's instruction i
  __device__ __forceinline__ static void where(int wave, int lane, int i, int& row, int& c) {
    const int n = (wave * INST + i) * 64 + lane;
    row = n / UPR;
    c = unit_home<KC, W, BK>(row, n % UPR);
  }
  // KC: rows [0, rows) of p from k0 on; `col` maps nothing.  KS: k-rows [k0, K) and columns 0 .. cols of p,
  // tile column q at col(q).
  template <class Col>
  __device__ __forceinline__ void init(const uint16_t* p, int64_t ld_, int64_t rows_or_cols, int64_t k0, int64_t K,
                                       int wave, int lane, Col col) {
    ld = ld_;
    if constexpr (KC) {
      rsrc = make_rsrc_v(p, rows_or_cols > 0 ? ((uint32_t)(((rows_or_cols - 1) * ld + K) * 2) + 15u) & ~15u : 0u);
      koff = (uint32_t)(k0 * 2);
    } else {
      cols = (int)rows_or_cols;
      rsrc = make_rsrc_v(p + k0 * ld, stage_bytes(BK));
    }
#pragma unroll
    for (int i = 0; i < INST; ++i) {
      int row, c;
      where(wave, lane, i, row, c);
      if constexpr (KC) src[i] = (uint32_t)(row * ld * 2 + c * 16);
      else src[i] = (uint32_t)(row * ld * 2 + (int64_t)col(c * 8) * 2);
    }
  }
  // fragments: rows (KC) or columns (KS) block(f) * 32 .. + 31 of the tile
  template <class Block>
  __device__ __forceinline__ void init_read(int lane, Block block) {
    if constexpr (KC) {
      const int row = block(0) * 32 + (lane & 31), g = lane >> 5;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) rd[kk] = row * ROW + (unit_home<KC, W, BK>(row, 2 * kk + g) << 4);
    } else {
      // in 16-lane group G, lane 4j+q supplies k-row 8(G/2) + j (+4 for the second half, +16 per K step) and
      // 4 columns of its block; after the transposing read the lane holds column (lane & 31) for those k-rows
      const int G = lane >> 4, jr = (lane >> 2) & 3, q = lane & 3, krow = 8 * (G >> 1) + jr;
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int c = 4 * block(f) + 2 * (G & 1) + (q >> 1);
        rd[f] = krow * ROW + (unit_home<KC, W, BK>(krow, c) << 4) + (q & 1) * 8;
      }
    }
  }
  __device__ __forceinline__ bf16x8 read(const char* s, int kk, int f) const {
    if constexpr (KC) {
      return *reinterpret_cast<const bf16x8*>(s + rd[kk] + f * 32 * ROW);
    } else {
      const bf16x4_t lo = lds_tr4(s + rd[f] + kk * 16 * ROW);
      const bf16x4_t hi = lds_tr4(s + rd[f] + kk * 16 * ROW + 4 * ROW);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // bytes of the first `rows` k-rows of a stage, to a whole unit (KS)
  __device__ __forceinline__ uint32_t stage_bytes(int rows) const {
    return ((uint32_t)(((rows - 1) * ld + cols) * 2) + 15u) & ~15u;
  }
  // The next stage into LDS.
  __device__ __forceinline__ void issue(uint32_t lds) {
    if constexpr (KC) {
      dma16_run<INST>(rsrc, lds, src, koff);
      koff += BK * 2;
    } else {
      dma16_run<INST>(rsrc, lds, src, 0u);
      const uint64_t at = ((uint64_t)rsrc[1] << 32 | rsrc[0]) + (uint64_t)(BK * 2) * (uint64_t)ld;
      rsrc[0] = (uint32_t)at;
      rsrc[1] = (uint32_t)(at >> 32);
    }
  }
  // The last stage, of 0 < kleft < BK elements of K.
  __device__ __forceinline__ void issue_short(uint32_t lds, int wave, int lane, int kleft) {
    if constexpr (KC) {
      uint32_t v[INST];
#pragma unroll
      for (int i = 0; i < INST; ++i) {
        int row, c;
        where(wave, lane, i, row, c);
        v[i] = c * 8 < kleft ? src[i] : 0x80000000u;
      }
      dma16_run<INST>(rsrc, lds, v, koff);
    } else {
      rsrc[2] = stage_bytes(kleft);
      dma16_run<INST>(rsrc, lds, src, 0u);
    }
  }
};

// ---------------------------------------------------------------------------
// Epilogue helpers: 8 neighbouring elements of a row
// ---------------------------------------------------------------------------

// As they come from memory, to be unpacked when they are needed.
struct Raw8 {
  uint4 a, b;  // b: the second half of fp32 values
};

// n < 8: the first n only, others 0.  vec: rows start at 16-byte boundaries.
__device__ __forceinline__ Raw8 load8_raw(const void* p, int64_t at, bool f32, bool vec, int n) {
  Raw8 v = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (f32) {
    const uint32_t* s = static_cast<const uint32_t*>(p) + at;
    if (vec && n >= 8) {
      v.a = *reinterpret_cast<const uint4*>(s);
      v.b = *reinterpret_cast<const uint4*>(s + 4);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = i < n ? s[i] : 0u;
      v.a = uint4{w[0], w[1], w[2], w[3]};
      v.b = uint4{w[4], w[5], w[6], w[7]};
    }
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(p) + at;
    if (vec && n >= 8) {
      v.a = *reinterpret_cast<const uint4*>(s);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = i < n ? s[i] : 0u;
      v.a = uint4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
    }
  }
  return v;
}
__device__ __forceinline__ void unpack8(const Raw8& v, bool f32, float (&x)[8]) {
  if (f32) {
    const uint32_t w[8] = {v.a.x, v.a.y, v.a.z, v.a.w, v.b.x, v.b.y, v.b.z, v.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  } else {
    const uint32_t w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
}
__device__ __forceinline__ void load8(const void* p, int64_t at, bool f32, bool vec, int n, float (&x)[8]) {
  unpack8(load8_raw(p, at, f32, vec, n), f32, x);
}

// The same for four elements, n <= 4 of them there.
__device__ __forceinline__ uint4 load4_raw(const void* p, int64_t at, bool f32, bool vec, int n) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (f32) {
    const uint32_t* s = static_cast<const uint32_t*>(p) + at;
    if (vec && n >= 4) return *reinterpret_cast<const uint4*>(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = i < n ? s[i] : 0u;
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(p) + at;
    if (vec && n >= 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(s);
      return uint4{v.x, v.y, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i / 2] |= (i < n ? (uint32_t)s[i] : 0u) << (16 * (i & 1));
  }
  return uint4{w[0], w[1], w[2], w[3]};
}
__device__ __forceinline__ f32x4 unpack4(const uint4& v, bool f32) {
  if (f32) return f32x4{__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
  return f32x4{bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)};
}

// NT: past the caches, for results that nothing reads soon (16384 x 8192
// x 3584 850 us without, 799 with).
template <bool NT = false>
__device__ __forceinline__ void store8(void* p, int64_t at, bool vec, int n, const float (&x)[8]) {
  uint16_t* d = static_cast<uint16_t*>(p) + at;
  const uint4 v = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  if (vec && n >= 8) {
    if constexpr (NT) __builtin_nontemporal_store(u32x4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_t*>(d));
    else *reinterpret_cast<uint4*>(d) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) d[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

// What bf16's rounding leaves of a number, exactly; nothing of what is infinite or NaN there.  (fp32's 24 bits are a
// rounded number's 8, those of the rest and those of what is left then.)
__device__ __forceinline__ float bf16_rest(float x) {
  const float r = bf16_lo(pack_bf16x2(x, 0.f));
  return fabsf(r) < INFINITY ? x - r : 0.f;
}

__device__ __forceinline__ void store4(float* d, bool vec, int n, f32x4 x) {
  if (vec && n == 4) {
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(d));
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (v < n) d[v] = x[v];
  }
}

__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Normal distribution function: 1 - Q(x) with Q by the five-term rational form of Abramowitz and Stegun 7.1.26
// (|error| < 1.5e-7; the library's erfc takes four times the instructions, 90 us of a 16384 x 3584 epilogue).
__device__ __forceinline__ float normal_cdf(float x) {
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * z);
  const float q = 0.5f * t * __expf(-z * z) *
                  (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return x < 0.f ? q : 1.0f - q;
}

template <int ACT>
__device__ __forceinline__ float act_of(float x) {
  if constexpr (ACT == kActRelu) return x < 0.f ? 0.f : x;
  else if constexpr (ACT == kActGelu) return x * normal_cdf(x);
  else if constexpr (ACT == kActGeluTanh) return x * sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
  else if constexpr (ACT == kActSilu) return x * sigmoid(x);
  else return x;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
  if constexpr (ACT == kActRelu) {
    return x > 0.f ? 1.f : x != x ? x : 0.f;
  } else if constexpr (ACT == kActGelu) {
    return normal_cdf(x) + x * 0.3989422804014327f * __expf(-0.5f * x * x);
  } else if constexpr (ACT == kActGeluTanh) {
    // (beyond 30 it is 0 or 1 to the last bit; squares of numbers beyond 2^64 would be infinite)
    x = x > 30.f ? 30.f : x < -30.f ? -30.f : x;
    const float s = sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
    return s + x * s * (1.f - s) * 1.5957691216057308f * (1.f + 0.134145f * x * x);
  } else if constexpr (ACT == kActSilu) {
    const float s = sigmoid(x);
    return s * (1.f + x * (1.f - s));
  } else {
    return 1.f;
  }
}
template <class F>
__device__ __forceinline__ void for_act(int act, F f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    default: f(std::integral_constant<int, kActNone>{});
  }
}

// (largest, sum of exponentials relative to it) of two sets of columns.
__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float to = fmaxf(a.x, b.x);
  const float ref = fabsf(to) == INFINITY ? 0.f : to;  // all of it -inf: sums are 0 (NaN stays); one inf: so is the sum
  return {to, a.y * __expf(a.x - ref) + b.y * __expf(b.x - ref)};
}

struct TokenRow {
  int label;
  float lse, dloss;
  int unused;
};

// Label of token m among this call's columns, -1: another shard's, -2: no loss.
__device__ __forceinline__ int64_t label_of(const ProductParams& p, int64_t m) {
  const int64_t l = p.labels64 ? static_cast<const int64_t*>(p.labels)[m] : static_cast<const int*>(p.labels)[m];
  if (l == p.ignore) return -2;
  const int64_t c = l - p.label0;
  return c >= 0 && c < p.vocab ? c : -1;
}

// ---------------------------------------------------------------------------
// The kernel
// ---------------------------------------------------------------------------

// A group and the workgroup's tile among the group's.
struct GroupTile {
  int e, beg, rows;  // its rows are beg .. beg + rows
  int tm, tn;
};

// Inclusive sums over the wave's lanes; MOST: sums stop there (all values up to 2^30).  By lane shifts inside the vector
// unit (1, 2, 4, 8 lanes within rows of 16, then the last lanes of rows to those behind): six shuffles through LDS, one
// after another, took a third of a microsecond.
template <bool MOST = false>
__device__ __forceinline__ uint32_t lanes_below(uint32_t v, uint32_t most = 0) {
  auto add = [&](uint32_t y) { v = MOST ? min(v + y, most) : v + y; };
  add(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));   // row_shr 1
  add(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));   // row_shr 2
  add(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));   // row_shr 4
  add(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));   // row_shr 8
  add(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast 15, into rows 1 and 3
  add(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // row_bcast 31, into rows 2 and 3
  return v;
}

// Tile i of XCD x, of all groups' tiles: false where there are fewer.
//
// The counts are what the device holds, so every workgroup adds them up by itself: 64 groups a step, sums over lanes.
// Every group's tiles are dealt to all XCDs, ragged 1 by columns (an XCD has all row tiles of a column, which share
// its weights in L2; from four row tiles on, half of them and twice the columns), ragged 2 by runs of an eighth: with
// whole groups per XCD, one with half of the rows kept one XCD busy while seven idled (gradient of 32 experts' weights,
// one of them with 47 % of 7643 rows, 877 us; even groups 385).  Groups of more rows than a tile (products are what
// bounds them) and of fewer (their weights, or their result, are) take turns while there are both, so that the chip has
// work of both kinds.
template <int BM>
__device__ __forceinline__ bool find_group_tile(const ProductParams& p, int x, int i, GroupTile& out) {
  const int ln = threadIdx.x & 63, E = p.E;
  const uint32_t M = (uint32_t)(p.ragged == 1 ? p.M : p.K);
  const uint32_t per = (uint32_t)(p.ragged == 1 ? p.tiles_n : p.tiles_m * p.tiles_n);
  // of the lane's group: its rows; its row tiles, first column (ragged 2: tile) and tiles on this XCD; sums of those
  uint32_t beg, rows, row0, nt, first, w, large, small;
  uint32_t carry = 0, carry_l = 0, carry_s = 0;
  uint32_t prev_l = 0, prev_s = 0;  // the sums in front of the step
  auto step = [&](int e0) {
    prev_l = carry_l;
    prev_s = carry_s;
    const int e = e0 + ln;
    const uint32_t n = e < E ? (uint32_t)min(max((int64_t)p.counts[e], (int64_t)0), (int64_t)M) : 0;
    const uint32_t incl = min(carry + lanes_below<true>(n, M), M);  // rows behind the buffers' last are nobody's
    beg = __builtin_amdgcn_update_dpp(carry, incl, 0x138, 0xf, 0xf, false);  // wave_shr 1, the carry into lane 0
    rows = incl - beg;
    const uint64_t y = (uint32_t)(x + e) & 7;
    const uint32_t tiles = p.ragged == 1 ? (rows + BM - 1) / BM : e < E;
    const bool many = p.ragged == 1 ? tiles > 1 : rows > 256, halves = p.ragged == 1 && tiles >= 4;
    const uint32_t sh = halves ? 2 : 3;
    const uint64_t yc = halves ? y & 3 : y, yr = halves ? y >> 2 : 0;
    row0 = yr ? tiles / 2 : 0;
    nt = halves ? (yr ? tiles - tiles / 2 : tiles / 2) : tiles;
    first = (uint32_t)(yc * per >> sh);
    w = ((uint32_t)((yc + 1) * per >> sh) - first) * nt;
    large = carry_l + lanes_below(many ? w : 0);
    small = carry_s + lanes_below(many ? 0 : w);
    carry = __builtin_amdgcn_readlane(incl, 63);
    carry_l = __builtin_amdgcn_readlane(large, 63);
    carry_s = __builtin_amdgcn_readlane(small, 63);
  };
  for (int e0 = 0; e0 < E; e0 += 64) step(e0);
  const uint32_t n_l = carry_l, n = carry_l + carry_s;
  if ((uint32_t)i >= n) return false;
  const uint32_t both = 2 * min(n_l, carry_s);
  const bool of_large = (uint32_t)i < both ? !(i & 1) : n_l > carry_s;
  const uint32_t idx = (uint32_t)i < both ? i / 2 : i - both / 2;
  carry = carry_l = carry_s = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    if (E > 64) step(e0);  // else as it stands
    const uint64_t behind = __ballot((of_large ? large : small) > idx);
    if (!behind) continue;
    const int l = __builtin_ctzll(behind);  // (groups without such tiles have the sum of the group before)
    const uint32_t up_to = __builtin_amdgcn_readlane(of_large ? large : small, max(l - 1, 0));
    // the sum up to the group: of the lane before, or of the steps before
    const uint32_t prev = l > 0 ? up_to : of_large ? prev_l : prev_s;
    out.e = e0 + l;
    out.beg = __builtin_amdgcn_readlane(beg, l);
    out.rows = __builtin_amdgcn_readlane(rows, l);
    const uint32_t j = idx - prev, f = __builtin_amdgcn_readlane(first, l);
    if (p.ragged == 1) {
      const uint32_t t = __builtin_amdgcn_readlane(nt, l), c = __builtin_amdgcn_readlane(w, l) / t;
      out.tm = (int)(__builtin_amdgcn_readlane(row0, l) + j / c);
      out.tn = (int)(f + j % c);
    } else {
      decode_grouped((int)(f + j), p.tiles_m, p.tiles_n, p.group_m, out.tm, out.tn);
    }
    return true;
  }
  return false;
}

// A tile's place: of its group, in C, and which part of its K.
struct TileSpot {
  const uint16_t* A;
  const uint16_t* B;
  int64_t M, K;      // rows of the group (the matrix), length of the sum
  int64_t crow;      // first row of the group in C (ragged 1)
  int64_t coff;      // element offset of the group's C (ragged 2)
  int tm, tn;        // in tiles of the launch's shape
  int64_t m0;
  uint32_t t, part;  // among the tiles that are cut
  int parts;
};

template <class C, bool AKC, bool BKC, int EPI>
__device__ __forceinline__ void product_tile(const ProductParams& p, const TileSpot& at, char* smem) {
  constexpr bool kSwiglu = EPI == kProdSwiglu, kDlogits = EPI == kProdDlogits || EPI == kProdDlogits3;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const uint16_t* A = at.A;
  const uint16_t* B = at.B;
  const int64_t M = at.M, K = at.K, crow = at.crow, coff = at.coff, m0 = at.m0;
  const uint32_t t = at.t, part = at.part;
  const int parts = at.parts, tn = at.tn;
  const int n0 = tn * (kSwiglu ? C::BN / 2 : C::BN);  // SwiGLU: of the output's columns
  const int64_t nk = (K + C::BK - 1) / C::BK;
  const int64_t s0 = part * nk / parts;
  const int ns = (int)((part + 1) * nk / parts - s0);
  const int64_t k0 = s0 * C::BK;

  // ---- operands ----
  Operand<AKC, C::BM, C::BK, C::A_INST, C::FM> a;
  Operand<BKC, C::BN, C::BK, C::B_INST, C::FN> b;
  if constexpr (AKC) a.init(A + m0 * p.lda, p.lda, min<int64_t>(M - m0, C::BM), k0, K, wave, lane, [](int q) { return q; });
  else a.init(A, p.lda, M, k0, K, wave, lane, [&](int q) { return (int)m0 + q; });
  if constexpr (BKC) b.init(B + (int64_t)n0 * p.ldb, p.ldb, min<int64_t>(p.N - n0, C::BN), k0, K, wave, lane, [](int q) { return q; });
  else b.init(B, p.ldb, p.b_cols, k0, K, wave, lane, [&](int q) {
    if constexpr (kSwiglu) return q < C::BN / 2 ? n0 + q : p.up + n0 + (q - C::BN / 2);
    else return n0 + q;
  });
  a.init_read(lane, [&](int f) { return wm * C::FM + f; });
  b.init_read(lane, [&](int f) {
    // SwiGLU: a wave's gate columns are adjacent, its up columns the same ones of the up half
    constexpr int H = C::FN / 2;
    if constexpr (kSwiglu) return f < H ? wn * H + f : C::WN * H + wn * H + (f - H);
    else return wn * C::FN + f;
  });

  // ---- main loop ----
  // vocabulary: a thread has one row's label (as a column of the tile; -1 elsewhere, -2 no loss) and numbers, loaded
  // before the products and kept in LDS for the epilogue (loaded there, one latency per eight rows, they took 12 us)
  TokenRow token = {-1, 0.f, 0.f, 0};
  if constexpr (EPI == kProdStats || kDlogits) {
    static_assert(C::NT >= C::BM, "a row per thread");
    if (tid < C::BM && m0 + tid < M) {
      const int64_t label = label_of(p, m0 + tid), c = label - p.first_col - n0;
      token.label = label < 0 ? (int)label : c >= 0 && c < C::BN ? (int)c : -1;
      if constexpr (kDlogits) {
        token.lse = p.lse[m0 + tid];
        // bf16 rounds this token's gradients of the logits; where every token has the same dloss (a mean's 1 / T), those
        // of the labels, about -dloss, would all be off by the same, up to 2^-8 of it: without its significand they are
        // about a power of two, and the products' sums take it back
        token.dloss = p.dloss[m0 + tid] / *p.scale;
      }
    }
  }
  constexpr bool SCALED = !(AKC && !BKC);  // gradients
  float scale = 1.f;
  if constexpr (SCALED) {
    if (p.scale) scale = *p.scale;
  }
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  f32x16 acc[C::FM][C::FN];
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  // whole stages, and what the sum's last one holds if it is shorter
  const int nf = (int)min<int64_t>(ns, (K - k0) / C::BK), rest = ns > nf ? (int)(K - k0 - (int64_t)nf * C::BK) : 0;
  uint32_t wr = lds_base, rd = 0;
  const uint32_t a_lds = wave * (C::A_INST * 1024), b_lds = C::A_BYTES + wave * (C::B_INST * 1024);
  auto next_slot = [](uint32_t o, uint32_t base) { return o + C::STAGE == base + C::S * C::STAGE ? base : o + C::STAGE; };
  auto issue = [&] {
    a.issue(wr + a_lds);
    b.issue(wr + b_lds);
    wr = next_slot(wr, lds_base);
  };
  auto issue_short = [&] {
    a.issue_short(wr + a_lds, wave, lane, rest);
    b.issue_short(wr + b_lds, wave, lane, rest);
  };
  // stage j, which may be the short one or none
  auto issue_any = [&](int j) {
    if (j < nf) issue();
    else if (j < ns) issue_short();
  };
  // Row blocks of 32 that hold a row: a wave leaves the others' reads and matrix instructions out, which is what makes
  // tall tiles stream a small group's weights as fast as flat ones would.
  const int active = (int)min<int64_t>(max<int64_t>((M - m0 - wm * C::WTM + 31) / 32, 0), C::FM);
  auto main_loop = [&](auto blocks_) {
    constexpr int F = decltype(blocks_)::value;
    if constexpr (C::PP) {
      // Two groups of four waves, one wave of each on every SIMD: while one
      // reads a stage's operands from LDS (and loads the stage S - 1 ahead into
      // the slot that the stage before left), the other runs its matrix
      // instructions, so each SIMD's matrix core is fed while the partner loads.
      // The loops over whole stages hold no test but their own: a memory step
      // has to fit beside the 512 cycles of the partner's matrix instructions.
      // (Reads or loads between the matrix instructions, which shorten it, cost
      // more there: 16384 x 8192 x 3584 755 to 835 us instead of 734.)  In forward
      // products its waves go first: 734 us without, 724 with; gradients took as
      // long or 1 % longer so.
      constexpr bool FIRST = AKC && !BKC;
      bf16x8 af[C::KSTEPS][F > 0 ? F : 1], bf[C::KSTEPS][C::FN];
      auto read_stage = [&] {
        if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
        if constexpr (F > 0) {
          const char* sA = smem + rd;
          const char* sB = sA + C::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < C::KSTEPS; ++kk) {
#pragma unroll
            for (int i = 0; i < F; ++i) af[kk][i] = a.read(sA, kk, i);
#pragma unroll
            for (int j = 0; j < C::FN; ++j) bf[kk][j] = b.read(sB, kk, j);
          }
          rd = next_slot(rd, 0u);
        }
      };
      auto mfma = [&] {
        if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int kk = 0; kk < C::KSTEPS; ++kk)
#pragma unroll
          for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[kk][j], af[kk][i], acc[i][j], 0, 0, 0);
      };
      // stage j + 1 has landed: S - 2 younger ones may be in flight, or as many as there are
      auto wait_next = [&](int j) {
        if (j + C::S - 1 < ns) wait_vm<(C::S - 2) * C::LOADS>();
        else if (j + 1 < ns) wait_stage<C::S + 1, C::LOADS>(min(C::S - 2, ns - 2 - j));
      };
      auto bar = [] {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
      };
      int j = 0;
      if (wave < C::WAVES / 2) {
#pragma clang loop unroll(disable)
        for (; j + C::S - 1 < nf; ++j) {
          issue();
          read_stage();
          bar();
          mfma();
          wait_vm<(C::S - 2) * C::LOADS>();
          bar();
        }
#pragma clang loop unroll(disable)
        for (; j < ns; ++j) {
          issue_any(j + C::S - 1);
          read_stage();
          bar();
          mfma();
          wait_next(j);
          bar();
        }
      } else {
#pragma clang loop unroll(disable)
        for (; j + C::S - 1 < nf; ++j) {
          bar();
          read_stage();
          issue();
          wait_vm<(C::S - 2) * C::LOADS>();
          bar();
          mfma();
        }
#pragma clang loop unroll(disable)
        for (; j < ns; ++j) {
          bar();
          read_stage();
          issue_any(j + C::S - 1);
          wait_next(j);
          bar();
          mfma();
        }
      }
    } else {
      // All of a stage's reads go out before matrix instructions: left alone, the compiler spares registers and waits
      // for one read after another.
      bf16x8 af[C::AHEAD + 1][C::KSTEPS][F > 0 ? F : 1], bf[C::AHEAD + 1][C::KSTEPS][C::FN];
      auto read_stage = [&](auto buf_) {
        constexpr int buf = decltype(buf_)::value;
        if constexpr (F > 0) {
          const char* sA = smem + rd;
          const char* sB = sA + C::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < C::KSTEPS; ++kk) {
#pragma unroll
            for (int i = 0; i < F; ++i) af[buf][kk][i] = a.read(sA, kk, i);
#pragma unroll
            for (int j = 0; j < C::FN; ++j) bf[buf][kk][j] = b.read(sB, kk, j);
          }
          rd = next_slot(rd, 0u);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto mfma = [&](auto buf_) {
        constexpr int buf = decltype(buf_)::value;
#pragma unroll
        for (int kk = 0; kk < C::KSTEPS; ++kk)
#pragma unroll
          for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[buf][kk][j], af[buf][kk][i], acc[i][j], 0, 0, 0);
      };
      using B0 = std::integral_constant<int, 0>;
      using B1 = std::integral_constant<int, C::AHEAD>;
      int j = 0;
      if constexpr (C::AHEAD) {
        // A stage's operands are read into registers while the matrix instructions of the one before run.  The barrier
        // of step j says that stage j + 1 has landed and that every wave has read stage j, whose slot takes stage j + S.
        issue_any(C::S - 1);
        wait_stage<C::S + 1, C::LOADS>(min(C::S - 1, ns - 1));
        __syncthreads();
        read_stage(B0{});
        auto step = [&](auto cur, auto next) {
          wait_vm<(C::S - 2) * C::LOADS>();
          __syncthreads();
          issue();
          read_stage(next);
          mfma(cur);
          __builtin_amdgcn_sched_barrier(0);
        };
        auto step_any = [&](auto cur, auto next, int j) {
          if (j + 1 < ns) {
            wait_stage<C::S + 1, C::LOADS>(min(C::S - 2, ns - 2 - j));
            __syncthreads();
            issue_any(j + C::S);
            read_stage(next);
          }
          mfma(cur);
          __builtin_amdgcn_sched_barrier(0);
        };
#pragma clang loop unroll(disable)
        for (; j + 1 + C::S < nf; j += 2) {
          step(B0{}, B1{});
          step(B1{}, B0{});
        }
#pragma clang loop unroll(disable)
        for (; j < ns; j += 2) {
          step_any(B0{}, B1{}, j);
          if (j + 1 < ns) step_any(B1{}, B0{}, j + 1);
        }
      } else {
        // Each barrier says that every wave's share of stage j has landed and that every wave has read stage j - 1,
        // whose slot the next DMA overwrites.
#pragma clang loop unroll(disable)
        for (; j + C::S - 1 < nf; ++j) {
          wait_vm<(C::S - 2) * C::LOADS>();
          __syncthreads();
          issue();
          read_stage(B0{});
          mfma(B0{});
        }
#pragma clang loop unroll(disable)
        for (; j < ns; ++j) {
          wait_stage<C::S + 1, C::LOADS>(min(C::S - 2, ns - 1 - j));
          __syncthreads();
          issue_any(j + C::S - 1);
          read_stage(B0{});
          mfma(B0{});
        }
      }
    }
  };
  if (ns > 0) {
#pragma unroll
    for (int s = 0; s < C::S - 1; ++s) issue_any(s);
    if constexpr (C::PP) {
      wait_stage<C::S + 1, C::LOADS>(min(C::S - 2, ns - 1));
      __syncthreads();
    }
    // (every variant passes the same barriers)
    if (active > C::FM / 2) main_loop(std::integral_constant<int, C::FM>{});
    else if (C::FM >= 4 && active > C::FM / 4) main_loop(std::integral_constant<int, C::FM / 2>{});
    else if (C::FM >= 2 && active > 0) main_loop(std::integral_constant<int, (C::FM + 3) / 4>{});
    else main_loop(std::integral_constant<int, 0>{});
    __syncthreads();  // the ring is free: the exchange and the epilogue use it
  }

  // ---- parts of the tile's K ----
  if (parts > 1) {
    constexpr int64_t TILE = (int64_t)C::BM * C::BN;
    float* slot0 = p.parts + (int64_t)t * parts * TILE;
    // 16-byte unit u of thread tid; rows behind the last are neither written nor read (offsets past the buffer's end)
    uint32_t off[C::FM];
#pragma unroll
    for (int i = 0; i < C::FM; ++i) off[i] = m0 + wm * C::WTM + 32 * i + (lane & 31) < M ? tid * 16 : 0x80000000u;
    {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(slot0 + part * TILE, (uint32_t)(TILE * 4));
#pragma unroll
      for (int u = 0; u < C::UNITS; ++u) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = acc[u / (C::FN * 4)][(u / 4) % C::FN][4 * (u % 4) + i];
        // SC1: performed at agent scope once vmcnt says that it is stored
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), r, off[u / (C::FN * 4)], u * C::NT * 16, 0x10);
      }
    }
    wait_vmem_all();
    __syncthreads();
    int* sh = reinterpret_cast<int*>(smem);
    if (tid == 0) {
      const uint32_t n = __hip_atomic_fetch_add(p.tickets + t * kTicketStride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (n == parts - 1u) __hip_atomic_store(p.tickets + t * kTicketStride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh[0] = (int)n;
    }
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(sh[0]) != parts - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    // Parts are added in order, the loads of several (of a large tile's part: of many units) in flight together: one
    // latency per part made 1 x 2048 x 2048 on 8 parts 10.8 us.
    constexpr int AT_ONCE = C::WAVES_PER_SIMD >= 4 ? 8 : C::UNITS < 16 ? 32 : 16;  // loads, as the registers allow
    constexpr int UNITS_AT_ONCE = C::UNITS < AT_ONCE ? C::UNITS : AT_ONCE, PARTS_AT_ONCE = AT_ONCE / UNITS_AT_ONCE;
    for (int q0 = 0; q0 < parts; q0 += PARTS_AT_ONCE) {
#pragma unroll
      for (int u0 = 0; u0 < C::UNITS; u0 += UNITS_AT_ONCE) {
        f32x4 v[PARTS_AT_ONCE][UNITS_AT_ONCE];
#pragma unroll
        for (int q = 0; q < PARTS_AT_ONCE; ++q) {
          const __amdgpu_buffer_rsrc_t r = make_rsrc(slot0 + min(q0 + q, parts - 1) * TILE, (uint32_t)(TILE * 4));
#pragma unroll
          for (int u = 0; u < UNITS_AT_ONCE; ++u)
            v[q][u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                    r, off[(u0 + u) / (C::FN * 4)], (u0 + u) * C::NT * 16, 0));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < PARTS_AT_ONCE; ++q)
          if (q0 + q < parts) {
#pragma unroll
            for (int u = 0; u < UNITS_AT_ONCE; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int w = u0 + u;
                const float x = acc[w / (C::FN * 4)][(w / 4) % C::FN][4 * (w % 4) + i];
                acc[w / (C::FN * 4)][(w / 4) % C::FN][4 * (w % 4) + i] = q0 + q == 0 ? v[q][u][i] : x + v[q][u][i];
              }
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();  // sh is read: the epilogue reuses the LDS
  }

  // ---- epilogue ----
  // lanes of a row: 8 columns each, with SwiGLU 8 gate and the 8 matching up columns
  constexpr int LPR = kSwiglu ? C::WTN / 16 : C::WTN / 8, RPI = 64 / LPR;
  int l = lane;
  asm volatile("" : "+v"(l));  // keep lane-derived addressing below the K loop
  const int ml = l & 31, kg = l >> 5, rr = l / LPR, cc = l % LPR;
  char* reg = smem + wave * 32 * C::PITCH;
  const int64_t row0 = m0 + wm * C::WTM;                                  // in the group
  const int64_t col = n0 + wn * (kSwiglu ? C::WTN / 2 : C::WTN) + cc * 8;  // of the lane's first element
  const int nc = (int)min<int64_t>(max<int64_t>(p.N - col, 0), 8);
  TokenRow* tokens = reinterpret_cast<TokenRow*>(smem + C::EPI_BYTES);
  float2* wave_stats = reinterpret_cast<float2*>(tokens + C::BM);
  if constexpr (EPI == kProdStats || kDlogits) {
    if (tid < C::BM) tokens[tid] = token;
    __syncthreads();
  }
  float bias[8];
  if constexpr (EPI == kProdStore) {
    if (p.bias && nc > 0) load8(p.bias, col, p.bias_f32, p.vec & kVecBias, nc, bias);
  }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    if (row0 + i * 32 >= M) break;
    constexpr int STEPS = 32 / RPI;
    auto row_of = [&](int r) { return row0 + i * 32 + r * RPI + rr; };
    // what the epilogue reads of memory, all of the block's in flight before anything waits
    constexpr int READS = EPI == kProdStore || EPI == kProdSwigluGrad ? STEPS : 1;
    Raw8 extra[READS];
    // fp32 results go four columns a lane, so that an instruction covers whole lines here too (eight columns a lane, in
    // two halves, wrote half lines: 60 experts' 2056 x 2768 gradients 346 us, 517 past the caches)
    constexpr int LPR4 = C::WTN / 4, STEPS4 = 32 * LPR4 / 64;
    const int cc4 = l % LPR4 * 4;
    const int64_t col4 = n0 + wn * C::WTN + cc4;
    const int nc4 = (int)min<int64_t>(max<int64_t>(p.N - col4, 0), 4);
    auto row4_of = [&](int r) { return row0 + i * 32 + r * (64 / LPR4) + l / LPR4; };
    if constexpr (EPI == kProdStore) {
      if (p.res && !p.c_f32) {
#pragma unroll
        for (int r = 0; r < STEPS; ++r)
          if (row_of(r) < M && nc > 0)
            extra[r] = load8_raw(p.res, coff + (crow + row_of(r)) * p.ldr + col, p.res_f32, p.vec & kVecRes, nc);
      } else if (p.res) {
#pragma unroll
        for (int r = 0; r < STEPS4; ++r)
          if (row4_of(r) < M && nc4 > 0) {
            const uint4 v = load4_raw(p.res, coff + (crow + row4_of(r)) * p.ldr + col4, p.res_f32, p.vec & kVecRes, nc4);
            if (r & 1) extra[r / 2].b = v;
            else extra[r / 2].a = v;
          }
      }
    }
    if constexpr (EPI == kProdSwigluGrad) {
#pragma unroll
      for (int r = 0; r < STEPS; ++r)
        if (row_of(r) < M && nc > 0) {
          const int64_t at = (crow + row_of(r)) * p.ldr + col;
          extra[r].a = load8_raw(p.res, at, false, p.vec & kVecRes, nc).a;
          extra[r].b = load8_raw(p.res, at + p.N, false, p.vec & kVecRes, nc).a;
        }
    }
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 w;
#pragma unroll
        for (int v = 0; v < 4; ++v) w[v] = SCALED ? acc[i][j][4 * q + v] * scale : acc[i][j][4 * q + v];
        *reinterpret_cast<f32x4*>(reg + ml * C::PITCH + (32 * j + 8 * q + 4 * kg) * 4) = w;
      }
    wait_lgkm_all();
    auto read = [&](int r, float (&x)[8]) {
      const f32x4* s = reinterpret_cast<const f32x4*>(reg + (r * RPI + rr) * C::PITCH + cc * 32);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        x[v] = s[0][v];
        x[4 + v] = s[1][v];
      }
    };
    if constexpr (EPI == kProdStore) {
      const bool later = p.res || p.c_f32;  // what is added last, and the results, in a loop of their own
      if (!later || p.bias || p.pre || p.act) {
#pragma clang loop unroll(disable)
        for (int r = 0; r < STEPS; ++r) {
          const int64_t m = row_of(r);
          if (m >= M || nc <= 0) continue;
          float x[8];
          read(r, x);
          if (p.bias) {
#pragma unroll
            for (int v = 0; v < 8; ++v) x[v] += bias[v];
          }
          if (p.pre) store8<true>(p.pre, m * p.ldp + col, p.vec & kVecPre, nc, x);
          if (p.act) for_act(p.act, [&](auto a_) {
#pragma unroll
            for (int v = 0; v < 8; ++v) x[v] = act_of<decltype(a_)::value>(x[v]);
          });
          if (later) {  // back to where they were
            f32x4* s = reinterpret_cast<f32x4*>(reg + (r * RPI + rr) * C::PITCH + cc * 32);
            s[0] = f32x4{x[0], x[1], x[2], x[3]};
            s[1] = f32x4{x[4], x[5], x[6], x[7]};
          } else {
            store8<true>(p.C, coff + (crow + m) * p.ldc + col, p.vec & kVecC, nc, x);
          }
        }
        if (later) wait_lgkm_all();
      }
      if (p.c_f32) {
#pragma unroll
        for (int r = 0; r < STEPS4; ++r) {
          const int64_t m = row4_of(r);
          if (m >= M || nc4 <= 0) continue;
          f32x4 x = *reinterpret_cast<const f32x4*>(reg + (r * (64 / LPR4) + l / LPR4) * C::PITCH + cc4 * 4);
          if (p.res) x += unpack4(r & 1 ? extra[r / 2].b : extra[r / 2].a, p.res_f32);
          store4(static_cast<float*>(p.C) + coff + (crow + m) * p.ldc + col4, p.vec & kVecC, nc4, x);
        }
      } else if (p.res) {
#pragma unroll
        for (int r = 0; r < STEPS; ++r) {
          const int64_t m = row_of(r);
          if (m >= M || nc <= 0) continue;
          float x[8], y[8];
          read(r, x);
          unpack8(extra[r], p.res_f32, y);
#pragma unroll
          for (int v = 0; v < 8; ++v) x[v] += y[v];
          store8<true>(p.C, coff + (crow + m) * p.ldc + col, p.vec & kVecC, nc, x);
        }
      }
    } else if constexpr (EPI == kProdPlain32) {
#pragma unroll
      for (int r = 0; r < STEPS4; ++r) {
        const int64_t m = row4_of(r);
        if (m >= M || nc4 <= 0) continue;
        const f32x4 x = *reinterpret_cast<const f32x4*>(reg + (r * (64 / LPR4) + l / LPR4) * C::PITCH + cc4 * 4);
        store4(static_cast<float*>(p.C) + coff + (crow + m) * p.ldc + col4, p.vec & kVecC, nc4, x);
      }
    } else {
#pragma unroll
      for (int r = 0; r < STEPS; ++r) {
        const int64_t m = row_of(r);
        float x[8];
        read(r, x);
        if constexpr (EPI == kProdPlain) {
          if (m < M && nc > 0) store8<true>(p.C, coff + (crow + m) * p.ldc + col, p.vec & kVecC, nc, x);
        } else if constexpr (kSwiglu) {
          if (m >= M || nc <= 0) continue;
          const f32x4* s = reinterpret_cast<const f32x4*>(reg + (r * RPI + rr) * C::PITCH + C::WTN * 2 + cc * 32);
          const float u[8] = {s[0][0], s[0][1], s[0][2], s[0][3], s[1][0], s[1][1], s[1][2], s[1][3]};
          if (p.pre) {
            const int64_t at = (crow + m) * p.ldp + col;
            store8<true>(p.pre, at, p.vec & kVecPre, nc, x);
            store8<true>(p.pre, at + p.N, p.vec & kVecPre, nc, u);
          }
#pragma unroll
          for (int v = 0; v < 8; ++v) x[v] = act_of<kActSilu>(x[v]) * u[v];
          store8<true>(p.C, (crow + m) * p.ldc + col, p.vec & kVecC, nc, x);
        } else if constexpr (EPI == kProdSwigluGrad) {
          // x = d out / d act of columns col ..; the gate's gradient goes to column col, the up's to N + col
          if (m >= M || nc <= 0) continue;
          float ga[8], up[8];
          unpack8(Raw8{extra[r].a, {}}, false, ga);
          unpack8(Raw8{extra[r].b, {}}, false, up);
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const float sg = sigmoid(ga[v]), d = x[v];
            x[v] = d * up[v] * sg * (1.f + ga[v] * (1.f - sg));
            up[v] = d * ga[v] * sg;
          }
          const int64_t to = (crow + m) * p.ldc + col;
          store8<true>(p.C, to, p.vec & kVecC, nc, x);
          store8<true>(p.C, to + p.N, p.vec & kVecC, nc, up);
        } else if constexpr (EPI == kProdStats) {
          // largest logit and sum of exponentials of the wave's columns, and the label's logit
          float mx = -INFINITY;
#pragma unroll
          for (int v = 0; v < 8; ++v) mx = v < nc ? fmaxf(mx, x[v]) : mx;
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
          float sum = 0.f;
          const float ref = fabsf(mx) == INFINITY ? 0.f : mx;
#pragma unroll
          for (int v = 0; v < 8; ++v) sum += v < nc ? __expf(x[v] - ref) : 0.f;
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1) sum += __shfl_xor(sum, d, 64);
          const int lr = wm * C::WTM + i * 32 + r * RPI + rr, at = tokens[lr].label - (wn * C::WTN + cc * 8);
          if (cc == 0) wave_stats[wn * C::BM + lr] = float2{mx, sum};
          if (m < M && at >= 0 && at < nc) {
            float z = x[0];
#pragma unroll
            for (int v = 1; v < 8; ++v) z = v == at ? x[v] : z;
            p.target[m] = z;
          }
        } else {  // kDlogits
          static_assert(kDlogits, "epilogue");
          if (m >= M) continue;
          const TokenRow t = tokens[wm * C::WTM + i * 32 + r * RPI + rr];
          const int at = t.label - (wn * C::WTN + cc * 8);
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            float d = __expf(x[v] - t.lse);
            if (v == at) d -= 1.f;
            // (a token without a loss, or a column behind the last, has none of it, whatever its logits are)
            x[v] = t.label == -2 || v >= nc ? 0.f : d * t.dloss;
          }
          // the scratch rows are whole units: columns behind the last are zeros, as the products behind read them
          if (col < p.ldc) {
            store8(p.C, m * p.ldc + col, true, 8, x);
            if constexpr (EPI == kProdDlogits3) {  // (4096 x 4096 x 16384: 493 us, 473 with the first part alone)
#pragma unroll
              for (int t = 1; t < 3; ++t) {
#pragma unroll
                for (int v = 0; v < 8; ++v) x[v] = bf16_rest(x[v]);
                store8(p.C, t * p.c_stride + m * p.ldc + col, true, 8, x);
              }
            }
          }
        }
      }
    }
    wait_lgkm_all();  // this block's reads are done before the next block's writes
  }
  if constexpr (EPI == kProdStats) {
    // the waves' columns of a row, joined in order
    __syncthreads();
    for (int r = tid; r < C::BM && m0 + r < M; r += C::NT) {
      float2 s = wave_stats[r];
#pragma unroll
      for (int w = 1; w < C::WN; ++w) s = join_stats(s, wave_stats[w * C::BM + r]);
      p.stats[(int64_t)tn * p.M + m0 + r] = s;
    }
  }
}

// FLAT: the shape for row tiles of at most its height (of small groups), C's otherwise; both as wide.
template <class C, class FLAT, bool AKC, bool BKC, int EPI>
__global__ __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(C::WAVES_PER_SIMD, C::WAVES_PER_SIMD)))
void product_kernel(ProductParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // Workgroups are dealt round-robin to the 8 XCDs: each XCD gets neighbouring tiles, for its L2.
  TileSpot at = {p.A, p.B, p.M, p.K, 0, 0, 0, 0, 0, 0, 0, 1};
  if (p.ragged) {
    GroupTile g;
    if (!find_group_tile<C::BM>(p, blockIdx.x & 7, blockIdx.x >> 3, g)) return;
    at.tm = g.tm;
    at.tn = g.tn;
    at.A += (int64_t)g.beg * p.lda;
    if (p.ragged == 1) {
      at.crow = g.beg;
      at.M = g.rows;
      at.B += g.e * p.b_stride;
    } else {
      at.K = g.rows;
      at.B += (int64_t)g.beg * p.ldb;
      at.coff = g.e * p.c_stride;
    }
  } else {
    // tiles below p.whole, then the parts of the others
    const bool whole = blockIdx.x < (uint32_t)p.whole;
    const uint32_t b = whole ? blockIdx.x : blockIdx.x - p.whole, n = whole ? p.whole : gridDim.x - p.whole;
    const uint32_t xcd = b & 7, id = xcd * (n >> 3) + min(xcd, n & 7) + (b >> 3);
    at.t = id;
    if (!whole) {
      at.parts = p.split;
      at.t = id / at.parts;
      at.part = id - at.t * at.parts;
    }
    decode_grouped((int)(whole ? at.t : at.t + p.whole), p.tiles_m, p.tiles_n, p.group_m, at.tm, at.tn);
  }
  at.tm = __builtin_amdgcn_readfirstlane(at.tm);
  at.tn = __builtin_amdgcn_readfirstlane(at.tn);
  at.m0 = (int64_t)at.tm * C::BM;
  if constexpr (!std::is_void_v<FLAT>) {
    static_assert(FLAT::BN == C::BN && FLAT::NT == C::NT, "flat tiles");
    if (p.ragged == 1 && at.M - at.m0 <= FLAT::BM) {
      product_tile<FLAT, AKC, BKC, EPI>(p, at, smem);
      return;
    }
  }
  product_tile<C, AKC, BKC, EPI>(p, at, smem);
}

template <class C, class FLAT, bool AKC, bool BKC, int EPI>
hipError_t launch_product_cfg(const ProductParams& p, int64_t grid, hipStream_t stream) {
  static PerDeviceFlag attr_set;
  uint32_t lds = C::LDS_BYTES;
  if constexpr (!std::is_void_v<FLAT>) lds = std::max<uint32_t>(lds, FLAT::LDS_BYTES);
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (!attr_set.is_set(dev)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&product_kernel<C, FLAT, AKC, BKC, EPI>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    attr_set.set(dev);
  }
  hipLaunchKernelGGL((product_kernel<C, FLAT, AKC, BKC, EPI>), dim3((unsigned)grid), dim3(C::NT), lds, stream, p);
  return hipGetLastError();
}

// The tile shapes, in the order of ProductTile.
using ProdTile32 = PCfg<32, 128, 1, 2, 64, 4>;
using ProdTile64 = PCfg<64, 64, 2, 1, 64, 4>;
using ProdTile64w = PCfg<64, 128, 2, 2, 64, 3>;
using ProdTile128 = PCfg<128, 128, 4, 2, 64, 2>;
using ProdTile256 = PCfg<256, 256, 2, 4, 32, 4, true>;
// gradients of weights: two workgroups per CU, one's stores beside the other's products
using ProdTile128w = PCfg<128, 256, 2, 4, 32, 3, true>;
// of 256-row tiles that hold 128 rows or fewer: the ring holds more of B's stages, 64 KB or more in flight instead of
// 48; rows along the sum come in whole 128-byte lines
template <bool BKC>
using ProdFlat256 = std::conditional_t<BKC, PCfg<128, 256, 2, 4, 64, 3>, PCfg<128, 256, 2, 4, 32, 6>>;

template <bool AKC, bool BKC, int EPI>
hipError_t launch_product_tile(const ProductParams& p, int tile, int64_t grid, hipStream_t stream) {
  switch (tile) {
    case kProd32: return launch_product_cfg<ProdTile32, void, AKC, BKC, EPI>(p, grid, stream);
    case kProd64: return launch_product_cfg<ProdTile64, void, AKC, BKC, EPI>(p, grid, stream);
    case kProd64w: return launch_product_cfg<ProdTile64w, void, AKC, BKC, EPI>(p, grid, stream);
    case kProd128: return launch_product_cfg<ProdTile128, void, AKC, BKC, EPI>(p, grid, stream);
    case kProd256:
      // only the epilogues of expert products see small groups
      if constexpr (EPI != kProdStats && EPI != kProdDlogits && EPI != kProdDlogits3)
        return launch_product_cfg<ProdTile256, ProdFlat256<BKC>, AKC, BKC, EPI>(p, grid, stream);
      else
        return launch_product_cfg<ProdTile256, void, AKC, BKC, EPI>(p, grid, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace mk
