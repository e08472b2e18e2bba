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
  static constexpr uint32_t LDS_BYTES = S * STAGE > EPI_BYTES ? S * STAGE : EPI_BYTES;
  static constexpr int PER_CU = 160 * 1024 / LDS_BYTES;
  static constexpr int WAVES_PER_SIMD = PER_CU * WAVES / 4 > 0 ? PER_CU * WAVES / 4 : 1;
  static constexpr int UNITS = FM * FN * 4;  // 16-byte units of sums per thread
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
  const uint16_t* base;  // of the next stage to load (KS), of the tile (KC)
  int64_t ld;
  uint32_t bytes, koff;
  int64_t left;          // k-rows behind the next stage's first (KS)
  int cols;              // valid columns of a k-row (KS)

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
      base = p;
      bytes = rows_or_cols > 0 ? ((uint32_t)(((rows_or_cols - 1) * ld + K) * 2) + 15u) & ~15u : 0u;
      koff = (uint32_t)(k0 * 2);
    } else {
      base = p + k0 * ld;
      left = K - k0;
      cols = (int)rows_or_cols;
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
  // The next stage into LDS; `kleft`: elements of K from its first on.
  __device__ __forceinline__ void issue(uint32_t lds, int wave, int lane, int kleft) {
    if constexpr (KC) {
      const u32x4_t r = make_rsrc_v(base, bytes);
      if (kleft < BK) {
        uint32_t v[INST];
#pragma unroll
        for (int i = 0; i < INST; ++i) {
          int row, c;
          where(wave, lane, i, row, c);
          v[i] = c * 8 < kleft ? src[i] : 0x80000000u;
        }
        dma16_run<INST>(r, lds, v, koff);
      } else {
        dma16_run<INST>(r, lds, src, koff);
      }
      koff += BK * 2;
    } else {
      const int rows = left < BK ? (int)left : BK;
      const u32x4_t r = make_rsrc_v(base, rows > 0 ? ((uint32_t)(((rows - 1) * ld + cols) * 2) + 15u) & ~15u : 0u);
      dma16_run<INST>(r, lds, src, 0u);
      base += BK * ld;
      left -= BK;
    }
  }
};

// ---------------------------------------------------------------------------
// Epilogue helpers: 8 neighbouring elements of a row
// ---------------------------------------------------------------------------

// n < 8: the first n only, others 0.  vec: rows start at 16-byte boundaries.
__device__ __forceinline__ void load8(const void* p, int64_t at, bool f32, bool vec, int n, float (&x)[8]) {
  if (f32) {
    const float* s = static_cast<const float*>(p) + at;
    if (vec && n >= 8) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(s), b = *reinterpret_cast<const f32x4*>(s + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < n ? s[i] : 0.f;
    }
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(p) + at;
    if (vec && n >= 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(s);
      x[0] = bf16_lo(v.x); x[1] = bf16_hi(v.x); x[2] = bf16_lo(v.y); x[3] = bf16_hi(v.y);
      x[4] = bf16_lo(v.z); x[5] = bf16_hi(v.z); x[6] = bf16_lo(v.w); x[7] = bf16_hi(v.w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < n ? __uint_as_float((uint32_t)s[i] << 16) : 0.f;
    }
  }
}

__device__ __forceinline__ void store8(void* p, int64_t at, bool f32, bool vec, int n, const float (&x)[8]) {
  if (f32) {
    float* d = static_cast<float*>(p) + at;
    if (vec && n >= 8) {
      *reinterpret_cast<f32x4*>(d) = f32x4{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<f32x4*>(d + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) d[i] = x[i];
    }
  } else {
    uint16_t* d = static_cast<uint16_t*>(p) + at;
    const uint4 v = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    if (vec && n >= 8) {
      *reinterpret_cast<uint4*>(d) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) d[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
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

// Running sums over the groups: rows of group e and of those before it, and the row tiles before it.  64 groups a
// step, sums by shuffles.  Calls f(lane's group index or more than E, rows, rows before, tiles, tiles before) for
// each 64; returns all tiles.
template <int BM, class F>
__device__ __forceinline__ int64_t scan_groups(const int* counts, int E, int64_t M, F f) {
  const int ln = threadIdx.x & 63;
  int64_t rows0 = 0, tiles0 = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    int64_t n = e0 + ln < E ? max(counts[e0 + ln], 0) : 0;
    int64_t incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(incl, d, 64);
      if (ln >= d) incl += y;
    }
    // rows behind the buffers' last belong to nobody
    const int64_t beg = min(rows0 + incl - n, M), end = min(rows0 + incl, M);
    const int64_t tiles = (end - beg + BM - 1) / BM;
    int64_t t = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(t, d, 64);
      if (ln >= d) t += y;
    }
    f(e0, beg, end - beg, tiles0 + t - tiles, tiles);
    rows0 += __shfl(incl, 63, 64);
    tiles0 += __shfl(t, 63, 64);
  }
  return tiles0;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)v) |
                   (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32)) << 32);
}

template <class C, bool AKC, bool BKC, int EPI>
__global__ __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(1, C::WAVES_PER_SIMD)))
void product_kernel(ProductParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr bool kSwiglu = EPI == kProdSwiglu;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;

  // ---- which tile ----
  int64_t M = p.M, K = p.K, G = gridDim.x;
  const uint16_t* A = p.A;
  const uint16_t* B = p.B;
  int64_t crow = 0;  // first row of the group in C (ragged 1)
  int64_t coff = 0;  // element offset of the group's C (ragged 2)
  if (p.ragged == 1) {
    const int64_t tiles = scan_groups<C::BM>(p.counts, p.E, p.M, [](int, int64_t, int64_t, int64_t, int64_t) {});
    G = uniform64(tiles) * p.tiles_n * p.split;
    if (blockIdx.x >= G) return;
  }
  // workgroups are dealt round-robin to the 8 XCDs: each XCD gets a contiguous run of ids, hence neighbouring
  // tiles, for its L2
  const uint32_t g = (uint32_t)G, xcd = blockIdx.x & 7;
  const uint32_t id = xcd * (g >> 3) + min(xcd, g & 7) + (blockIdx.x >> 3);
  const uint32_t t = id / p.split, part = id - t * p.split;
  int tm, tn;
  if (p.ragged == 1) {
    // group by group, column by column: a group's row tiles share each column of its weights
    const int64_t rt = t / p.tiles_n;
    int e = 0;
    int64_t beg = 0, rows = 0, first = 0, n = 1;
    scan_groups<C::BM>(p.counts, p.E, p.M, [&](int e0, int64_t b, int64_t r, int64_t t0, int64_t tl) {
      const uint64_t mine = __ballot(rt >= t0 && rt < t0 + tl);
      if (mine) {
        const int l = __builtin_ctzll(mine);
        e = e0 + l;
        beg = __shfl(b, l, 64);
        rows = __shfl(r, l, 64);
        first = __shfl(t0, l, 64);
        n = __shfl(tl, l, 64);
      }
    });
    e = __builtin_amdgcn_readfirstlane(e);
    crow = uniform64(beg);
    M = uniform64(rows);
    const int q = (int)(t - uniform64(first) * p.tiles_n), nt = (int)uniform64(n);
    tm = q % nt;
    tn = q / nt;
    A += crow * p.lda;
    B += e * p.b_stride;
  } else if (p.ragged == 2) {
    const int per = p.tiles_m * p.tiles_n, e = t / per;
    int64_t beg = 0, rows = 0;
    scan_groups<C::BM>(p.counts, p.E, p.K, [&](int e0, int64_t b, int64_t r, int64_t, int64_t) {
      if (e >= e0 && e < e0 + 64) {
        beg = __shfl(b, e - e0, 64);
        rows = __shfl(r, e - e0, 64);
      }
    });
    beg = uniform64(beg);
    K = uniform64(rows);
    A += beg * p.lda;
    B += beg * p.ldb;
    coff = e * p.c_stride;
    decode_grouped(t - e * per, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
  } else {
    decode_grouped((int)t, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
  }
  tm = __builtin_amdgcn_readfirstlane(tm);
  tn = __builtin_amdgcn_readfirstlane(tn);
  const int64_t m0 = (int64_t)tm * C::BM;
  const int n0 = tn * (kSwiglu ? C::BN / 2 : C::BN);  // SwiGLU: of the output's columns
  const int64_t nk = (K + C::BK - 1) / C::BK;
  const int64_t s0 = part * nk / p.split;
  const int ns = (int)((part + 1) * nk / p.split - s0);
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
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  f32x16 acc[C::FM][C::FN];
#pragma unroll
  for (int i = 0; i < C::FM; ++i)
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  uint32_t wr = 0;
  int64_t kleft = K - k0;
  auto issue = [&] {
    const int kl = kleft < C::BK ? (int)kleft : C::BK;
    a.issue(lds_base + wr + wave * (C::A_INST * 1024), wave, lane, kl);
    b.issue(lds_base + wr + C::A_BYTES + wave * (C::B_INST * 1024), wave, lane, kl);
    kleft -= C::BK;
    wr = wr + C::STAGE == C::S * C::STAGE ? 0u : wr + C::STAGE;
  };
  if (ns > 0) {
    if constexpr (C::PP) {
      // Two groups of four waves, one wave of each on every SIMD: while one
      // reads a stage's operands from LDS (and loads the stage S - 1 ahead into
      // the slot that the stage before left), the other runs its matrix
      // instructions, so each SIMD's matrix core is fed while the partner loads.
      bf16x8 af[C::KSTEPS][C::FM], bf[C::KSTEPS][C::FN];
      uint32_t rd = 0;
      auto read_stage = [&] {
        const char* sA = smem + rd;
        const char* sB = sA + C::A_BYTES;
#pragma unroll
        for (int kk = 0; kk < C::KSTEPS; ++kk) {
#pragma unroll
          for (int i = 0; i < C::FM; ++i) af[kk][i] = a.read(sA, kk, i);
#pragma unroll
          for (int j = 0; j < C::FN; ++j) bf[kk][j] = b.read(sB, kk, j);
        }
        rd = rd + C::STAGE == C::S * C::STAGE ? 0u : rd + C::STAGE;
      };
      auto mfma = [&] {
#pragma unroll
        for (int kk = 0; kk < C::KSTEPS; ++kk)
#pragma unroll
          for (int i = 0; i < C::FM; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[kk][j], af[kk][i], acc[i][j], 0, 0, 0);
      };
      const bool first = wave < C::WAVES / 2;
      auto mem_step = [&](int j) {
        if (first && j + C::S - 1 < ns) issue();
        read_stage();
        if (!first && j + C::S - 1 < ns) issue();
      };
      auto wait_next = [&](int j) {
        if (j + C::S - 1 < ns) wait_vm<(C::S - 2) * C::LOADS>();
        else if (j + 1 < ns) wait_stage<C::S + 1, C::LOADS>(min(C::S - 2, ns - 2 - j));
      };
      auto bar = [] {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int s = 0; s < C::S - 1; ++s)
        if (s < ns) issue();
      wait_stage<C::S + 1, C::LOADS>(min(C::S - 2, ns - 1));
      __syncthreads();
      if (first) {
        mem_step(0);
        for (int j = 0; j < ns; ++j) {
          bar();
          mfma();
          wait_next(j);
          bar();
          if (j + 1 < ns) mem_step(j + 1);
        }
      } else {
        for (int j = 0; j < ns; ++j) {
          bar();
          mem_step(j);
          wait_next(j);
          bar();
          mfma();
        }
      }
      __syncthreads();
    } else {
      uint32_t rd = 0;
      auto compute = [&] {
        const char* sA = smem + rd;
        const char* sB = sA + C::A_BYTES;
#pragma unroll
        for (int kk = 0; kk < C::KSTEPS; ++kk) {
          bf16x8 af[C::FM], bf[C::FN];
#pragma unroll
          for (int i = 0; i < C::FM; ++i) af[i] = a.read(sA, kk, i);
#pragma unroll
          for (int j = 0; j < C::FN; ++j) bf[j] = b.read(sB, kk, j);
#pragma unroll
          for (int i = 0; i < C::FM; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf[j], af[i], acc[i][j], 0, 0, 0);
        }
        rd = rd + C::STAGE == C::S * C::STAGE ? 0u : rd + C::STAGE;
      };
#pragma unroll
      for (int s = 0; s < C::S - 1; ++s)
        if (s < ns) issue();
      // Each barrier says that every wave's share of stage j has landed and that every wave has read stage j - 1,
      // whose slot the next DMA overwrites.
      int j = 0;
      for (; j + C::S - 1 < ns; ++j) {
        wait_vm<(C::S - 2) * C::LOADS>();
        __syncthreads();
        issue();
        compute();
      }
      for (; j < ns; ++j) {
        wait_stage<C::S + 1, C::LOADS>(ns - 1 - j);
        __syncthreads();
        compute();
      }
      __syncthreads();  // the ring is free: the exchange and the epilogue use it
    }
  }

  // ---- parts of the tile's K ----
  if (p.split > 1) {
    constexpr int64_t TILE = (int64_t)C::BM * C::BN;
    float* slot0 = p.parts + (int64_t)t * p.split * TILE;
    {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(slot0 + part * TILE, (uint32_t)(TILE * 4));
#pragma unroll
      for (int u = 0; u < C::UNITS; ++u) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = acc[u / (C::FN * 4)][(u / 4) % C::FN][4 * (u % 4) + i];
        // SC1: performed at agent scope once vmcnt says that it is stored
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), r, tid * 16, u * C::NT * 16, 0x10);
      }
    }
    wait_vmem_all();
    __syncthreads();
    int* sh = reinterpret_cast<int*>(smem);
    if (tid == 0) {
      const uint32_t n = __hip_atomic_fetch_add(p.tickets + t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (n == p.split - 1u) __hip_atomic_store(p.tickets + t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh[0] = (int)n;
    }
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(sh[0]) != p.split - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    for (int q = 0; q < p.split; ++q) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(slot0 + q * TILE, (uint32_t)(TILE * 4));
      // eight loads in flight: more take registers that the sums need
      constexpr int AT_ONCE = C::UNITS < 8 ? C::UNITS : 8;
#pragma unroll
      for (int u0 = 0; u0 < C::UNITS; u0 += AT_ONCE) {
        f32x4 v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
          v[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, tid * 16, (u0 + u) * C::NT * 16, 0));
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int w = u0 + u;
            const float x = acc[w / (C::FN * 4)][(w / 4) % C::FN][4 * (w % 4) + i];
            acc[w / (C::FN * 4)][(w / 4) % C::FN][4 * (w % 4) + i] = q == 0 ? v[u][i] : x + v[u][i];
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
  float bias[8];
  if constexpr (EPI == kProdStore) {
    if (p.bias && nc > 0) load8(p.bias, col, p.bias_f32, p.vec & kVecBias, nc, bias);
  }
#pragma unroll
  for (int i = 0; i < C::FM; ++i) {
    if (row0 + i * 32 >= M) break;
#pragma unroll
    for (int j = 0; j < C::FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 w;
#pragma unroll
        for (int v = 0; v < 4; ++v) w[v] = acc[i][j][4 * q + v];
        *reinterpret_cast<f32x4*>(reg + ml * C::PITCH + (32 * j + 8 * q + 4 * kg) * 4) = w;
      }
    wait_lgkm_all();
    for (int r = 0; r < 32 / RPI; ++r) {
      const int lr = r * RPI + rr;
      const int64_t m = row0 + i * 32 + lr;
      const char* s = reg + lr * C::PITCH + cc * 32;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(s), hi = *reinterpret_cast<const f32x4*>(s + 16);
      float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if constexpr (EPI == kProdStore) {
        if (m >= M || nc <= 0) continue;
        if (p.bias) {
#pragma unroll
          for (int v = 0; v < 8; ++v) x[v] += bias[v];
        }
        if (p.pre) store8(p.pre, m * p.ldp + col, false, p.vec & kVecPre, nc, x);
        if (p.act) for_act(p.act, [&](auto a_) {
#pragma unroll
          for (int v = 0; v < 8; ++v) x[v] = act_of<decltype(a_)::value>(x[v]);
        });
        if (p.res) {
          float y[8];
          load8(p.res, coff + (crow + m) * p.ldr + col, p.res_f32, p.vec & kVecRes, nc, y);
#pragma unroll
          for (int v = 0; v < 8; ++v) x[v] += y[v];
        }
        store8(p.C, coff + (crow + m) * p.ldc + col, p.c_f32, p.vec & kVecC, nc, x);
      } else if constexpr (kSwiglu) {
        if (m >= M || nc <= 0) continue;
        const f32x4 ul = *reinterpret_cast<const f32x4*>(s + C::WTN * 2), uh = *reinterpret_cast<const f32x4*>(s + C::WTN * 2 + 16);
        const float u[8] = {ul[0], ul[1], ul[2], ul[3], uh[0], uh[1], uh[2], uh[3]};
        if (p.pre) {
          const int64_t at = (crow + m) * p.ldp + col;
          store8(p.pre, at, false, p.vec & kVecPre, nc, x);
          store8(p.pre, at + p.N, false, p.vec & kVecPre, nc, u);
        }
#pragma unroll
        for (int v = 0; v < 8; ++v) x[v] = act_of<kActSilu>(x[v]) * u[v];
        store8(p.C, (crow + m) * p.ldc + col, false, p.vec & kVecC, nc, x);
      } else if constexpr (EPI == kProdSwigluGrad) {
        // x = d out / d act of columns col ..; the gate's gradient goes to column col, the up's to N + col
        if (m >= M || nc <= 0) continue;
        float ga[8], up[8];
        const int64_t at = (crow + m) * p.ldr + col;
        load8(p.res, at, false, p.vec & kVecRes, nc, ga);
        load8(p.res, at + p.N, false, p.vec & kVecRes, nc, up);
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          const float sg = sigmoid(ga[v]), d = x[v];
          x[v] = d * up[v] * sg * (1.f + ga[v] * (1.f - sg));
          up[v] = d * ga[v] * sg;
        }
        const int64_t to = (crow + m) * p.ldc + col;
        store8(p.C, to, false, p.vec & kVecC, nc, x);
        store8(p.C, to + p.N, false, p.vec & kVecC, nc, up);
      } else if constexpr (EPI == kProdStats) {
        // largest logit and sum of exponentials of the wave's columns, and the label's logit
        float mx = -INFINITY;
#pragma unroll
        for (int v = 0; v < 8; ++v) mx = v < nc ? fmaxf(mx, x[v]) : mx;
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        float sum = 0.f;
        const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int v = 0; v < 8; ++v) sum += v < nc ? __expf(x[v] - ref) : 0.f;
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) sum += __shfl_xor(sum, d, 64);
        if (m < M) {
          if (cc == 0) p.stats[(int64_t)(tn * C::WN + wn) * p.M + m] = float2{mx, sum};
          const int64_t at = label_of(p, m) - col;
          if (at >= 0 && at < nc) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              if (v == at) p.target[m] = x[v];
          }
        }
      } else {  // kProdDlogits
        if (m >= M) continue;
        const int64_t label = label_of(p, m);
        const float w = label == -2 ? 0.f : p.dloss[m], lse = p.lse[m];
        const int64_t at = label - p.first_col - col;
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          float d = __expf(x[v] - lse);
          if (v == at) d -= 1.f;
          // (a token without a loss, or a column behind the last, has none of it, whatever its logits are)
          x[v] = label == -2 || v >= nc ? 0.f : d * w;
        }
        // the scratch rows are whole units: columns behind the last are zeros, as the products behind read them
        if (col < p.ldc) store8(p.C, m * p.ldc + col, false, true, 8, x);
      }
    }
    wait_lgkm_all();  // this block's reads are done before the next block's writes
  }
}

template <class C, bool AKC, bool BKC, int EPI>
hipError_t launch_product_cfg(const ProductParams& p, int64_t grid, hipStream_t stream) {
  static PerDeviceFlag attr_set;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (!attr_set.is_set(dev)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&product_kernel<C, AKC, BKC, EPI>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES);
    if (e != hipSuccess) return e;
    attr_set.set(dev);
  }
  hipLaunchKernelGGL((product_kernel<C, AKC, BKC, EPI>), dim3((unsigned)grid), dim3(C::NT), C::LDS_BYTES, stream, p);
  return hipGetLastError();
}

// The tile shapes, in the order of ProductTile.
using ProdTile32 = PCfg<32, 128, 1, 2, 64, 4>;
using ProdTile64 = PCfg<64, 128, 2, 2, 64, 3>;
using ProdTile128 = PCfg<128, 128, 4, 2, 64, 2>;
using ProdTile256 = PCfg<256, 256, 2, 4, 32, 4, true>;

template <bool AKC, bool BKC, int EPI>
hipError_t launch_product_tile(const ProductParams& p, int tile, int64_t grid, hipStream_t stream) {
  switch (tile) {
    case kProd32: return launch_product_cfg<ProdTile32, AKC, BKC, EPI>(p, grid, stream);
    case kProd64: return launch_product_cfg<ProdTile64, AKC, BKC, EPI>(p, grid, stream);
    case kProd128: return launch_product_cfg<ProdTile128, AKC, BKC, EPI>(p, grid, stream);
    case kProd256: return launch_product_cfg<ProdTile256, AKC, BKC, EPI>(p, grid, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace mk
