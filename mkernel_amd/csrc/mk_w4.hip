// mk_w4.hip — products of a few rows with 4-bit weights and group scales
// (gfx950): dense, and for the routed experts of a small batch.
//
//   y[m, n] = sum_k x[m, k] * (q[k, n] - z[g(k), n]) * s[g(k), n]
//
// q in 0 .. 15, z 8 or a zero point, s bf16 per `group` rows of K.  Weights lie
// in the order in which the matrix instruction reads them: a 16-byte unit per
// lane holds the 32 codes that lane feeds to four 16 x 16 x 32 MFMAs (16
// columns, 128 rows of K), so a wave reads 1 KB in one piece and nothing goes
// through LDS on the way in.  Two such tiles of neighbouring columns and their
// scales and zero points are one block, the blocks of a pair of tiles one run
// along K: a wave's reads stay in few pages.
//
// A code becomes the bf16 number 128 + q by setting bits (0x4300 | q, exact);
// the product with the constant -(128 + z) is one more MFMA into the same
// accumulator.  A group's sum of x * (q - z) is then multiplied with its scale
// in fp32: no rounding but the fp32 sums' and the one of the result.
//
// x is the first operand, so a lane of the result holds one column of four rows
// of x, and needs that column's scale only.  The waves of a workgroup share a
// column tile and split K; their sums meet in LDS in wave order.
#include <algorithm>
#include <type_traits>

#include "mk_device.h"
#include "mk_internal.h"

namespace mk {
namespace {

constexpr int kTile = 16;    // columns of a tile
constexpr int kBlock = 128;  // rows of K of a 16-byte unit per lane

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight codes of one word as bf16 128 + q: nibbles i and i + 4 are elements
// 2i and 2i + 1.  `mask` and `bias` are 0x000f000f and 0x43004300 in registers,
// so that a pair is one v_and_or_b32 (with literals it is two instructions).
__device__ __forceinline__ bf16x8 expand(uint32_t w, uint32_t mask, uint32_t bias) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((w >> (4 * i)) & mask) | bias;
  return __builtin_bit_cast(bf16x8, v);
}

// All eight elements bf16 -(128 + z), z in 0 .. 127.
__device__ __forceinline__ bf16x8 minus_offset(uint32_t z) {
  const uint32_t h = 0xc300u | z, hh = h | h << 16;
  return __builtin_bit_cast(bf16x8, (u32x4{hh, hh, hh, hh}));
}

__device__ __forceinline__ float silu(float x) { return x / (1.f + __expf(-x)); }

// Loads past a range give zeros without traffic: offsets from here on are past
// every range (all are checked to span less).
constexpr uint32_t kNowhere = 0x80000000u;

__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

// What one step of 128 rows of K needs: packed codes, scales and zero points of
// this lane's column (a word has both tiles of a pair, group by group), and x.
//
// An MFMA takes x as 16 rows by 32 of K, 16 bytes per lane; the step's four are
// XQ = 4 loads.  With at most 4 rows three quarters of those lanes would load
// nothing, so one load (XQ = 1) brings the four MFMAs' parts at once, lane
// 4 j + r of 16 the part of row r for MFMA j, and a rotation by 4 j lanes moves
// them in place (the other lanes then hold parts of other MFMAs, which end in
// rows that are not stored).  The loads of x, mostly empty, were the largest
// cost of a decode step beside the weights: 12 of 67 us.
template <int MT, int NT, int SUB, bool ZEROS, int XQ>
struct Step {
  u32x4 w[NT];
  static constexpr int PAIRS = NT == 4 ? 2 : NT;  // four tiles are two pairs; else each tile reads its pair's
  uint32_t s[PAIRS][4 / SUB];
  uint32_t z[ZEROS ? PAIRS : 1][SUB == 1 ? 2 : 1];
  u32x4 x[MT][XQ];
};

// Lane i of each 16 gets lane i + 4 J.
template <int J>
__device__ __forceinline__ u32x4 from_quarter(u32x4 v) {
  if constexpr (J > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (uint32_t)__builtin_amdgcn_mov_dpp((int)v[i], 0x120 + 16 - 4 * J /* row_ror */, 0xf, 0xf, true);
  }
  return v;
}

// Bytes of a block: two tiles' codes, their scales [16 columns][groups][2 tiles]
// and zero points (the same order).
constexpr uint32_t block_bytes(int groups, bool zeros) { return 2048u + 64u * groups + (zeros ? 32u * groups : 0u); }

// A wave's pairs of column tiles (the run of blocks of each) and its rows of x.
template <int MT, int NT>
struct Source {
  __amdgpu_buffer_rsrc_t w[NT == 4 ? 2 : NT], x;
  int odd[NT];       // which of its pair a tile is
  uint32_t row[MT];  // byte offset of this lane's row, kNowhere where there is none
  int32_t most;      // last multiple of 8 below K, less this lane's first k in a step
};

template <int MT, int NT, int SUB, bool ZEROS, int XQ>
__device__ __forceinline__ void load(Step<MT, NT, SUB, ZEROS, XQ>& st, const Source<MT, NT>& t, uint32_t kb, int lane) {
  constexpr int G = 4 / SUB;
  const uint32_t at = kb * block_bytes(G, ZEROS), sat = at + (lane & 15) * (4 * G), zat = at + (lane & 15) * (2 * G);
#pragma unroll
  for (int n = 0; n < NT; ++n)
    st.w[n] = load16(t.w[NT == 4 ? n / 2 : n], at + lane * 16 + 1024 * (NT == 4 ? n % 2 : t.odd[n]));
#pragma unroll
  for (int n = 0; n < st.PAIRS; ++n) {
    if constexpr (G == 1) {
      st.s[n][0] = __builtin_amdgcn_raw_buffer_load_b32(t.w[n], (int)sat + 2048, 0, 0);
    } else if constexpr (G == 2) {
      const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(t.w[n], (int)sat + 2048, 0, 0));
      st.s[n][0] = v[0];
      st.s[n][1] = v[1];
    } else {
      const u32x4 v = load16(t.w[n], sat + 2048);
#pragma unroll
      for (int i = 0; i < 4; ++i) st.s[n][i] = v[i];
    }
    if constexpr (ZEROS) {
      const int zo = (int)zat + 2048 + 64 * G;
      if constexpr (G == 1) {
        st.z[n][0] = __builtin_amdgcn_raw_buffer_load_b16(t.w[n], zo, 0, 0);
      } else if constexpr (G == 2) {
        st.z[n][0] = __builtin_amdgcn_raw_buffer_load_b32(t.w[n], zo, 0, 0);
      } else {
        const u32x2 zv = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(t.w[n], zo, 0, 0));
        st.z[n][0] = zv[0];
        st.z[n][1] = zv[1];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < XQ; ++j) {
    const bool in = (int32_t)(kb * kBlock) + j * 32 <= t.most;
#pragma unroll
    for (int m = 0; m < MT; ++m) st.x[m][j] = load16(t.x, in ? t.row[m] + kb * 256 + 64 * j : kNowhere);
  }
}

template <int MT, int NT, int SUB, bool ZEROS, int XQ>
__device__ __forceinline__ void multiply(const Step<MT, NT, SUB, ZEROS, XQ>& st, const int (&odd)[NT], uint32_t mask,
                                         uint32_t bias, f32x4 (&acc)[NT][MT]) {
  bf16x8 x[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    x[m][0] = __builtin_bit_cast(bf16x8, st.x[m][0]);
    x[m][1] = __builtin_bit_cast(bf16x8, XQ == 1 ? from_quarter<1>(st.x[m][0]) : st.x[m][1 % XQ]);
    x[m][2] = __builtin_bit_cast(bf16x8, XQ == 1 ? from_quarter<2>(st.x[m][0]) : st.x[m][2 % XQ]);
    x[m][3] = __builtin_bit_cast(bf16x8, XQ == 1 ? from_quarter<3>(st.x[m][0]) : st.x[m][3 % XQ]);
  }
#pragma unroll
  for (int g = 0; g < 4 / SUB; ++g) {
    f32x4 base[MT];  // sum of -136 x: the same for every column where there are no zero points
    if constexpr (!ZEROS) {
      const bf16x8 off = minus_offset(8u);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        base[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SUB; ++i)
          base[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[m][g * SUB + i], off, base[m], 0, 0, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // this lane's column: scale (and zero point) of the tile in its pair's word
      const int pair = NT == 4 ? n / 2 : n;
      const uint32_t sw = st.s[pair][g];
      const float s = __uint_as_float(NT == 4 ? (n % 2 ? sw & 0xffff0000u : sw << 16) : sw >> (16 * odd[n]) << 16);
      bf16x8 off;
      if constexpr (ZEROS) off = minus_offset(st.z[pair][g / 2] >> (16 * (g % 2) + 8 * (NT == 4 ? n % 2 : odd[n])) & 255u);
      f32x4 part[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) part[m] = ZEROS ? f32x4{0.f, 0.f, 0.f, 0.f} : base[m];
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const bf16x8 q = expand(st.w[n][g * SUB + i], mask, bias);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const bf16x8 xv = x[m][g * SUB + i];
          if constexpr (ZEROS) part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv, off, part[m], 0, 0, 0);
          part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv, q, part[m], 0, 0, 0);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[n][m][r] = fmaf(s, part[m][r], acc[n][m][r]);
    }
  }
}

// The steps kb = first, first + stride, ... of a wave's tiles and rows: a ring
// of P steps in registers.  The barriers keep a step's loads behind the step
// before, in order: loads return in the order of their issue, so a step waits
// for its own only.  The last P steps load nothing more (a load that nobody
// needs would still be waited for before its registers are used again); those
// past the end found zeros.
template <int MT, int NT, int SUB, bool ZEROS, int XQ, int P>
__device__ __forceinline__ void sweep(const Source<MT, NT>& t, uint32_t KB, uint32_t first, uint32_t stride, int lane,
                                      f32x4 (&acc)[NT][MT]) {
  uint32_t mask = 0x000f000fu, bias = 0x43004300u;
  asm volatile("" : "+s"(mask));
  asm volatile("" : "+v"(bias));
  Step<MT, NT, SUB, ZEROS, XQ> st[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    load(st[i], t, first + i * stride, lane);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint32_t kb = first;
  for (; kb + P * stride < KB; kb += P * stride) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      multiply(st[i], t.odd, mask, bias, acc);
      __builtin_amdgcn_sched_barrier(0);
      load(st[i], t, kb + (i + P) * stride, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) multiply(st[i], t.odd, mask, bias, acc);
}

// One value of the result.
__device__ __forceinline__ void store(const W4KParams& p, int64_t r, int64_t c, int64_t width, float v) {
  if (p.out_type == kW4F32) {
    static_cast<float*>(p.C)[r * p.ldc + c] = v;
    return;
  }
  uint16_t* out = static_cast<uint16_t*>(p.C) + r * p.ldc + c;
  const __bf16 hi = (__bf16)v;
  out[0] = __builtin_bit_cast(uint16_t, hi);
  // what the rounding left, in the second half of the row
  if (p.out_type == kW4Pair) out[width] = __builtin_bit_cast(uint16_t, (__bf16)(v - (float)hi));
}

// How many of a workgroup's W waves share an item's K: few items are cut into
// more parts so that all waves have work, many are left whole; between, what
// needs the fewest steps in the longest wave (a round costs about kRoundSteps
// steps beside its own: row tables, first loads, the sum over waves).
constexpr int kRoundSteps = 3;
__host__ __device__ __forceinline__ int choose_split(uint32_t items, uint32_t waves, uint32_t KB, int W) {
  int best = 1;
  uint64_t least = ~0ull;
  for (int log = 0; 1 << log <= W; ++log) {
    // rounds of items << log wave tasks; items < 2^31, so a wave's items are counted first
    const uint32_t each = waves >> log ? waves >> log : 1;
    const uint64_t cost = (uint64_t)((items + each - 1) / each) * (((KB + (1u << log) - 1) >> log) + kRoundSteps);
    if (cost < least) least = cost, best = 1 << log;
  }
  return best;
}

// The real row blocks' experts and rows, and the passes of ROWS rows that they
// take, for up to kListed blocks: read once per workgroup, so that an item
// starts without a chain of loads.
constexpr int kListed = 512;
template <int ROWS>
struct PassList {
  int expert[kListed];
  uint16_t rows[kListed], first[kListed + 1];    // first pass of each block
  uint16_t block[kListed * (kFlagRows / ROWS)];  // block of each pass
  int scratch[17];
};

// Inclusive prefix sum over the workgroup's 64 W threads.
template <int W>
__device__ __forceinline__ int prefix(int v, int* s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(v, d, 64);
    if (lane >= d) v += y;
  }
  if (lane == 63) s[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += s[w];
  return v;
}

__device__ __forceinline__ int block_rows(const W4KParams& p, int64_t b) {
  const int e = p.rb_expert[b];
  if (e < 0 || e >= p.w.E) return 0;
  return p.rb_rows ? max(0, min(p.rb_rows[b], kFlagRows)) : kFlagRows;
}

// Steps in flight per wave: what 120 registers hold, at least two.
constexpr int steps_ahead(int mt, int nt, int sub, bool zeros, int xq) {
  const int pairs = nt == 4 ? 2 : nt;
  const int regs = 4 * nt + pairs * (4 / sub) + (zeros ? pairs * (sub == 1 ? 2 : 1) : 0) + 4 * mt * xq;
  return 120 / regs < 2 ? 2 : 120 / regs > 6 ? 6 : 120 / regs;
}

// W waves.  An item is NT column tiles (with SwiGLU: the first half gate tiles,
// the second the matching up tiles) of a pass of up to 16 MTX rows; `split`
// waves share its K.  Where x goes as bf16 pairs (PARTS 2) the halves of a row
// take two lanes of a row tile, and their two sums are added at the end.  The
// workgroups of the grid walk the items in turn, as many as the device's row
// count and tables say there are.  FEW, MANY: whether passes of at most 4 row
// lanes, and of more, come (see Step).
template <int MTX, int NT, int W, int SUB, bool ZEROS, int PARTS, bool EXPERTS, bool FEW, bool MANY>
__global__ __launch_bounds__(64 * W, NT == 4 ? 2 : 1) void w4_kernel(W4KParams p) {
  extern __shared__ f32x4 red[];  // [W][NT * MTX][64], used where K is split
  constexpr int ROWS = 16 * MTX / PARTS, kPasses = EXPERTS ? kFlagRows / ROWS : 1;
  __shared__ PassList<EXPERTS ? ROWS : kFlagRows> list;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const uint32_t KB = (uint32_t)((p.w.K + kBlock - 1) / kBlock);
  const int64_t pairs = (p.w.N + 2 * kTile - 1) / (2 * kTile), tile_run = (int64_t)KB * block_bytes(4 / SUB, ZEROS);
  const int per_item = p.swiglu ? NT / 2 : NT;  // output tiles
  const int col_items = (p.tile_cols + per_item - 1) / per_item;
  const int64_t width = p.swiglu ? (int64_t)p.tile_cols * kTile : p.w.N;
  uint32_t passes = p.row_blocks;
  bool listed = false;
  if constexpr (EXPERTS) {
    constexpr int per = (kListed + 64 * W - 1) / (64 * W);
    int n[per], sum = 0, blocks = p.row_blocks;
    int64_t rows_dev = p.rows_dev ? *p.rows_dev : p.M;
#pragma unroll
    for (int i = 0; i < per; ++i) {  // (not held back by the row count)
      const int b = threadIdx.x * per + i;
      n[i] = b < min(p.row_blocks, kListed) ? block_rows(p, b) : 0;
      if (b < min(p.row_blocks, kListed)) list.expert[b] = p.rb_expert[b];
    }
    blocks = (int)min((int64_t)blocks, max((int64_t)0, rows_dev / kFlagRows));
    listed = blocks <= kListed;
    passes = blocks * kPasses;
    if (listed) {
#pragma unroll
      for (int i = 0; i < per; ++i) {
        if ((int)threadIdx.x * per + i >= blocks) n[i] = 0;
        sum += (n[i] + ROWS - 1) / ROWS;
      }
      int at = prefix<W>(sum, list.scratch);
      if (threadIdx.x == 64 * W - 1) {
        list.scratch[16] = at;
        list.first[kListed] = (uint16_t)at;
      }
      at -= sum;
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const int b = threadIdx.x * per + i;
        if (b >= kListed) break;
        list.first[b] = (uint16_t)at;
        list.rows[b] = (uint16_t)n[i];
        for (int j = 0; j < (n[i] + ROWS - 1) / ROWS; ++j) list.block[at++] = (uint16_t)b;
      }
      __syncthreads();
      passes = list.scratch[16];
    }
  }
  const uint32_t items = passes * col_items;
  // (a dense launch knows its items on the host)
  const int split = EXPERTS ? __builtin_amdgcn_readfirstlane(choose_split(items, gridDim.x * W, KB, W)) : p.split;
  const int log = __builtin_ctz(split), per = W >> log, ks = wave & (split - 1);
  for (uint32_t it0 = blockIdx.x * per; it0 < items; it0 += gridDim.x * per) {
    const uint32_t it = it0 + (wave >> log);
    int64_t row0 = 0, expert = 0;
    int ci = 0, left = 0;
    if (it < items) {
      uint32_t q = it / col_items;
      if constexpr (EXPERTS) {
        // the passes of one column item side by side: they read the same weights
        int np = kPasses, b;
        if (listed) {
          b = __builtin_amdgcn_readfirstlane((int)list.block[q]);
          q = __builtin_amdgcn_readfirstlane((int)list.first[b]);
          np = __builtin_amdgcn_readfirstlane((int)list.first[b + 1]) - (int)q;
          left = __builtin_amdgcn_readfirstlane((int)list.rows[b]);
          expert = __builtin_amdgcn_readfirstlane(list.expert[b]);
        } else {
          b = q / kPasses;
          q = b * kPasses;
          left = __builtin_amdgcn_readfirstlane(block_rows(p, b));
          expert = __builtin_amdgcn_readfirstlane(p.rb_expert[b]);
        }
        const int local = (int)(it - q * col_items), pass = local % np;
        ci = local / np;
        left = min(left - ROWS * pass, ROWS);
        row0 = (int64_t)b * kFlagRows + ROWS * pass;
      } else {
        ci = (int)(it - q * col_items);
        row0 = (int64_t)q * ROWS;
        left = (int)min(p.M - row0, (int64_t)ROWS);
      }
    }
    const bool any = left > 0, few = FEW && left <= 4 / PARTS;
    const int lanes = few ? 4 : 16;  // of a row tile
    f32x4 acc[NT][MTX];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MTX; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto run = [&](auto mt, auto xq) {
      constexpr int MT = decltype(mt)::value, XQ = decltype(xq)::value;
      Source<MT, NT> t;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bool up = p.swiglu && n >= NT / 2;
        // (a last item's missing tile: its pair's other one again, which is not stored)
        const int tile = min(ci * per_item + (up ? n - NT / 2 : n), p.tile_cols - 1) + (up ? p.tile_cols : 0);
        t.odd[n] = tile & 1;
        if (NT < 4 || n % 2 == 0)
          t.w[NT == 4 ? n / 2 : n] = make_rsrc(p.w.packed + (expert * pairs + tile / 2) * tile_run, (uint32_t)tile_run);
      }
      // This lane's row of a tile, which half of a pair, and its first k in a step
      // (see Step).  Lanes past the last row read nothing; their results are not
      // stored.
      constexpr int LANES = XQ == 1 ? 4 : 16, EACH = LANES / PARTS;
      const int r = col % EACH, half = col % LANES / EACH, k0 = (XQ == 1 ? col / 4 * 32 : 0) + quad * 8;
      t.most = (int32_t)p.w.K - 8 - k0;
      const uint32_t in_row = 2 * (uint32_t)(k0 + half * p.w.K);
      if (EXPERTS && p.gather_pull) {
        t.x = make_rsrc(p.A, (uint32_t)(p.gather_rows * p.lda * 2));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          t.row[m] = kNowhere;
          if (EACH * m + r < left) {
            const int* pr = p.gather_pull + 3 * (row0 + EACH * m + r);
            const int64_t src = ((int64_t)pr[0] * p.gather_devs + pr[1]) * p.gather_tps + pr[2];
            if (pr[0] >= 0 && pr[2] >= 0 && src >= 0 && src < p.gather_rows) t.row[m] = (uint32_t)(src * p.lda * 2) + in_row;
          }
        }
      } else {
        t.x = make_rsrc(p.A + row0 * p.lda, (uint32_t)(left * p.lda * 2));
#pragma unroll
        for (int m = 0; m < MT; ++m) t.row[m] = EACH * m + r < left ? (uint32_t)((EACH * m + r) * p.lda * 2) + in_row : kNowhere;
      }
      f32x4 a[NT][MT];
      sweep<MT, NT, SUB, ZEROS, XQ, steps_ahead(MT, NT, SUB, ZEROS, XQ)>(t, KB, ks, split, lane, a);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if constexpr (PARTS == 2 && XQ == 1) {  // rows 0 and 1, then their second halves
            a[n][m][0] += a[n][m][2];
            a[n][m][1] += a[n][m][3];
          } else if constexpr (PARTS == 2) {  // second halves: rows 8 to 15, two quads on
#pragma unroll
            for (int i = 0; i < 4; ++i) a[n][m][i] += __shfl_xor(a[n][m][i], 32, 64);
          }
          acc[n][m] = a[n][m];
        }
    };
    using std::integral_constant;
    int mt = 1;
    if (any) {
      if (FEW && (few || !MANY)) {
        if constexpr (FEW) run(integral_constant<int, 1>(), integral_constant<int, 1>());
      } else if (MTX == 1 || left <= 16 / PARTS) {
        if constexpr (MANY) run(integral_constant<int, 1>(), integral_constant<int, 4>());
      } else {
        mt = MTX;
        if constexpr (MANY && MTX > 1) run(integral_constant<int, MTX>(), integral_constant<int, 4>());
      }
    }
    auto finish = [&](int n, int m, f32x4 v, f32x4 up) {
      const int64_t c = (int64_t)(ci * per_item + n) * kTile + col;
      if (c >= width) return;
      if constexpr (NT >= 2)
        if (p.swiglu)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = silu(v[i]) * up[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * quad + i;
        if (r < lanes / PARTS && lanes / PARTS * m + r < left) store(p, row0 + lanes / PARTS * m + r, c, width, v[i]);
      }
    };
    if (split == 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MTX; ++m)
          if (n < per_item && m < mt) finish(n, m, acc[n][m], acc[NT >= 2 ? (n + NT / 2) % NT : n][m]);
      continue;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MTX; ++m)
        if (m < mt) red[(wave * NT * MTX + n * MTX + m) * 64 + lane] = acc[n][m];
    __syncthreads();
    auto total = [&](int u) {
      f32x4 v = red[((wave - ks) * NT * MTX + u) * 64 + lane];
      for (int o = 1; o < split; ++o) v += red[((wave - ks + o) * NT * MTX + u) * 64 + lane];
      return v;
    };
    if (any)
      for (int u = ks; u < per_item * mt; u += split) {
        const int n = u / mt, m = u - n * mt;
        const f32x4 v = total(n * MTX + m);
        finish(n, m, v, p.swiglu ? total((n + NT / 2) * MTX + m) : v);
      }
    __syncthreads();
  }
}

template <int MTX, int NT, int W, int SUB, bool ZEROS, int PARTS, bool EXPERTS, bool FEW, bool MANY>
void launch(const W4KParams& p, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((w4_kernel<MTX, NT, W, SUB, ZEROS, PARTS, EXPERTS, FEW, MANY>), dim3(grid), dim3(64 * W),
                     W * NT * MTX * 64 * sizeof(f32x4), stream, p);
}

// One thread per 4 bytes of the packed weights.
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros,
                                                      int64_t K, int64_t N, int64_t KB, int64_t pairs, int64_t given,
                                                      int groups, int64_t words, uint32_t* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= words) return;
  const int unit = (int)(block_bytes(groups, zeros != nullptr) / 4);
  const int64_t block = i / unit, kb = block % KB, pair = block / KB % pairs, e = block / KB / pairs;
  const int at = (int)(i - block * unit);
  uint32_t w = 0;
  if (at < 512) {  // codes: [2 tiles][64 lanes][4 MFMAs], see expand()
    const int j = at & 3, lane = (at >> 2) & 63;
    const int64_t n = (2 * pair + (at >> 8)) * kTile + (lane & 15), k0 = kb * kBlock + j * 32 + (lane >> 4) * 8;
#pragma unroll
    for (int o = 0; o < 8; ++o) {
      const int64_t k = k0 + o;
      const uint32_t q = k < K && n < N ? codes[(e * K + k) * N + n] & 15u : 8u;
      w |= q << (4 * ((o & 1) * 4 + (o >> 1)));
    }
  } else {
    // scales, two to a word, then zero points, four: [16 columns][groups][2 tiles]
    const bool zero = at >= 512 + 16 * groups;
    const int first = zero ? 4 * (at - 512 - 16 * groups) : 2 * (at - 512);
    for (int o = 0; o < (zero ? 4 : 2); ++o) {
      const int u = first + o;
      const int64_t n = (2 * pair + u % 2) * kTile + u / (2 * groups), g = kb * groups + u / 2 % groups;
      const bool in = g < given && n < N;
      const int64_t src = (e * given + g) * N + n;
      if (zero) w |= (in ? zeros[src] & 15u : 8u) << (8 * o);
      else w |= (in ? (uint32_t)scales[src] : 0u) << (16 * o);
    }
  }
  out[i] = w;
}

// One thread per group and column: scale = bf16(largest magnitude / 7), code =
// round(w / scale) + 8.
__global__ __launch_bounds__(256) void w4_quantize_kernel(const uint16_t* W, int64_t K, int64_t N, int group,
                                                          int64_t groups, int64_t count, uint8_t* codes,
                                                          uint16_t* scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const int64_t n = i % N, g = i / N % groups, e = i / N / groups;
  const int64_t k0 = g * group, k1 = min(K, k0 + group);
  auto value = [&](int64_t k) { return __uint_as_float((uint32_t)W[(e * K + k) * N + n] << 16); };
  float most = 0.f;
  for (int64_t k = k0; k < k1; ++k) most = fmaxf(most, fabsf(value(k)));
  const __bf16 s = (__bf16)(most / 7.f);
  const float scale = (float)s;
  scales[i] = __builtin_bit_cast(uint16_t, s);
  for (int64_t k = k0; k < k1; ++k) {
    const float q = scale > 0.f ? rintf(value(k) / scale) : 0.f;
    codes[(e * K + k) * N + n] = (uint8_t)((int)fminf(fmaxf(q, -8.f), 7.f) + 8);
  }
}

unsigned blocks256(int64_t n) { return (unsigned)((n + 255) / 256); }

}  // namespace

int64_t w4_packed_bytes(int64_t K, int64_t N, int64_t E, int group, bool zeros) {
  return E * ((N + 2 * kTile - 1) / (2 * kTile)) * ((K + kBlock - 1) / kBlock) * block_bytes(kBlock / group, zeros);
}

hipError_t launch_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int64_t K, int64_t N,
                          int64_t E, int group, unsigned char* packed, hipStream_t stream) {
  const int64_t KB = (K + kBlock - 1) / kBlock, pairs = (N + 2 * kTile - 1) / (2 * kTile);
  const int64_t words = w4_packed_bytes(K, N, E, group, zeros != nullptr) / 4;
  hipLaunchKernelGGL(w4_pack_kernel, dim3(blocks256(words)), dim3(256), 0, stream, codes, scales, zeros, K, N, KB, pairs,
                     (K + group - 1) / group, kBlock / group, words, reinterpret_cast<uint32_t*>(packed));
  return hipGetLastError();
}

hipError_t launch_w4_quantize(const uint16_t* W, int64_t K, int64_t N, int64_t E, int group, uint8_t* codes,
                              uint16_t* scales, hipStream_t stream) {
  const int64_t groups = (K + group - 1) / group, count = E * groups * N;
  hipLaunchKernelGGL(w4_quantize_kernel, dim3(blocks256(count)), dim3(256), 0, stream, W, K, N, group, groups, count,
                     codes, scales);
  return hipGetLastError();
}

// Waves that a CU holds (by registers), the grid of a launch.
constexpr int waves_per_cu(int mt, int nt) {
  return nt == 4 ? (mt == 1 ? 12 : 8) : (mt == 1 ? 16 : 12);
}

hipError_t launch_w4(const W4KParams& args, int cus, hipStream_t stream) {
  if (args.M == 0) return hipSuccess;
  W4KParams p = args;
  const bool experts = p.rb_expert != nullptr;
  auto go = [&](auto mt, auto nt, auto w, auto sub, auto zeros, auto parts, auto ex) {
    constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value, W = decltype(w)::value;
    p.row_blocks = (int)(decltype(ex)::value ? p.M / kFlagRows : (p.M + 16 * MT - 1) / (16 * MT));
    const int per_item = p.swiglu ? NT / 2 : NT;
    const int passes = decltype(ex)::value ? kFlagRows * decltype(parts)::value / (16 * MT) : 1;
    const int64_t items = (int64_t)p.row_blocks * passes * ((p.tile_cols + per_item - 1) / per_item);
    const int64_t most = (int64_t)cus * waves_per_cu(MT, NT) / W;
    int64_t grid = std::min<int64_t>(items, most);
    if (!decltype(ex)::value) {
      p.split = choose_split((uint32_t)items, (uint32_t)(most * W), (uint32_t)((p.w.K + kBlock - 1) / kBlock), W);
      grid = std::min<int64_t>(most, (items * p.split + W - 1) / W);
    }
    constexpr int SUB = decltype(sub)::value, PARTS = decltype(parts)::value;
    constexpr bool ZEROS = decltype(zeros)::value;
    if constexpr (decltype(ex)::value) {
      launch<MT, NT, W, SUB, ZEROS, PARTS, true, true, true>(p, (int)grid, stream);
    } else if constexpr (MT == 1) {
      if (p.M <= 4) launch<MT, NT, W, SUB, ZEROS, PARTS, false, true, false>(p, (int)grid, stream);
      else launch<MT, NT, W, SUB, ZEROS, PARTS, false, false, true>(p, (int)grid, stream);
    } else {
      launch<MT, NT, W, SUB, ZEROS, PARTS, false, false, true>(p, (int)grid, stream);
    }
  };
  using std::integral_constant;
  auto with_zeros = [&](auto mt, auto nt, auto w, auto sub, auto parts, auto ex) {
    if (p.w.zeros) go(mt, nt, w, sub, std::true_type(), parts, ex);
    else go(mt, nt, w, sub, std::false_type(), parts, ex);
  };
  auto with_group = [&](auto mt, auto nt, auto w, auto parts, auto ex) {
    if (p.w.group == 32) with_zeros(mt, nt, w, integral_constant<int, 1>(), parts, ex);
    else if (p.w.group == 64) with_zeros(mt, nt, w, integral_constant<int, 2>(), parts, ex);
    else with_zeros(mt, nt, w, integral_constant<int, 4>(), parts, ex);
  };
  constexpr integral_constant<int, 1> one;
  constexpr integral_constant<int, 2> two;
  constexpr integral_constant<int, 4> four;
  constexpr integral_constant<int, 8> eight;
  if (experts) {
    // SwiGLU's gate and up tiles go in pairs where the width is a whole number of them
    const bool pairs = !p.swiglu || p.tile_cols % 2 == 0;
    if (p.parts == 2 && pairs) with_group(two, four, four, two, std::true_type());
    else if (p.parts == 2) with_group(two, two, four, two, std::true_type());
    else if (pairs) with_group(two, four, four, one, std::true_type());
    else with_group(two, two, four, one, std::true_type());
  } else if (p.M <= 16) {
    with_group(one, one, eight, one, std::false_type());
  } else {
    with_group(two, four, eight, one, std::false_type());
  }
  return hipGetLastError();
}

}  // namespace mk
