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
// A code becomes the bf16 number 16 + q by setting bits (0x4180 | q << 3, exact);
// the product with the constant -(16 + z) is one more MFMA into the same
// accumulator.  A group's sum of x * (q - z) is then multiplied with its scale
// in fp32: no rounding but the fp32 sums' and the one of the result.
//
// x is the first operand, so a lane of the result holds one column of four rows
// of x, and needs that column's scale only.  The waves of a workgroup share a
// column tile and split K; their sums meet in LDS in wave order.
//
// What bounds it: for few rows the weights' bytes.  1 x 8192 x 3584: 5.8 us for
// 15 MB, 3 of them launch and first loads; 64 tokens on 18 experts of 7168 x
// 4096 (273 MB, not in a cache): 61 us, 4.5 TB/s, where a kernel that only reads
// them takes 46.  With more rows a step's instructions beside (128 x 64 weights
// against 16 rows: 166 to 183 vector instructions, 128 of them the expansion, and
// 20 MFMAs; against 32 rows 230 to 270 and 40, by group): 64 x 3584 x 8192 in
// 10.9 us (in a graph) is 345 TFLOP/s.  The expansion is paid once per 16 or 32 rows: bf16
// weights through mk_gemm are as fast at 128 rows of 3584 x 8192 (19 us) and
// twice as fast at 1024 (108 and 55); the experts' layer of 7168 / 2048 takes as
// long as its bf16 form at 1024 tokens (600 us) and twice as long at 4096.
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

// Eight codes of one word as bf16 16 + q: nibbles i and i + 4 are elements 2i
// and 2i + 1.  `mask` and `bias` are 0x00780078 and 0x41804180 in registers, so
// that a pair is a shift and one v_and_or_b32 (with literals it is three
// instructions).  128 + q, with the code in the last four bits, needs one shift
// less and is 1 to 2 % faster (64 x 8192 x 8192: 17.8 us of 18.1), but the sums
// round at up to 8 times the magnitude (1 x 2048 x 2048, fp32 result against 64
// bits: 1.3e-6 instead of 1.7e-7; 64 x 3584 x 8192: 6.0e-7 instead of 0.9e-7).
__device__ __forceinline__ bf16x8 expand(uint32_t w, uint32_t mask, uint32_t bias) {
  const u32x4 v = {((w << 3) & mask) | bias, ((w >> 1) & mask) | bias, ((w >> 5) & mask) | bias, ((w >> 9) & mask) | bias};
  return __builtin_bit_cast(bf16x8, v);
}

// All eight elements bf16 -(16 + z), z in 0 .. 15.
__device__ __forceinline__ bf16x8 minus_offset(uint32_t z) {
  const uint32_t h = 0xc180u | z << 3, hh = h | h << 16;
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
// rows that are not stored).
//
// FLIP: odd rows load the step's parts 1, 0, 3, 2 instead of 0, 1, 2, 3, and are
// put in order by 16 selects.  Rows lie a multiple of 128 bytes apart as a rule,
// and 64 bytes of each in one load come from the same half of a cache line: its
// banks are read one row after another (64 x 8192 x 8192 with one row tile 25 us,
// flipped 21, and 20 as it is where rows are 16 bytes off).  The experts' kernel is slower with
// it where few rows come (64 tokens, GEMM1 / GEMM2: 62 / 37 us, flipped 65 / 39)
// and no faster where many do (256 tokens: 142 / 93 and 143 / 92).
template <int NT, int SUB, bool ZEROS, int XQ, bool FLIP, int MT>
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
template <int NT, int MT>
struct Source {
  __amdgpu_buffer_rsrc_t w[NT == 4 ? 2 : NT], x;
  int odd[NT];       // which of its pair a tile is
  uint32_t row[MT];  // byte offset of this lane's row, kNowhere where there is none
  int32_t most;      // last multiple of 8 below K, less this lane's first k in a step
};

template <int NT, int SUB, bool ZEROS, int XQ, bool FLIP, int MT>
__device__ __forceinline__ void load(Step<NT, SUB, ZEROS, XQ, FLIP, MT>& st, const Source<NT, MT>& t, uint32_t kb, int lane) {
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
    const int part = FLIP ? j + (j % 2 ? -(lane & 1) : lane & 1) : j;
    const bool in = (int32_t)(kb * kBlock) + part * 32 <= t.most;
#pragma unroll
    for (int m = 0; m < MT; ++m) st.x[m][j] = load16(t.x, in ? t.row[m] + kb * 256 + 64 * part : kNowhere);
  }
}

template <int NT, int SUB, bool ZEROS, int XQ, bool FLIP, int MT>
__device__ __forceinline__ void multiply(const Step<NT, SUB, ZEROS, XQ, FLIP, MT>& st, const int (&odd)[NT], uint32_t mask,
                                         uint32_t bias, f32x4 (&acc)[MT][NT]) {
  bf16x8 x[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[m][j] = __builtin_bit_cast(bf16x8, st.x[m][j % XQ]);
    if constexpr (XQ == 1) {
      x[m][1] = __builtin_bit_cast(bf16x8, from_quarter<1>(st.x[m][0]));
      x[m][2] = __builtin_bit_cast(bf16x8, from_quarter<2>(st.x[m][0]));
      x[m][3] = __builtin_bit_cast(bf16x8, from_quarter<3>(st.x[m][0]));
    } else if constexpr (FLIP) {
      const bool flipped = threadIdx.x & 1;
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        u32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = st.x[m][j][i], v = st.x[m][j + 1][i];
          a[i] = flipped ? v : u;
          b[i] = flipped ? u : v;
        }
        x[m][j] = __builtin_bit_cast(bf16x8, a);
        x[m][j + 1] = __builtin_bit_cast(bf16x8, b);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < 4 / SUB; ++g) {
    f32x4 base[MT];  // sum of -24 x: the same for every column where there are no zero points
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      base[m] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (!ZEROS) {
        const bf16x8 off = minus_offset(8u);
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
      for (int m = 0; m < MT; ++m) part[m] = base[m];
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const bf16x8 q = expand(st.w[n][g * SUB + i], mask, bias);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if constexpr (ZEROS) part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[m][g * SUB + i], off, part[m], 0, 0, 0);
          part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[m][g * SUB + i], q, part[m], 0, 0, 0);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[m][n][r] = fmaf(s, part[m][r], acc[m][n][r]);
    }
  }
}

// The steps kb = first, first + stride, ... of a wave's tiles and rows: a ring
// of P steps in registers.  The barriers keep a step's loads behind the step
// before, in order: loads return in the order of their issue, so a step waits
// for its own only.  The last P steps load nothing more (a load that nobody
// needs would still be waited for before its registers are used again); those
// past the end found zeros.
template <int NT, int SUB, bool ZEROS, int XQ, bool FLIP, int P, int MT>
__device__ __forceinline__ void sweep(const Source<NT, MT>& t, uint32_t KB, uint32_t first, uint32_t stride, int lane,
                                      f32x4 (&acc)[MT][NT]) {
  uint32_t mask = 0x00780078u, bias = 0x41804180u;
  asm volatile("" : "+s"(mask));
  asm volatile("" : "+v"(bias));
  Step<NT, SUB, ZEROS, XQ, FLIP, MT> st[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    load(st[i], t, first + i * stride, lane);
    __builtin_amdgcn_sched_barrier(0);
  }
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
__host__ __device__ inline int choose_split(uint32_t items, uint32_t waves, uint32_t KB, int W) {
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

// Waves of a workgroup, and those that a CU holds (by registers): the grid of a
// launch.  Items of two row tiles take 188 to 195 registers in groups of 32 and
// 64: with 12 waves they spill (64 x 3584 x 8192 12.9 us, with 8 11.2).  In
// groups of 128 they take 155 to 162, which 12 waves have room for; that was not
// tried, nor were four row tiles.
constexpr int group_waves(int nt, int mt) { return nt == 1 || mt == 2 ? 8 : 4; }
constexpr int waves_per_cu(int nt, int mt) { return nt == 1 ? 16 : mt == 2 ? 8 : 12; }

// Steps in flight per wave.  More than about 96 KB on their way into a CU is
// slower, not faster (64 tokens on 32 experts, GEMM1 / GEMM2: 12 waves of 2
// steps of 4 KB 59 / 36 us, 12 of 4 steps 72 / 45, 16 of 2 steps 69 / 42, 8 of
// 2 steps 63 / 41; 1 x 8192 x 3584: 2 steps 5.9 us, 6 steps 7.5).  With two row
// tiles a step is 12 KB and one is enough (64 x 3584 x 8192 11.3 us, two 12.5;
// 64 x 8192 x 8192 19.4 and 19.1).
constexpr int kAhead = 2, kAheadWide = 1;

// An item is NT column tiles (with SwiGLU: the first half gate tiles, the second
// the matching up tiles) of a pass of up to 16 MT rows; `split` waves of a
// workgroup share its K.  MT = 2 expands a code once for two row tiles.  Where x
// goes as bf16 pairs (PARTS 2) the halves of a row take two lanes of the row
// tile, and their two sums are added at the end.  The workgroups of the grid walk
// the items in turn, as many as the device's row count and tables say there are;
// the passes of one column item lie side by side, since they read the same
// weights.  FEW, MANY: whether passes of at most 4 row lanes, and of more, come
// (see Step).
template <int NT, int SUB, bool ZEROS, int PARTS, bool EXPERTS, bool FEW, bool MANY, int MT>
__global__ __launch_bounds__(64 * group_waves(NT, MT), waves_per_cu(NT, MT) / 4) void w4_kernel(W4KParams p) {
  extern __shared__ f32x4 red[];  // [W][NT][64], used where K is split
  constexpr int W = group_waves(NT, MT), ROWS = 16 * MT / PARTS, kPasses = kFlagRows / ROWS;
  __shared__ PassList<EXPERTS ? ROWS : kFlagRows> list;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const uint32_t KB = (uint32_t)((p.w.K + kBlock - 1) / kBlock);
  const int64_t pairs = (p.w.N + 2 * kTile - 1) / (2 * kTile), tile_run = (int64_t)KB * block_bytes(4 / SUB, ZEROS);
  const int per_item = p.swiglu ? NT / 2 : NT;  // output tiles
  const int col_items = (p.tile_cols + per_item - 1) / per_item;
  const int64_t width = p.swiglu ? (int64_t)p.tile_cols * kTile : p.w.N;
  uint32_t passes = p.passes;
  bool listed = false;
  if constexpr (EXPERTS) {
    constexpr int per = (kListed + 64 * W - 1) / (64 * W);
    const int most = (int)(p.M / kFlagRows);
    int n[per], sum = 0;
    int64_t rows_dev = p.rows_dev ? *p.rows_dev : p.M;
#pragma unroll
    for (int i = 0; i < per; ++i) {  // (not held back by the row count)
      const int b = threadIdx.x * per + i;
      n[i] = b < min(most, kListed) ? block_rows(p, b) : 0;
      if (b < min(most, kListed)) list.expert[b] = p.rb_expert[b];
    }
    const int blocks = (int)min((int64_t)most, max((int64_t)0, rows_dev / kFlagRows));
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
  // Dense passes of one column item read the same weights: neighbouring ids lie
  // on one XCD (64 x 3584 x 8192 with one row tile 13.6 us, as launched 15.1).  Experts' seldom
  // have several, and are faster with neighbours on all XCDs (16 tokens, GEMM1:
  // 21 us and 33, 64 tokens 62 and 66).
  const uint32_t xcd = blockIdx.x & 7, G = gridDim.x;
  const uint32_t id = EXPERTS ? blockIdx.x : xcd * (G >> 3) + min(xcd, G & 7) + (blockIdx.x >> 3);
  for (uint32_t it0 = id * per; it0 < items; it0 += G * per) {
    const uint32_t it = it0 + (wave >> log);
    int64_t row0 = 0, expert = 0;
    int ci = 0, left = 0;
    if (it < items) {
      if constexpr (EXPERTS) {
        uint32_t q = it / col_items;  // a pass of the item's block
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
        ci = (int)(it / passes);
        row0 = (int64_t)(it - ci * passes) * ROWS;
        left = (int)min(p.M - row0, (int64_t)ROWS);
      }
    }
    const bool any = left > 0, few = FEW && left <= 4 / PARTS;
    const int lanes = few ? 4 : 16;  // of a row tile
    f32x4 acc[MT][NT];
#pragma unroll
    for (int n = 0; n < MT * NT; ++n) acc[n / NT][n % NT] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto run = [&](auto xq) {
      constexpr int XQ = decltype(xq)::value;
      Source<NT, MT> t;
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
#pragma unroll
      for (int m = 0; m < MT; ++m) t.row[m] = kNowhere;
      if (EXPERTS && p.gather_pull) {
        t.x = make_rsrc(p.A, (uint32_t)(p.gather_rows * p.lda * 2));
        if (r < left) {
          const int* pr = p.gather_pull + 3 * (row0 + r);
          const int64_t src = ((int64_t)pr[0] * p.gather_devs + pr[1]) * p.gather_tps + pr[2];
          if (pr[0] >= 0 && pr[2] >= 0 && src >= 0 && src < p.gather_rows) t.row[0] = (uint32_t)(src * p.lda * 2) + in_row;
        }
      } else {
        t.x = make_rsrc(p.A + row0 * p.lda, (uint32_t)(left * p.lda * 2));
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (r + 16 * m < left) t.row[m] = (uint32_t)((r + 16 * m) * p.lda * 2) + in_row;
      }
      sweep<NT, SUB, ZEROS, XQ, XQ == 4 && !EXPERTS, MT == 2 ? kAheadWide : kAhead, MT>(t, KB, ks, split, lane, acc);
      if constexpr (PARTS == 2) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (XQ == 1) {  // rows 0 and 1, then their second halves
            acc[0][n][0] += acc[0][n][2];
            acc[0][n][1] += acc[0][n][3];
          } else {  // second halves: rows 8 to 15, two quads on
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[0][n][i] += __shfl_xor(acc[0][n][i], 32, 64);
          }
        }
      }
    };
    if (any) {
      if (FEW && (few || !MANY)) {
        if constexpr (FEW) run(std::integral_constant<int, 1>());
      } else {
        if constexpr (MANY) run(std::integral_constant<int, 4>());
      }
    }
    auto finish = [&](int m, int n, f32x4 v, f32x4 up) {
      const int64_t c = (int64_t)(ci * per_item + n) * kTile + col;
      if (c >= width) return;
      if constexpr (NT >= 2)
        if (p.swiglu)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = silu(v[i]) * up[i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (MT == 1 ? 4 * quad + i < min(left, lanes / PARTS) : 16 * m + 4 * quad + i < left)
          store(p, row0 + 16 * m + 4 * quad + i, c, width, v[i]);
    };
    if (split == 1) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (n < per_item) finish(m, n, acc[m][n], acc[m][NT >= 2 ? (n + NT / 2) % NT : n]);
      continue;
    }
#pragma unroll
    for (int n = 0; n < MT * NT; ++n) red[(wave * MT * NT + n) * 64 + lane] = acc[n / NT][n % NT];
    __syncthreads();
    auto total = [&](int n) {
      f32x4 v = red[((wave - ks) * MT * NT + n) * 64 + lane];
      for (int o = 1; o < split; ++o) v += red[((wave - ks + o) * MT * NT + n) * 64 + lane];
      return v;
    };
    if (any) {
      if constexpr (MT == 1) {
        for (int n = ks; n < per_item; n += split) {
          const f32x4 v = total(n);
          finish(0, n, v, p.swiglu ? total(n + NT / 2) : v);
        }
      } else {  // (dense: no SwiGLU)
        for (int n = ks; n < MT * NT; n += split) {
          const f32x4 v = total(n);
          finish(n / NT, n % NT, v, v);
        }
      }
    }
    __syncthreads();
  }
}

// One thread per 4 bytes of the packed weights.
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros,
                                                      int64_t K, int64_t N, int64_t KB, int64_t pairs, int64_t given,
                                                      int groups, int64_t words, uint32_t* out) {
  const int unit = (int)(block_bytes(groups, zeros != nullptr) / 4);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
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
}

// One thread per group and column: scale = bf16(largest magnitude / 7), code =
// round(w / scale) + 8.  A NaN in a group is its largest magnitude.
__global__ __launch_bounds__(256) void w4_quantize_kernel(const uint16_t* W, int64_t K, int64_t N, int group,
                                                          int64_t groups, int64_t count, uint8_t* codes,
                                                          uint16_t* scales) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i % N, g = i / N % groups, e = i / N / groups;
    const int64_t k0 = g * group, k1 = min(K, k0 + group);
    auto value = [&](int64_t k) { return __uint_as_float((uint32_t)W[(e * K + k) * N + n] << 16); };
    float most = 0.f;
    for (int64_t k = k0; k < k1; ++k) {
      const float v = fabsf(value(k));
      most = v > most || v != v ? v : most;  // (once NaN it stays: no comparison with it holds)
    }
    const __bf16 s = (__bf16)(most / 7.f);
    const float scale = (float)s;
    scales[i] = __builtin_bit_cast(uint16_t, s);
    for (int64_t k = k0; k < k1; ++k) {
      const float v = value(k), q = !(scale > 0.f) ? 0.f : isinf(v) ? v : rintf(v / scale);
      codes[(e * K + k) * N + n] = (uint8_t)((int)fminf(fmaxf(q, -8.f), 7.f) + 8);
    }
  }
}

unsigned blocks256(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, 1 << 22); }

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

hipError_t launch_w4(const W4KParams& args, int cus, hipStream_t stream) {
  if (args.M == 0) return hipSuccess;
  W4KParams p = args;
  using std::integral_constant;
  auto launch = [&](auto kernel, int nt, bool experts, int mt = 1) {
    const int w = group_waves(nt, mt), rows = 16 * mt / p.parts, per_item = p.swiglu ? nt / 2 : nt;
    p.passes = (uint32_t)((p.M + rows - 1) / rows);  // (experts: at most so many)
    const int64_t items = (int64_t)p.passes * ((p.tile_cols + per_item - 1) / per_item);
    const int64_t most = (int64_t)cus * waves_per_cu(nt, mt) / w;
    int64_t grid = std::min<int64_t>(items, most);
    if (!experts) {
      p.split = choose_split((uint32_t)items, (uint32_t)(most * w), (uint32_t)((p.w.K + kBlock - 1) / kBlock), w);
      grid = std::min<int64_t>(most, (items * p.split + w - 1) / w);
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * w), w * nt * mt * 64 * sizeof(f32x4), stream, p);
  };
  bool two_rows = false;
  auto go = [&](auto nt, auto sub, auto zeros) {
    constexpr int NT = decltype(nt)::value, SUB = decltype(sub)::value;
    constexpr bool Z = decltype(zeros)::value;
    if (!p.rb_expert) {
      if constexpr (NT == 1)
        if (p.M <= 4) return launch(w4_kernel<1, SUB, Z, 1, false, true, false, 1>, 1, false);
      if constexpr (NT == 4)
        if (two_rows) return launch(w4_kernel<4, SUB, Z, 1, false, false, true, 2>, 4, false, 2);
      launch(w4_kernel<NT, SUB, Z, 1, false, false, true, 1>, NT, false);
    } else if constexpr (NT != 1) {
      if (p.parts == 2) launch(w4_kernel<NT, SUB, Z, 2, true, true, true, 1>, NT, true);
      else launch(w4_kernel<NT, SUB, Z, 1, true, true, true, 1>, NT, true);
    }
  };
  auto with_zeros = [&](auto nt, auto sub) {
    if (p.w.zeros) go(nt, sub, std::true_type());
    else go(nt, sub, std::false_type());
  };
  auto with_group = [&](auto nt) {
    if (p.w.group == 32) with_zeros(nt, integral_constant<int, 1>());
    else if (p.w.group == 64) with_zeros(nt, integral_constant<int, 2>());
    else with_zeros(nt, integral_constant<int, 4>());
  };
  // Column tiles of an item.  Experts: four, or two (one gate, one up) where
  // SwiGLU's tiles are no whole pairs.  Dense up to 4 rows: one tile, and more
  // waves (1 x 8192 x 8192 8.6 us, with four tiles 11.2).  Dense with more rows:
  // x is read once per item and codes are expanded once per row tile or two, so
  // as many tiles an item as leave one for every CU.  Row tiles x column tiles,
  // and us with 1, 2, 4 column tiles an item and with 4 times two row tiles: 256
  // (32 x 3584 x 2048) 5.9, 6.3, 8.0; 320 (16 x 4096 x 5120) 7.9, 6.2, 8.1; 512
  // (64 x 7168 x 2048) 13.9, 9.3, 11.6; 640 (16 x 4096 x 10240) 12.3, 9.4, 8.6;
  // 1024 (32 x 3584 x 8192) -, 10.3, 8.2, 10.1; 1280 (64 x 3584 x 5120) -, -,
  // 12.2, 10.1; 2048 (64 x 3584 x 8192) -, 16.7, 13.6, 11.2.
  // (Measured with codes expanded to 128 + q, see expand().)
  const int64_t tiles = (p.M + 15) / 16 * p.tile_cols;
  const int wide = p.rb_expert ? (p.swiglu && p.tile_cols % 2 ? 2 : 4)
                   : p.M <= 4 || tiles <= cus ? 1 : tiles <= 2 * (int64_t)cus ? 2 : 4;
  two_rows = p.M > 16 && tiles > 4 * (int64_t)cus;
  if (wide == 1) with_group(integral_constant<int, 1>());
  else if (wide == 2) with_group(integral_constant<int, 2>());
  else with_group(integral_constant<int, 4>());
  return hipGetLastError();
}

}  // namespace mk
