// mk_w4.hip — products of a few rows with 4-bit weights and group scales
// (gfx950): dense, and for the routed experts of a small batch.
//
//   y[m, n] = sum_k x[m, k] * (q[k, n] - z[g(k), n]) * s[g(k), n]
//
// q in 0 .. 15, z 8 or a zero point, s bf16 per `group` rows of K.  Weights lie
// in the order in which the matrix instruction reads them: a 16-byte unit per
// lane holds the 32 codes that lane feeds to four 16 x 16 x 32 MFMAs (16
// columns, 128 rows of K), so a wave reads 1 KB in one piece and nothing goes
// through LDS on the way in.
//
// A code becomes the bf16 number 128 + q by setting bits (0x4300 | q, exact);
// the product with the constant -(128 + z) is one more MFMA into the same
// accumulator.  A group's sum of x * (q - z) is then multiplied with its scale
// in fp32: no rounding but the fp32 sums' and the one of the result.
//
// The weights are the first operand, so a lane of the result holds four
// neighbouring columns of one row of x.  The waves of a workgroup share a
// column tile and split K; their sums meet in LDS in wave order.
#include <algorithm>
#include <type_traits>

#include "mk_device.h"
#include "mk_internal.h"

#ifndef W4_NT
#define W4_NT 1
#define W4_W 8
#define W4_NT2 4
#define W4_W2 8
#define W4_P1 3
#endif
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

// What one step of 128 rows of K needs: packed codes, scales (of this lane's
// four columns, group by group), zero points (of its one column) and x.
template <int MT, int NT, int SUB, bool ZEROS>
struct Step {
  u32x4 w[NT];
  uint32_t s[NT][2 * (4 / SUB)];
  uint32_t z[ZEROS ? NT : 1];
  u32x4 x[MT][4];
};

// Descriptors of a wave's column tiles (each tile's codes, scales and zeros are
// one piece) and of its rows of x.
template <int MT, int NT>
struct Source {
  __amdgpu_buffer_rsrc_t w[NT], x;
  const char* s[NT];
  const uint8_t* z[NT];
  uint32_t last;     // last step
  uint32_t row[MT];  // byte offset of this lane's row, kNowhere where there is none
  int32_t most;      // last multiple of 8 below K, less this lane's first k in a step
};

template <int MT, int NT, int SUB, bool ZEROS>
__device__ __forceinline__ void load(Step<MT, NT, SUB, ZEROS>& st, const Source<MT, NT>& t, uint32_t kb, int lane) {
  constexpr int G = 4 / SUB;
  // scales past the last step are the last one's: they multiply zeros
  const uint32_t sb = min(kb, t.last);
  const uint32_t at = sb * (32 * G) + (lane >> 4) * (8 * G), zt = sb * (16 * G) + (lane & 15) * G;
#pragma unroll
  for (int n = 0; n < NT; ++n) st.w[n] = load16(t.w[n], kb * 1024 + lane * 16);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    typedef uint32_t words __attribute__((ext_vector_type(G == 4 ? 4 : 2 * G)));
#pragma unroll
    for (int h = 0; h < (G == 4 ? 2 : 1); ++h) {
      const words v = *reinterpret_cast<const words*>(t.s[n] + at + 16 * h);
#pragma unroll
      for (int i = 0; i < (G == 4 ? 4 : 2 * G); ++i) st.s[n][4 * h + i] = v[i];
    }
    if constexpr (ZEROS) {
      if constexpr (G == 1) st.z[n] = t.z[n][zt];
      else if constexpr (G == 2) st.z[n] = *reinterpret_cast<const uint16_t*>(t.z[n] + zt);
      else st.z[n] = *reinterpret_cast<const uint32_t*>(t.z[n] + zt);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = (int32_t)(kb * kBlock) + j * 32 <= t.most;
#pragma unroll
    for (int m = 0; m < MT; ++m) st.x[m][j] = load16(t.x, in ? t.row[m] + kb * 256 + 64 * j : kNowhere);
  }
}

template <int MT, int NT, int SUB, bool ZEROS>
__device__ __forceinline__ void multiply(const Step<MT, NT, SUB, ZEROS>& st, uint32_t mask, uint32_t bias,
                                         f32x4 (&acc)[NT][MT]) {
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
          base[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(off, __builtin_bit_cast(bf16x8, st.x[m][g * SUB + i]), base[m], 0, 0, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 part[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) part[m] = ZEROS ? f32x4{0.f, 0.f, 0.f, 0.f} : base[m];
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const bf16x8 q = expand(st.w[n][g * SUB + i], mask, bias);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const bf16x8 xv = __builtin_bit_cast(bf16x8, st.x[m][g * SUB + i]);
          if constexpr (ZEROS)
            part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(minus_offset((st.z[n] >> (8 * g)) & 255u), xv, part[m], 0, 0, 0);
          part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q, xv, part[m], 0, 0, 0);
        }
      }
      const f32x4 s = {bf16_lo(st.s[n][2 * g]), bf16_hi(st.s[n][2 * g]), bf16_lo(st.s[n][2 * g + 1]), bf16_hi(st.s[n][2 * g + 1])};
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[n][m][r] = fmaf(s[r], part[m][r], acc[n][m][r]);
    }
  }
}

// The steps kb = first, first + stride, ... of a wave's tiles and rows: a ring
// of P steps in registers.  The barriers keep a step's loads behind the step
// before, in order: loads return in the order of their issue, so a step waits
// for its own only.  The last P steps load nothing more (a load that nobody
// needs would still be waited for before its registers are used again); those
// past the end found zeros.
template <int MT, int NT, int SUB, bool ZEROS, int P>
__device__ __forceinline__ void sweep(const Source<MT, NT>& t, uint32_t KB, uint32_t first, uint32_t stride, int lane,
                                      f32x4 (&acc)[NT][MT]) {
  uint32_t mask = 0x000f000fu, bias = 0x43004300u;
  asm volatile("" : "+s"(mask));
  asm volatile("" : "+v"(bias));
  Step<MT, NT, SUB, ZEROS> st[P];
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
      multiply(st[i], mask, bias, acc);
      __builtin_amdgcn_sched_barrier(0);
      load(st[i], t, kb + (i + P) * stride, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) multiply(st[i], mask, bias, acc);
}

// One unit of the result: 16 columns of 16 rows, this lane's four columns `c` ..
// of row `r`.
__device__ __forceinline__ void store(const W4KParams& p, int64_t r, int64_t c, int64_t width, f32x4 v) {
  if (p.out_type == kW4F32) {
    float* out = static_cast<float*>(p.C) + r * p.ldc + c;
    if (c + 4 <= width && p.ldc % 4 == 0) {
      *reinterpret_cast<f32x4*>(out) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < width) out[i] = v[i];
    }
    return;
  }
  uint16_t* out = static_cast<uint16_t*>(p.C) + r * p.ldc + c;
  for (int h = 0; h < (p.out_type == kW4Pair ? 2 : 1); ++h) {
    const u32x2 o = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    if (c + 4 <= width && p.ldc % 4 == 0 && width % 4 == 0) {
      *reinterpret_cast<u32x2*>(out) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < width) out[i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
    }
    // what the rounding left, in the second half of the row
    v = f32x4{v[0] - bf16_lo(o[0]), v[1] - bf16_hi(o[0]), v[2] - bf16_lo(o[1]), v[3] - bf16_hi(o[1])};
    out += width;
  }
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

// The row passes of the real rows of up to kListed row blocks: 16 rows each, or
// 8 where x goes as bf16 pairs, whose second halves take the other 8 lanes (the
// two sums of a row are added at the end).
constexpr int kListed = 512;
template <int ROWS>
struct PassList {
  int first[kListed + 1];                        // first pass of each block
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

// W waves.  An item is NT column tiles (with SwiGLU: the first half gate tiles,
// the second the matching up tiles) of 16 MT rows; `split` waves share its K.
// The workgroups of the grid walk the items in turn, as many as the device's
// row count and tables say there are.
template <int MT, int NT, int W, int SUB, bool ZEROS, int PARTS, bool EXPERTS>
__global__ __launch_bounds__(64 * W) void w4_kernel(W4KParams p) {
  extern __shared__ f32x4 red[];  // [W][NT * MT][64], used where K is split
  constexpr int ROWS = PARTS == 2 ? 8 : 16, kPasses = kFlagRows / ROWS;  // of a pass over experts' rows
  __shared__ PassList<ROWS> list;
  static_assert(MT == 1 || (!EXPERTS && PARTS == 1), "passes of 16 rows");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const uint32_t KB = (uint32_t)((p.w.K + kBlock - 1) / kBlock);
  const int tiles = (int)((p.w.N + kTile - 1) / kTile);
  const int64_t groups = (int64_t)KB * (4 / SUB);
  const int per_item = p.swiglu ? NT / 2 : NT;  // output tiles
  const int col_items = (p.tile_cols + per_item - 1) / per_item;
  const int64_t width = p.swiglu ? (int64_t)p.tile_cols * kTile : p.w.N;
  int blocks = p.row_blocks;
  uint32_t passes = p.row_blocks;
  bool listed = false;
  if constexpr (EXPERTS) {
    if (p.rows_dev) blocks = (int)min((int64_t)blocks, max((int64_t)0, *p.rows_dev / kFlagRows));
    listed = blocks <= kListed;
    passes = blocks * kPasses;
    if (listed) {
      constexpr int per = kListed / (64 * W) > 0 ? kListed / (64 * W) : 1;
      int n[per], sum = 0;
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const int b = threadIdx.x * per + i;
        n[i] = b < blocks ? (block_rows(p, b) + ROWS - 1) / ROWS : 0;
        sum += n[i];
      }
      int at = prefix<W>(sum, list.scratch);
      if (threadIdx.x == 64 * W - 1) list.scratch[16] = at;
      at -= sum;
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const int b = threadIdx.x * per + i;
        if (b <= kListed) list.first[b] = at;
        for (int j = 0; j < n[i]; ++j) list.block[at + j] = (uint16_t)b;
        at += n[i];
      }
      if (threadIdx.x == 64 * W - 1) list.first[kListed] = at;
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
      if constexpr (EXPERTS) {
        // the passes of one column item side by side: they read the same weights
        uint32_t q = it / col_items;
        int np = kPasses, pass, b;
        if (listed) {
          b = __builtin_amdgcn_readfirstlane((int)list.block[q]);
          const int first = __builtin_amdgcn_readfirstlane(list.first[b]);
          np = __builtin_amdgcn_readfirstlane(list.first[b + 1]) - first;
          q = first;
        } else {
          b = q / kPasses;
          q = b * kPasses;
        }
        const int local = (int)(it - q * col_items);
        ci = local / np;
        pass = local - ci * np;
        left = __builtin_amdgcn_readfirstlane(block_rows(p, b)) - ROWS * pass;
        expert = __builtin_amdgcn_readfirstlane(p.rb_expert[b]);
        row0 = (int64_t)b * kFlagRows + ROWS * pass;
      } else {
        const uint32_t b = it / col_items;
        ci = (int)(it - b * col_items);
        row0 = (int64_t)b * 16 * MT;
        left = (int)min(p.M - row0, (int64_t)16 * MT);
      }
    }
    Source<MT, NT> t;
    int tile[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool up = p.swiglu && n >= NT / 2;
      tile[n] = min(ci * per_item + (up ? n - NT / 2 : n), p.tile_cols - 1) + (up ? p.tile_cols : 0);
      const int64_t at = left > 0 ? expert * tiles + tile[n] : 0;
      t.w[n] = make_rsrc(p.w.packed + at * KB * 256, KB * 1024);
      t.s[n] = reinterpret_cast<const char*>(p.w.scales + at * groups * kTile);
      if constexpr (ZEROS) t.z[n] = p.w.zeros + at * groups * kTile;
    }
    t.last = KB - 1;
    t.most = (int32_t)p.w.K - 8 - quad * 8;
    // lanes past the last row read nothing; their results are not stored
    if (EXPERTS && p.gather_pull) {
      t.x = make_rsrc(p.A, (uint32_t)(p.gather_rows * p.lda * 2));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        t.row[m] = kNowhere;
        if (16 * m + col < left) {
          const int* pr = p.gather_pull + 3 * (row0 + 16 * m + col);
          const int64_t src = ((int64_t)pr[0] * p.gather_devs + pr[1]) * p.gather_tps + pr[2];
          if (pr[0] >= 0 && pr[2] >= 0 && src >= 0 && src < p.gather_rows) t.row[m] = (uint32_t)(src * p.lda * 2) + quad * 16;
        }
      }
    } else {
      t.x = make_rsrc(p.A + row0 * p.lda, (uint32_t)(min(max(left, 0), 16 * MT) * p.lda * 2));
      const int r = PARTS == 2 ? col & 7 : col;
#pragma unroll
      for (int m = 0; m < MT; ++m)
        t.row[m] = 16 * m + r < left ? (uint32_t)((16 * m + r) * p.lda * 2 + (r < col ? 2 * p.w.K : 0)) + quad * 16 : kNowhere;
    }
    f32x4 acc[NT][MT];
    sweep<MT, NT, SUB, ZEROS, (MT * NT == 1 ? W4_P1 : 2)>(t, KB, left > 0 ? ks : KB, split, lane, acc);
    auto finish = [&](int n, int m, f32x4 v, f32x4 up) {
      if constexpr (PARTS == 2) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] += __shfl_xor(v[r], 8, 64);
          up[r] += __shfl_xor(up[r], 8, 64);
        }
        if (col >= 8) return;
      }
      if (16 * m + col >= left || ci * per_item + n >= p.tile_cols) return;
      if constexpr (NT >= 2)
        if (p.swiglu)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = silu(v[r]) * up[r];
      store(p, row0 + 16 * m + col, (int64_t)(ci * per_item + n) * kTile + 4 * quad, width, v);
    };
    if (split == 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (n < per_item) finish(n, m, acc[n][m], acc[NT >= 2 ? (n + NT / 2) % NT : n][m]);
      continue;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) red[(wave * NT * MT + n * MT + m) * 64 + lane] = acc[n][m];
    __syncthreads();
    auto total = [&](int u) {
      f32x4 v = red[((wave - ks) * NT * MT + u) * 64 + lane];
      for (int o = 1; o < split; ++o) v += red[((wave - ks + o) * NT * MT + u) * 64 + lane];
      return v;
    };
    for (int u = ks; u < per_item * MT; u += split) {
      const f32x4 v = total(u);
      finish(u / MT, u % MT, v, p.swiglu ? total(u + (NT / 2) * MT) : v);
    }
    __syncthreads();
  }
}

template <int MT, int NT, int W, int SUB, bool ZEROS, int PARTS, bool EXPERTS>
void launch(const W4KParams& p, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((w4_kernel<MT, NT, W, SUB, ZEROS, PARTS, EXPERTS>), dim3(grid), dim3(64 * W),
                     W * NT * MT * 64 * sizeof(f32x4), stream, p);
}

__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* codes, int64_t K, int64_t N, int64_t KB,
                                                      int64_t tiles, int64_t words, uint32_t* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= words) return;
  const int j = (int)(i & 3), lane = (int)((i >> 2) & 63);
  const int64_t block = i >> 8, kb = block % KB, tile = block / KB % tiles, e = block / KB / tiles;
  const int64_t n = tile * kTile + (lane & 15), k0 = kb * kBlock + j * 32 + (lane >> 4) * 8;
  uint32_t w = 0;
#pragma unroll
  for (int o = 0; o < 8; ++o) {
    const int64_t k = k0 + o;
    const uint32_t q = k < K && n < N ? codes[(e * K + k) * N + n] & 15u : 8u;
    w |= q << (4 * ((o & 1) * 4 + (o >> 1)));
  }
  out[i] = w;
}

__global__ __launch_bounds__(256) void w4_pack_groups_kernel(const uint16_t* scales, const uint8_t* zeros, int64_t N,
                                                             int64_t given, int64_t groups, int per, int64_t tiles,
                                                             int64_t count, uint16_t* out_scales, uint8_t* out_zeros) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  // scales: [tile][block][4 quads][per block][4 columns]; zeros: [tile][block][16 columns][per block]
  const int64_t unit = kTile * per, block = i / unit, in_block = i % unit;
  const int64_t kb = block % (groups / per), tile = block / (groups / per) % tiles, e = block / (groups / per) / tiles;
  auto source = [&](int64_t g, int64_t n) {
    return g < given && n < N ? (e * given + g) * N + n : (int64_t)-1;
  };
  const int64_t at = source(kb * per + in_block / 4 % per, tile * kTile + in_block / (4 * per) * 4 + in_block % 4);
  out_scales[i] = at >= 0 ? scales[at] : 0;
  if (out_zeros) {
    const int64_t zt = source(kb * per + in_block % per, tile * kTile + in_block / per);
    out_zeros[i] = zt >= 0 ? zeros[zt] & 15u : 8u;
  }
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

int64_t w4_packed_words(int64_t K, int64_t N, int64_t E) {
  return E * ((N + kTile - 1) / kTile) * ((K + kBlock - 1) / kBlock) * 256;
}

int64_t w4_scale_count(int64_t K, int64_t N, int64_t E, int group) {
  return E * ((N + kTile - 1) / kTile) * ((K + kBlock - 1) / kBlock) * (kBlock / group) * kTile;
}

hipError_t launch_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int64_t K, int64_t N,
                          int64_t E, int group, uint32_t* packed, uint16_t* packed_scales, uint8_t* packed_zeros,
                          hipStream_t stream) {
  const int64_t KB = (K + kBlock - 1) / kBlock, tiles = (N + kTile - 1) / kTile;
  const int64_t words = w4_packed_words(K, N, E), count = w4_scale_count(K, N, E, group);
  hipLaunchKernelGGL(w4_pack_kernel, dim3(blocks256(words)), dim3(256), 0, stream, codes, K, N, KB, tiles, words, packed);
  hipLaunchKernelGGL(w4_pack_groups_kernel, dim3(blocks256(count)), dim3(256), 0, stream, scales, zeros, N,
                     (K + group - 1) / group, KB * (kBlock / group), kBlock / group, tiles, count, packed_scales, packed_zeros);
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
    const int passes = decltype(ex)::value ? kFlagRows / (decltype(parts)::value == 2 ? 8 : 16) : 1;
    const int64_t items = (int64_t)p.row_blocks * passes * ((p.tile_cols + per_item - 1) / per_item);
    const int64_t most = (int64_t)cus * waves_per_cu(MT, NT) / W;
    int64_t grid = std::min<int64_t>(items, most);
    if (!decltype(ex)::value) {
      p.split = choose_split((uint32_t)items, (uint32_t)(most * W), (uint32_t)((p.w.K + kBlock - 1) / kBlock), W);
      grid = std::min<int64_t>(most, (items * p.split + W - 1) / W);
    }
    launch<MT, NT, W, decltype(sub)::value, decltype(zeros)::value, decltype(parts)::value, decltype(ex)::value>(
        p, (int)grid, stream);
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
    if (p.parts == 2) with_group(one, four, four, two, std::true_type());
    else with_group(one, four, four, one, std::true_type());
  } else if (p.M <= 16) {
    with_group(one, integral_constant<int, W4_NT>(), integral_constant<int, W4_W>(), one, std::false_type());
  } else {
    with_group(two, integral_constant<int, W4_NT2>(), integral_constant<int, W4_W2>(), one, std::false_type());
  }
  return hipGetLastError();
}

}  // namespace mk
