// mk_product.hip — the small kernels around the products (mk_product.h): rows laid
// out anew where their alignment does not allow 16-byte loads, the gradient of an
// activation with the bias's, and the join of the vocabulary's column groups.
// All are bound by the bytes they move.
#include "mk_product.h"

namespace mk {
namespace {

// 16 bytes that start at any element
typedef uint32_t words_at_any __attribute__((ext_vector_type(4), aligned(2)));

// ---------------------------------------------------------------------------
// One row or two against B [K, N], where latency counts (or B's rows allow no
// 16-byte loads): a workgroup has 32 or 64 columns and all of K, a wave's load
// covers 16 or 8 k-rows, so no sums cross workgroups and each lane's loads for
// 8 k-rows are in flight together.  Sums on the vector units: 8 columns a lane,
// then over the lanes of a column by shuffles, then over the waves through LDS.
// us in a graph, weights from HBM, against 32-row tiles with K in parts: 1 x 512 x
// 1024 3.9 and 6.1, 1 x 2048 x 2048 7.0 and 8.9, 2 x 1024 x 1024 about 6 and 7; a
// longer K turns it round (1 x 4096 x 4096 18.7 and 14.7: as many bytes in flight,
// but a workgroup's K goes through one CU), four rows too (4 x 2048 x 2048 10.9, 9.0).
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 8;

template <int ROWS, int COLS>
__global__ __launch_bounds__(64 * kFewWaves) void product_few_rows_kernel(ProductParams p) {
  __shared__ float sums[kFewWaves][ROWS][COLS];
  constexpr int LANES = COLS / 8, KROWS = 64 / LANES;  // lanes of a k-row, k-rows of a wave's load
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // each XCD has neighbouring columns
  const uint32_t n = gridDim.x, xcd = blockIdx.x & 7, id = xcd * (n >> 3) + min(xcd, n & 7) + (blockIdx.x >> 3);
  // the last columns' loads end with the row: a workgroup's columns start at col0, some of them its neighbour's
  const int64_t col0 = max<int64_t>(min<int64_t>((int64_t)id * COLS, p.N - COLS), 0);
  const int64_t col = min<int64_t>(col0 + lane % LANES * 8, p.N - 8);  // (N is 8 or more)
  float acc[ROWS][8];
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[m][c] = 0.f;
  // a lane has 8 neighbouring k-rows at a time, whose elements of A are one load
  constexpr int U = 8;
  for (int64_t k0 = (int64_t)(wave * KROWS + lane / LANES) * U; k0 < p.K; k0 += (int64_t)kFewWaves * KROWS * U) {
    words_at_any w[U], x[ROWS];
    const bool whole = k0 + U <= p.K;
#pragma unroll
    for (int u = 0; u < U; ++u)
      w[u] = *reinterpret_cast<const words_at_any*>(p.B + (whole ? k0 + u : min(k0 + u, p.K - 1)) * p.ldb + col);
    if (whole) {
#pragma unroll
      for (int m = 0; m < ROWS; ++m) x[m] = *reinterpret_cast<const words_at_any*>(p.A + min<int64_t>(m, p.M - 1) * p.lda + k0);
    } else {
      // k-rows behind the last are zeros on both sides
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k0 + u >= p.K) w[u] = words_at_any{0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        x[m] = words_at_any{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (k0 + u < p.K) x[m][u / 2] |= (uint32_t)p.A[min<int64_t>(m, p.M - 1) * p.lda + k0 + u] << (16 * (u & 1));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        const float a = u & 1 ? bf16_hi(x[m][u / 2]) : bf16_lo(x[m][u / 2]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[m][2 * i] += a * bf16_lo(w[u][i]);
          acc[m][2 * i + 1] += a * bf16_hi(w[u][i]);
        }
      }
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int d = LANES; d < 64; d <<= 1) acc[m][c] += __shfl_xor(acc[m][c], d, 64);
      if (lane < LANES) sums[wave][m][col - col0 + c] = acc[m][c];  // (lanes of one column have the same sum)
    }
  __syncthreads();
  if (threadIdx.x >= ROWS * COLS) return;
  const int m = threadIdx.x / COLS, c = threadIdx.x % COLS;
  const int64_t at = col0 + c;
  if (m >= p.M || at < (int64_t)id * COLS || at >= p.N) return;  // a neighbour has its columns
  float x = 0.f;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) x += sums[w][m][c];
  auto get = [](const void* q, int64_t i, int f32) {
    return f32 ? static_cast<const float*>(q)[i] : __uint_as_float((uint32_t)static_cast<const uint16_t*>(q)[i] << 16);
  };
  if (p.bias) x += get(p.bias, at, p.bias_f32);
  if (p.pre) p.pre[m * p.ldp + at] = (uint16_t)pack_bf16x2(x, 0.f);
  if (p.act) for_act(p.act, [&](auto a_) { x = act_of<decltype(a_)::value>(x); });
  if (p.res) x += get(p.res, m * p.ldr + at, p.res_f32);
  if (p.c_f32) static_cast<float*>(p.C)[m * p.ldc + at] = x;
  else static_cast<uint16_t*>(p.C)[m * p.ldc + at] = (uint16_t)pack_bf16x2(x, 0.f);
}

// Whether a token has no loss.
__device__ __forceinline__ bool ignored(const RepackParams& p, int64_t row) {
  return (p.labels64 ? static_cast<const int64_t*>(p.labels)[row] : static_cast<const int*>(p.labels)[row]) == p.ignore;
}

// A wave copies 512 columns of a row; one workgroup four rows of group blockIdx.z, columns from 2048 * blockIdx.y on.
// (Loads of single elements moved 1.4 TB/s, a 1024 x 5003 matrix in 14.3 us.)
// The first workgroup finds the scale of dloss too (4096 tokens 24 us, 12.6 without).
__global__ __launch_bounds__(256) void repack_kernel(RepackParams p) {
  const int lane = threadIdx.x & 63;
  if (p.scale && blockIdx.x == 0 && blockIdx.y == 0) {
    __shared__ uint32_t largest[4];
    uint32_t most = 0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < p.rows; i += 256) {
      const uint32_t b = __float_as_uint(p.dloss[i]) & 0x7fffffffu;
      if (b < 0x7f800000u && !ignored(p, i)) most = max(most, b);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
    if (lane == 0) largest[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      most = max(max(largest[0], largest[1]), max(largest[2], largest[3]));
      *p.scale = most < 0x00800000u ? 1.f : __uint_as_float((most & 0x007fffffu) | 0x3f800000u);
    }
  }
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows || (p.counts && p.counts[blockIdx.z] <= 0)) return;
  const uint16_t* src = p.src + blockIdx.z * p.src_stride + row * p.ld;
  uint16_t* dst = p.dst + blockIdx.z * p.dst_stride + row * p.width * p.parts;
  bool off = false;
  if (p.labels) off = ignored(p, row);
  for (int part = 0; part < p.parts; ++part, src += p.cols, dst += p.width) {
    words_at_any w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = blockIdx.y * 2048 + u * 512 + lane * 8;
      w[u] = words_at_any{0, 0, 0, 0};
      if (off || c >= p.cols) continue;
      if (c + 8 <= p.cols) {
        w[u] = *reinterpret_cast<const words_at_any*>(src + c);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.cols) w[u][i / 2] |= (uint32_t)src[c + i] << (16 * (i & 1));
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = blockIdx.y * 2048 + u * 512 + lane * 8;
      if (c < p.width) *reinterpret_cast<uint4*>(dst + c) = uint4{w[u][0], w[u][1], w[u][2], w[u][3]};
    }
  }
}

constexpr int kGradCols = 512;  // columns of a workgroup: 8 per lane of each of its four waves

// Rows blockIdx.y of row_blocks, 512 columns: dpre, and the columns' sums over the rows in fp32, rows of a wave in
// order, then the four waves.
__global__ __launch_bounds__(256) void act_grad_kernel(ActGradParams p) {
  __shared__ float sums[4][kGradCols];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * kGradCols + lane * 8;
  const int nc = (int)min<int64_t>(max<int64_t>(p.N - col, 0), 8);
  const int64_t r0 = blockIdx.y * p.M / p.row_blocks, r1 = (blockIdx.y + 1) * p.M / p.row_blocks;
  float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for_act(p.act, [&](auto a_) {
    constexpr int ACT = decltype(a_)::value;
    for (int64_t r = r0 + wave; r < r1; r += 4) {
      float d[8], x[8];
      load8(p.dC, r * p.ldc + col, false, p.vec_c, nc, d);
      if constexpr (ACT != kActNone) {
        load8(p.pre, r * p.ldp + col, false, p.vec_p, nc, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= act_slope<ACT>(x[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= nc) d[i] = 0.f;
        s[i] += d[i];
      }
      if (!p.dpre || col >= p.width) continue;
      store8(p.dpre, r * p.width + col, true, 8, d);
      for (int t = 1; t < p.terms; ++t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = bf16_rest(d[i]);
        store8(p.dpre, (t * p.M + r) * p.width + col, true, 8, d);
      }
    }
  });
  if (!p.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[wave][lane * 8 + i] = s[i];
  __syncthreads();
  for (int c = threadIdx.x; c < kGradCols; c += 256) {
    const int64_t at = (int64_t)blockIdx.x * kGradCols + c;
    if (at < p.N) p.part[blockIdx.y * p.N + at] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
  }
}

// 64 columns a workgroup: each wave adds a quarter of the row blocks, then the four.
__global__ __launch_bounds__(256) void column_sums_kernel(const float* part, int64_t blocks, int64_t N, float* out,
                                                          int accumulate) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < N) {
    const int64_t b1 = (wave + 1) * blocks / 4;
#pragma unroll 8
    for (int64_t b = wave * blocks / 4; b < b1; ++b) s += part[b * N + c];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < N) {
    const float v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    out[c] = accumulate ? out[c] + v : v;
  }
}

constexpr int kJoinTokens = 16, kJoinSlices = 32;

// lse = max + log sum of the column groups' (max, sum of exponentials) pairs: 16 tokens a workgroup (a line of pairs),
// 32 slices of the groups each, joined in order.
__global__ __launch_bounds__(512) void vocab_join_kernel(VocabJoinParams p) {
  __shared__ float2 part[kJoinSlices][kJoinTokens];
  const int tok = threadIdx.x % kJoinTokens, slice = threadIdx.x / kJoinTokens;
  const int64_t m = (int64_t)blockIdx.x * kJoinTokens + tok;
  float2 s = {-INFINITY, 0.f};
  if (m < p.T) {
    const int64_t g1 = (slice + 1) * p.groups / kJoinSlices;
#pragma unroll 8
    for (int64_t g = slice * p.groups / kJoinSlices; g < g1; ++g) s = join_stats(s, p.stats[g * p.T + m]);
  }
  part[slice][tok] = s;
  __syncthreads();
  if (slice != 0 || m >= p.T) return;
  for (int i = 1; i < kJoinSlices; ++i) s = join_stats(s, part[i][tok]);
  const int64_t l = p.labels64 ? static_cast<const int64_t*>(p.labels)[m] : static_cast<const int*>(p.labels)[m];
  const bool none = l == p.ignore, here = !none && l >= p.label0 && l - p.label0 < p.vocab;
  const float lse = none ? 0.f : s.x + logf(s.y), target = here ? p.target[m] : 0.f;
  p.lse[m] = lse;
  p.target[m] = target;
  if (p.loss) p.loss[m] = none ? 0.f : lse - target;
}

}  // namespace

hipError_t launch_product_few_rows(const ProductParams& p, hipStream_t stream) {
  // 64 columns where that is a workgroup for every CU: whole lines (1 x 512 x 16384 10.4 us with 32, 7.0 with 64;
  // 1 x 2048 x 2048 7.0 and 7.2)
  const bool wide = p.N >= 64 * 256;
  const int cols = wide ? 64 : 32;
  const dim3 grid((unsigned)((p.N + cols - 1) / cols)), block(64 * kFewWaves);
  if (p.M == 1 && wide) hipLaunchKernelGGL((product_few_rows_kernel<1, 64>), grid, block, 0, stream, p);
  else if (p.M == 1) hipLaunchKernelGGL((product_few_rows_kernel<1, 32>), grid, block, 0, stream, p);
  else if (wide) hipLaunchKernelGGL((product_few_rows_kernel<2, 64>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((product_few_rows_kernel<2, 32>), grid, block, 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_repack(const RepackParams& p, hipStream_t stream) {
  if (p.rows == 0 || p.E == 0 || p.width == 0) return hipSuccess;
  hipLaunchKernelGGL(repack_kernel, dim3((unsigned)((p.rows + 3) / 4), (unsigned)((p.width + 2047) / 2048), (unsigned)p.E),
                     dim3(256), 0, stream, p);
  return hipGetLastError();
}

// enough workgroups to fill the chip, at least 16 rows each
int64_t act_grad_blocks(int64_t M, int64_t N) {
  const int64_t cols = (N + kGradCols - 1) / kGradCols, want = (1024 + cols - 1) / std::max<int64_t>(cols, 1);
  return std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 256), M / 16));
}

hipError_t launch_act_grad(const ActGradParams& p, hipStream_t stream) {
  if (p.N == 0) return hipSuccess;
  const int64_t width = std::max(p.N, p.dpre ? p.width : 0);
  hipLaunchKernelGGL(act_grad_kernel, dim3((unsigned)((width + kGradCols - 1) / kGradCols), (unsigned)p.row_blocks),
                     dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.part) return e;
  hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((p.N + 63) / 64)), dim3(256), 0, stream, p.part, p.row_blocks,
                     p.N, p.dbias, p.accumulate);
  return hipGetLastError();
}

hipError_t launch_vocab_join(const VocabJoinParams& p, hipStream_t stream) {
  if (p.T == 0) return hipSuccess;
  hipLaunchKernelGGL(vocab_join_kernel, dim3((unsigned)((p.T + kJoinTokens - 1) / kJoinTokens)), dim3(kJoinTokens * kJoinSlices), 0,
                     stream, p);
  return hipGetLastError();
}

}  // namespace mk
