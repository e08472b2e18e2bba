// mk_product.hip — the small kernels around the products (mk_product.h): rows laid
// out anew where their alignment does not allow 16-byte loads, the gradient of an
// activation with the bias's, and the join of the vocabulary's column groups.
// All are bound by the bytes they move.
#include "mk_product.h"

namespace mk {
namespace {

// One workgroup copies rows blockIdx.x * 4 .. of group blockIdx.y, a row per wave.
__global__ __launch_bounds__(256) void repack_kernel(RepackParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows || (p.counts && p.counts[blockIdx.y] <= 0)) return;
  const uint16_t* src = p.src + blockIdx.y * p.src_stride + row * p.ld;
  uint16_t* dst = p.dst + blockIdx.y * p.dst_stride + row * p.width * p.parts;
  bool off = false;
  if (p.labels)
    off = (p.labels64 ? static_cast<const int64_t*>(p.labels)[row] : static_cast<const int*>(p.labels)[row]) == p.ignore;
  const bool vec = !((reinterpret_cast<uintptr_t>(p.src) & 15) || p.ld % 8 || p.cols % 8 || p.src_stride % 8);
  for (int part = 0; part < p.parts; ++part, src += p.cols, dst += p.width) {
    for (int64_t c = lane * 8; c < p.width; c += 512) {
      uint32_t w[4] = {0, 0, 0, 0};
      if (!off) {
        if (vec) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + c);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
          // (eight 2-byte loads: lanes of a wave cover the same lines, which stay in L1)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < p.cols) w[i / 2] |= (uint32_t)src[c + i] << (16 * (i & 1));
        }
      }
      *reinterpret_cast<uint4*>(dst + c) = uint4{w[0], w[1], w[2], w[3]};
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
      if (p.dpre && col < p.width) store8(p.dpre, r * p.width + col, false, true, 8, d);
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

// lse = max + log sum of the column groups' (max, sum of exponentials) pairs: 32 tokens a workgroup, eight slices of
// the groups each, joined in order.
__global__ __launch_bounds__(256) void vocab_join_kernel(VocabJoinParams p) {
  __shared__ float2 part[8][32];
  const int tok = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t m = (int64_t)blockIdx.x * 32 + tok;
  float mx = -INFINITY, sum = 0.f;
  auto join = [&](float2 v) {
    const float to = fmaxf(mx, v.x);
    const float ref = to == -INFINITY ? 0.f : to;  // all of it -inf: sums are 0 (or NaN, which stays)
    sum = sum * __expf(mx - ref) + v.y * __expf(v.x - ref);
    mx = to;
  };
  if (m < p.T) {
    const int64_t g1 = (slice + 1) * p.groups / 8;
#pragma unroll 4
    for (int64_t g = slice * p.groups / 8; g < g1; ++g) join(p.stats[g * p.T + m]);
  }
  part[slice][tok] = float2{mx, sum};
  __syncthreads();
  if (slice != 0 || m >= p.T) return;
  for (int s = 1; s < 8; ++s) join(part[s][tok]);
  const int64_t l = p.labels64 ? static_cast<const int64_t*>(p.labels)[m] : static_cast<const int*>(p.labels)[m];
  const bool none = l == p.ignore, here = !none && l >= p.label0 && l - p.label0 < p.vocab;
  const float lse = none ? 0.f : mx + logf(sum), target = here ? p.target[m] : 0.f;
  p.lse[m] = lse;
  p.target[m] = target;
  if (p.loss) p.loss[m] = none ? 0.f : lse - target;
}

}  // namespace

hipError_t launch_repack(const RepackParams& p, hipStream_t stream) {
  if (p.rows == 0 || p.E == 0 || p.width == 0) return hipSuccess;
  hipLaunchKernelGGL(repack_kernel, dim3((unsigned)((p.rows + 3) / 4), (unsigned)p.E), dim3(256), 0, stream, p);
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
  hipLaunchKernelGGL(vocab_join_kernel, dim3((unsigned)((p.T + 31) / 32)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mk
