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

namespace mk {
namespace {

constexpr int kTile = 16;    // columns of a tile
constexpr int kBlock = 128;  // rows of K of a 16-byte unit per lane

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight codes of one word as bf16 128 + q: nibbles i and i + 4 are elements
// 2i and 2i + 1.
__device__ __forceinline__ bf16x8 expand(uint32_t w) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
  return __builtin_bit_cast(bf16x8, v);
}

// All eight elements bf16 -(128 + z), z in 0 .. 127.
__device__ __forceinline__ bf16x8 minus_offset(uint32_t z) {
  const uint32_t h = 0xc300u | z, hh = h | h << 16;
  return __builtin_bit_cast(bf16x8, (u32x4{hh, hh, hh, hh}));
}

__device__ __forceinline__ float silu(float x) { return x / (1.f + __expf(-x)); }

// MT tiles of 16 rows of x, NT weight tiles (2 with SwiGLU: gate and up), W
// waves, SUB 32-row steps of K per scale.
template <int MT, int NT, int W, int SUB, bool ZEROS>
__global__ __launch_bounds__(64 * W) void w4_kernel(W4KParams p) {
  extern __shared__ f32x4 red[];  // [W][NT][MT][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, quad = lane >> 4;
  const int64_t KB = (p.w.K + kBlock - 1) / kBlock, tiles = (p.w.N + kTile - 1) / kTile;
  const int64_t groups = KB * (4 / SUB);

  // rows of this workgroup
  int64_t row0 = (int64_t)blockIdx.y * 16 * MT, rows = p.M - row0;
  int64_t expert = 0;
  if (p.rb_expert) {
    const int64_t b = blockIdx.y / (kFlagRows / (16 * MT)), part = blockIdx.y % (kFlagRows / (16 * MT));
    if (b * kFlagRows >= (p.rows_dev ? min(p.M, *p.rows_dev) : p.M)) return;
    expert = p.rb_expert[b];
    if (expert < 0 || expert >= p.w.E) return;
    rows = (p.rb_rows ? min(p.rb_rows[b], kFlagRows) : kFlagRows) - part * 16 * MT;
    row0 = b * kFlagRows + part * 16 * MT;
  }
  if (rows <= 0) return;
  rows = min(rows, (int64_t)16 * MT);

  // this lane's row of x in each row tile; lanes past the last row read it
  // again, and their results are not stored
  const uint16_t* x[MT];
  bool have[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t r = row0 + min(rows - 1, (int64_t)16 * m + col);
    int64_t src = r;
    have[m] = true;
    if (p.gather_pull) {
      const int* pr = p.gather_pull + 3 * r;
      src = ((int64_t)pr[0] * p.gather_devs + pr[1]) * p.gather_tps + pr[2];
      have[m] = pr[0] >= 0 && src >= 0 && src < p.gather_rows;
      if (!have[m]) src = 0;
    }
    x[m] = p.A + src * p.lda;
  }
  int64_t tile[NT];
  tile[0] = blockIdx.x * (p.swiglu ? 1 : NT);
  if constexpr (NT == 2) tile[1] = p.swiglu ? tile[0] + p.tile_cols : min(tile[0] + 1, tiles - 1);

  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int64_t kb = wave; kb < KB; kb += W) {
    u32x4 w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      w[n] = *reinterpret_cast<const u32x4*>(p.w.packed + (((expert * tiles + tile[n]) * KB + kb) * 64 + lane) * 4);
    bf16x8 xv[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t k = kb * kBlock + j * 32 + quad * 8;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (k < p.w.K && have[m]) v = *reinterpret_cast<const u32x4*>(x[m] + k);
        xv[m][j] = __builtin_bit_cast(bf16x8, v);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int g = 0; g < 4 / SUB; ++g) {
        const int64_t at = ((expert * tiles + tile[n]) * groups + kb * (4 / SUB) + g) * kTile;
        const u32x2 sw = *reinterpret_cast<const u32x2*>(p.w.scales + at + 4 * quad);
        const bf16x8 off = minus_offset(ZEROS ? p.w.zeros[at + col] : 8u);
        const f32x4 s = {bf16_lo(sw[0]), bf16_hi(sw[0]), bf16_lo(sw[1]), bf16_hi(sw[1])};
        f32x4 part[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) part[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
          const bf16x8 q = expand(w[n][g * SUB + i]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(off, xv[m][g * SUB + i], part[m], 0, 0, 0);
            part[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q, xv[m][g * SUB + i], part[m], 0, 0, 0);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[n][m][r] = fmaf(s[r], part[m][r], acc[n][m][r]);
      }
  }

#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) red[((wave * NT + n) * MT + m) * 64 + lane] = acc[n][m];
  __syncthreads();
  auto total = [&](int n, int m) {
    f32x4 v = red[(n * MT + m) * 64 + lane];
#pragma unroll
    for (int o = 1; o < W; ++o) v += red[((o * NT + n) * MT + m) * 64 + lane];
    return v;
  };
  const int64_t width = p.swiglu ? (int64_t)p.tile_cols * kTile : p.w.N;
  const int units = p.swiglu ? MT : NT * MT;
  for (int u = wave; u < units; u += W) {
    const int m = u % MT, n = u / MT;
    if (16 * m + col >= rows) continue;
    f32x4 v = total(n, m);
    if constexpr (NT == 2)
      if (p.swiglu) {
        const f32x4 up = total(1, m);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = silu(v[r]) * up[r];
      }
    if (!p.swiglu && tile[0] + n >= tiles) continue;
    const int64_t c = (tile[0] + n) * kTile + 4 * quad;
    uint16_t* out = p.C + (row0 + 16 * m + col) * p.ldc + c;
    if (c + 4 <= width && p.ldc % 4 == 0) {
      *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (c + r < width) out[r] = __builtin_bit_cast(uint16_t, (__bf16)v[r]);
    }
  }
}

template <int MT, int NT, int SUB, bool ZEROS>
void launch(const W4KParams& p, hipStream_t stream) {
  constexpr int W = 8;
  const unsigned gx = (unsigned)(p.swiglu ? p.tile_cols : (p.tile_cols + NT - 1) / NT);
  const unsigned gy = (unsigned)(p.rb_expert ? p.M / (16 * MT) : (p.M + 16 * MT - 1) / (16 * MT));
  hipLaunchKernelGGL((w4_kernel<MT, NT, W, SUB, ZEROS>), dim3(gx, gy), dim3(64 * W), W * NT * MT * 64 * sizeof(f32x4),
                     stream, p);
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
                                                             int64_t given, int64_t groups, int64_t tiles,
                                                             int64_t count, uint16_t* out_scales, uint8_t* out_zeros) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const int64_t g = i / kTile % groups, tile = i / kTile / groups % tiles, e = i / kTile / groups / tiles;
  const int64_t n = tile * kTile + i % kTile, at = (e * given + g) * N + n;
  const bool in = g < given && n < N;
  out_scales[i] = in ? scales[at] : 0;
  if (out_zeros) out_zeros[i] = in ? zeros[at] & 15u : 8u;
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
                     (K + group - 1) / group, KB * (kBlock / group), tiles, count, packed_scales, packed_zeros);
  return hipGetLastError();
}

hipError_t launch_w4_quantize(const uint16_t* W, int64_t K, int64_t N, int64_t E, int group, uint8_t* codes,
                              uint16_t* scales, hipStream_t stream) {
  const int64_t groups = (K + group - 1) / group, count = E * groups * N;
  hipLaunchKernelGGL(w4_quantize_kernel, dim3(blocks256(count)), dim3(256), 0, stream, W, K, N, group, groups, count,
                     codes, scales);
  return hipGetLastError();
}

hipError_t launch_w4(const W4KParams& p, hipStream_t stream) {
  if (p.M == 0) return hipSuccess;
  auto zeros = [&](auto mt, auto nt, auto sub) {
    if (p.w.zeros) launch<decltype(mt)::value, decltype(nt)::value, decltype(sub)::value, true>(p, stream);
    else launch<decltype(mt)::value, decltype(nt)::value, decltype(sub)::value, false>(p, stream);
  };
  auto sub = [&](auto mt, auto nt) {
    if (p.w.group == 32) zeros(mt, nt, std::integral_constant<int, 1>());
    else if (p.w.group == 64) zeros(mt, nt, std::integral_constant<int, 2>());
    else zeros(mt, nt, std::integral_constant<int, 4>());
  };
  auto nt = [&](auto mt) {
    if (p.swiglu) sub(mt, std::integral_constant<int, 2>());
    else sub(mt, std::integral_constant<int, 1>());
  };
  if (p.M <= 16 && !p.rb_expert) nt(std::integral_constant<int, 1>());
  else if (p.M <= 32 && !p.rb_expert) nt(std::integral_constant<int, 2>());
  else nt(std::integral_constant<int, 4>());
  return hipGetLastError();
}

}  // namespace mk
