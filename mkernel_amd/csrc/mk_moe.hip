// mk_moe.hip — HBM-bound MoE data movement on gfx950:
//   * permute: expert-contiguous gather of token rows (reference
//     src/dispatch_gemm.cu:106-198 dispatch_fused), 128-bit loads/stores;
//   * combine: deterministic gather of the top-k expert rows of each source
//     token, weighted and summed in fp32 (reference
//     src/dispatch_gemm_glu_combine.cu:736-818 combine_gather_owner; the
//     reference pre-rounds w*y to bf16 in its producer step, here the product
//     stays fp32 because the rows are read in place on the same GPU).
#include <algorithm>

#include "mk_device.h"
#include "mk_internal.h"

namespace mk {

// One workgroup per padded row; padding rows (src_node < 0) are zero-filled.
// With a device row count, rows past it (capacity rows) are left untouched.
__global__ __launch_bounds__(kThreads) void permute_kernel(PermuteKParams p) {
  const int64_t r = blockIdx.x;
  if (p.rows_dev && r >= *p.rows_dev) return;
  const int* pr = p.pull + 3 * r;
  const int src_node = pr[0], src_dev = pr[1], src_tok = pr[2];
  const int64_t vec = p.H / 8;
  uint4* dst = reinterpret_cast<uint4*>(p.post + r * p.H);
  if (src_node < 0 || src_tok < 0) {
    const uint4 z = {0u, 0u, 0u, 0u};
    for (int64_t c = threadIdx.x; c < vec; c += kThreads) dst[c] = z;
    return;
  }
  const int64_t srow = ((int64_t)src_node * p.devs_per_node + src_dev) * p.tokens_per_src + src_tok;
  const uint4* src = reinterpret_cast<const uint4*>(p.tokens + srow * p.H);
  for (int64_t c = threadIdx.x; c < vec; c += kThreads) dst[c] = src[c];
}

hipError_t launch_permute(const PermuteKParams& p, hipStream_t stream) {
  if (p.R_pad == 0) return hipSuccess;
  hipLaunchKernelGGL(permute_kernel, dim3((unsigned)p.R_pad), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// One workgroup per source token (several, each with a share of the column
// chunks, when the tokens alone do not fill the chip: the loop over chunks is a
// chain of load latencies); each thread owns V contiguous columns, 16 bytes of
// the output: 8 of bf16, 4 of fp32, so that neighbouring lanes store
// neighbouring 16-byte pieces.
// The token's (row, weight) pairs are loaded once per thread, before the
// column loop (at most kMaxSlots of them; more fall back to the slot loop),
// and all of a chunk's row loads are issued before they are summed: the
// kernel is latency-bound, and the dependent owner -> slot -> row -> data
// chain per column chunk made it so.  Sums stay in slot order
// (deterministic, bit-identical to the plain loop).
// Rows are bf16, or fp32 (F32: the 4-bit expert layer's, which are not rounded
// before the sum).
template <int V, bool F32>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombineKParams p) {
  constexpr int kMaxSlots = 8, kWords = F32 ? V : V / 2;  // 32-bit words of a row chunk
  typedef uint32_t words __attribute__((ext_vector_type(kWords)));
  const int64_t t = blockIdx.x;
  const int s0 = p.owner_offset[t], s1 = p.owner_offset[t + 1];
  const int n = p.rows > 0 ? s1 - s0 : 0;  // (without rows the tables may be NULL)
  const int64_t vec = p.H / V;
  int rows[kMaxSlots];
  float wts[kMaxSlots];
  const bool few = n <= kMaxSlots;
#pragma unroll
  for (int k = 0; k < kMaxSlots; ++k)
    if (few && k < n) rows[k] = p.slot_to_row[s0 + k];
  // a slot whose row is -1 was not produced on this GPU (another owner's
  // combine covers it), and one at or past the rows' count not at all: it
  // contributes nothing (as unsigned numbers both are at or past the count)
  auto has = [&](int row) { return (uint32_t)row < p.rows; };
#pragma unroll
  for (int k = 0; k < kMaxSlots; ++k)
    if (few && k < n) wts[k] = has(rows[k]) ? p.row_weight[rows[k]] : 0.f;
  for (int64_t c = (int64_t)blockIdx.y * kThreads + threadIdx.x; c < vec; c += (int64_t)gridDim.y * kThreads) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    auto add = [&](float w, const words& v) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (F32) {
          acc[i] += w * __uint_as_float(v[i]);
        } else {
          acc[2 * i] += w * bf16_lo(v[i]);
          acc[2 * i + 1] += w * bf16_hi(v[i]);
        }
      }
    };
    auto load = [&](int64_t row) {
      return *reinterpret_cast<const words*>(static_cast<const char*>(p.y_expert) + (row * p.H + c * V) * (F32 ? 4 : 2));
    };
    if (few) {
      words v[kMaxSlots];
#pragma unroll
      for (int k = 0; k < kMaxSlots; ++k)
        if (k < n && has(rows[k])) v[k] = load(rows[k]);
#pragma unroll
      for (int k = 0; k < kMaxSlots; ++k)
        if (k < n && has(rows[k])) add(wts[k], v[k]);
    } else {
      for (int s = s0; s < s1; ++s) {
        const int row = p.slot_to_row[s];
        if (!has(row)) continue;
        add(p.row_weight[row], load(row));
      }
    }
    // the layer's output is not read again here: nontemporal stores
    // (config 5 layer -7 us against plain stores)
    if constexpr (V == 4) {
      __builtin_nontemporal_store(f32x4{acc[0], acc[1], acc[2], acc[3]},
                                  reinterpret_cast<f32x4*>(static_cast<float*>(p.y_out) + t * p.H + c * V));
    } else {
      typedef uint32_t u4 __attribute__((ext_vector_type(4)));
      __builtin_nontemporal_store(u4{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]),
                                     pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7])},
                                  reinterpret_cast<u4*>(static_cast<uint16_t*>(p.y_out) + t * p.H + c * V));
    }
  }
}

hipError_t launch_combine(const CombineKParams& p, hipStream_t stream) {
  if (p.num_tokens == 0) return hipSuccess;
  const int64_t v = p.out_dtype == 0 ? 4 : 8;
  const int64_t chunks = (p.H / v + kThreads - 1) / kThreads;
  // workgroups per token: enough for 1024 in all, at most one per column chunk
  const unsigned split = (unsigned)std::max<int64_t>(1, std::min<int64_t>(chunks, 1024 / p.num_tokens));
  auto* kernel = p.f32_rows ? (v == 4 ? combine_kernel<4, true> : combine_kernel<8, true>)
                            : (v == 4 ? combine_kernel<4, false> : combine_kernel<8, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.num_tokens, split), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// Gradient of the combine.
//   dy_expert[r] = row_weight[r] * dy[t]            (one bf16 rounding)
//   dgates[t, j] = sum_c dy[t, c] * y_expert[r, c]  (fp32), r the row of (t, j)
// Bound by its bytes (dy and the routed rows read, dy_expert's whole row blocks
// written).  Workgroup t has token t's rows, kAtOnce of them against one read of
// dy; those behind the tokens zero kPadRows padding rows each (a whole row
// block's in one workgroup was the longest of the launch).  2048 x 7168, fp32
// dy, 32 of 256 experts: 34 us.
// The row of (t, j) is found as the index build gave it out: the token's local
// choices, ordered by (expert, j), have its slots in turn.
constexpr int kAtOnce = 4, kPadRows = 8;
template <class T>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(CombineBwdKParams p) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  constexpr int U = 4;  // pieces of 8 columns a thread has on their way
  const int64_t R = p.rows_dev ? min(p.R_pad, *p.rows_dev) : p.R_pad;
  const int64_t vec = p.H / 8;
  if ((int64_t)blockIdx.x >= p.T) {
    const int64_t r0 = (int64_t)(blockIdx.x - p.T) * kPadRows, b = r0 / kFlagRows;
    if (r0 >= R) return;
    const int64_t from = max(r0, b * kFlagRows + min(max(p.rb_rows[b], 0), kFlagRows));
    words* dst = reinterpret_cast<words*>(p.dy_expert);
    for (int64_t c = from * vec + threadIdx.x; c < (r0 + kPadRows) * vec; c += kThreads) dst[c] = words{0u, 0u, 0u, 0u};
    return;
  }
  const int64_t t = blockIdx.x;
  __shared__ int rows[kMaxTopk], choice[kMaxTopk], count;
  __shared__ float part[kThreads / 64][kAtOnce];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave == 0) {
    const int e = lane < p.k ? p.ids[t * p.k + lane] - p.e0 : -1;
    const bool local = e >= 0 && e < p.n_local;
    int slot = p.owner_offset[t], row = -1;
    for (int i = 0; i < p.k; ++i) {
      const int o = __shfl(e, i, 64);
      slot += o >= 0 && o < p.n_local && (o < e || (o == e && i < lane));
    }
    // (without rows there may be no slot_to_row either)
    if (R > 0 && local && slot < p.owner_offset[t + 1]) row = p.slot_to_row[slot];
    if (row >= R) row = -1;
    const uint64_t there = __ballot(row >= 0);
    const int at = __popcll(there & ((1ull << lane) - 1));
    if (row >= 0) {
      rows[at] = row;
      choice[at] = lane;
    } else if (lane < p.k) {
      p.dgates[t * p.k + lane] = 0.f;
    }
    if (lane == 0) count = __popcll(there);
  }
  __syncthreads();
  const T* dy = static_cast<const T*>(p.dy) + t * p.H;
  for (int j0 = 0; j0 < count; j0 += kAtOnce) {
    const int n = min(count - j0, kAtOnce);
    int64_t row[kAtOnce];
    float w[kAtOnce], dot[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      row[j] = rows[min(j0 + j, count - 1)];
      w[j] = p.row_weight[row[j]];
      dot[j] = 0.f;
    }
    for (int64_t c0 = threadIdx.x; c0 < vec; c0 += U * kThreads) {
      float d[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t c = c0 + u * kThreads;
        if (c >= vec) continue;
        if constexpr (sizeof(T) == 2) {
          const words v = *reinterpret_cast<const words*>(dy + 8 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            d[u][2 * i] = bf16_lo(v[i]);
            d[u][2 * i + 1] = bf16_hi(v[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(dy + 8 * c + 4 * i);
#pragma unroll
            for (int b = 0; b < 4; ++b) d[u][4 * i + b] = v[b];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (j >= n) continue;
        words y[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + u * kThreads < vec) y[u] = *reinterpret_cast<const words*>(p.y_expert + row[j] * p.H + 8 * (c0 + u * kThreads));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t c = c0 + u * kThreads;
          if (c >= vec) continue;
          words o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dot[j] += d[u][2 * i] * bf16_lo(y[u][i]);
            dot[j] += d[u][2 * i + 1] * bf16_hi(y[u][i]);
            o[i] = pack_bf16x2(w[j] * d[u][2 * i], w[j] * d[u][2 * i + 1]);
          }
          if (p.dy_expert) *reinterpret_cast<words*>(p.dy_expert + row[j] * p.H + 8 * c) = o;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
#pragma unroll
      for (int s = 32; s; s >>= 1) dot[j] += __shfl_xor(dot[j], s, 64);
      if (lane == 0) part[wave][j] = dot[j];
    }
    __syncthreads();
    if ((int)threadIdx.x < n) {
      float sum = 0.f;
      for (int v = 0; v < kThreads / 64; ++v) sum += part[v][threadIdx.x];
      p.dgates[t * p.k + choice[j0 + threadIdx.x]] = sum;
    }
    __syncthreads();
  }
}

hipError_t launch_combine_backward(CombineBwdKParams p, hipStream_t stream) {
  p.pad_blocks = p.dy_expert ? (int)(p.R_pad / kPadRows) : 0;
  const int64_t blocks = p.T + p.pad_blocks;
  if (blocks == 0) return hipSuccess;
  if (p.dy_dtype == 0)
    hipLaunchKernelGGL(combine_backward_kernel<float>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(combine_backward_kernel<uint16_t>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// One workgroup per 128-row block: count rows with a real source token.
__global__ __launch_bounds__(128) void tile_rows_kernel(const int* pull, int64_t R_pad, int* rb_rows) {
  const int64_t r = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int real = (r < R_pad && pull[3 * r] >= 0) ? 1 : 0;
  const int n = __syncthreads_count(real);
  if (threadIdx.x == 0) rb_rows[blockIdx.x] = n;
}

hipError_t launch_tile_rows(const int* pull, int64_t R_pad, int* rb_rows, hipStream_t stream) {
  if (R_pad == 0) return hipSuccess;
  hipLaunchKernelGGL(tile_rows_kernel, dim3((unsigned)((R_pad + 127) / 128)), dim3(128), 0, stream, pull, R_pad, rb_rows);
  return hipGetLastError();
}

__global__ void fill_i32_kernel(int* dst, int64_t n, int value) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) dst[i] = value;
}

// Rows of `owner` only; a slot outside [0, cap) is skipped and reported.
__global__ void invert_slots_kernel(const int* row_to_slot, const int* row_to_owner, int64_t R_pad, int owner,
                                    int64_t cap, int* slot_to_row, uint32_t* err) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= R_pad || row_to_owner[r] != owner) return;
  const int s = row_to_slot[r];
  if (s >= 0 && s < cap) slot_to_row[s] = (int)r;
  else if (err) __hip_atomic_fetch_or(err, 2u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

hipError_t launch_invert_slots(const int* row_to_slot, const int* row_to_owner, int64_t R_pad, int owner,
                               int64_t cap, int* slot_to_row, uint32_t* err, hipStream_t stream) {
  // a fill kernel, not hipMemsetAsync, so the pair can be recorded in a graph
  if (cap > 0)
    hipLaunchKernelGGL(fill_i32_kernel, dim3((unsigned)((cap + 255) / 256)), dim3(256), 0, stream, slot_to_row, cap, -1);
  if (R_pad > 0)
    hipLaunchKernelGGL(invert_slots_kernel, dim3((unsigned)((R_pad + 255) / 256)), dim3(256), 0, stream, row_to_slot,
                       row_to_owner, R_pad, owner, cap, slot_to_row, err);
  return hipGetLastError();
}

}  // namespace mk
