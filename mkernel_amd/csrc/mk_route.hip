// mk_route.hip — the router of the MoE layer on gfx950: top-k choice, gates,
// per-expert counts and the balance loss in one pass over the logits, and the
// gradient of the logits.
//
// One wavefront per token; lane l holds experts l, l + 64, ... in registers.
// A choice is the maximum over (ordered bits of the logit, lowest index), so
// ids do not depend on how a sum is ordered, and ties go to the lowest index.
// The balance loss needs sums over all tokens: every workgroup writes its
// tokens' sums to the workspace and a second kernel adds them in workgroup
// order, so results do not depend on timing either.
#include <algorithm>
#include <type_traits>

#include "mk_device.h"
#include "mk_internal.h"

namespace mk {
namespace {

constexpr int kWaves = 4, kThreadsR = 64 * kWaves;
constexpr int kMaxBlocks = 1024;   // workgroups of a launch with balance sums
constexpr int kFinishExperts = 16; // experts per workgroup of the second kernel

// Bits of x ordered as unsigned integers: -0 equals +0, NaN above all.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kOrderedNegInf = 0x007fffffu;

// exp(x) for x <= 0 to about an ulp: the product with log2 e carried in two
// parts, since one rounding of it is |x| times as large in the result.
__device__ __forceinline__ float exp_neg(float x) {
  constexpr float kLog2e = 1.44269502162933349609375f, kLog2eLo = 1.92596299112661746887e-8f;
  const float hi = x * kLog2e;
  float lo = fmaf(x, kLog2e, -hi);
  lo = fmaf(x, kLog2eLo, lo);
  const float e = __builtin_amdgcn_exp2f(hi);
  return hi == -INFINITY ? 0.f : fmaf(e, lo * 0.693147182464599609375f, e);
}

template <class T>
__device__ __forceinline__ float load_logit(const T* p) {
  if constexpr (sizeof(T) == 2) return __uint_as_float((uint32_t)*p << 16);
  else return *p;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

// V values per lane (64 V >= E).
template <class T, int V>
__global__ __launch_bounds__(kThreadsR) void route_kernel(RouteKParams p) {
  __shared__ float psum[kWaves][64 * V];
  __shared__ int cnt[64 * V];
  __shared__ int live_s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool balance = p.part_sum != nullptr;
  if (balance) {
    for (int e = threadIdx.x; e < 64 * V; e += kThreadsR) cnt[e] = 0;
    if (threadIdx.x == 0) live_s = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
    __syncthreads();
  }
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int live = 0;
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave; t < p.T; t += (int64_t)gridDim.x * kWaves) {
    if (p.mask && !p.mask[t]) {
      if (lane < p.k) {
        p.ids[t * p.k + lane] = -1;
        p.gates[t * p.k + lane] = 0.f;
      }
      continue;
    }
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    float x[V];
    uint64_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + 64 * j;
      x[j] = e < p.E ? load_logit(row + e) : -INFINITY;
      key[j] = (uint64_t)ordered(x[j]) << 32 | (uint32_t)(0xffff - e);
    }
    int my_id = -1;
    float my_x = -INFINITY, m = -INFINITY;
    for (int r = 0; r < p.k; ++r) {
      uint64_t best = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) best = key[j] > best ? key[j] : best;
#pragma unroll
      for (int d = 32; d; d >>= 1) {
        const uint64_t o = (uint64_t)__shfl_xor((uint32_t)(best >> 32), d, 64) << 32 | __shfl_xor((uint32_t)best, d, 64);
        best = o > best ? o : best;
      }
      if ((uint32_t)(best >> 32) <= kOrderedNegInf) break;
      const int id = 0xffff - (int)(uint32_t)best;
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (key[j] == best) {
          key[j] = 0;
          v = x[j];
        }
      v = __shfl(v, id & 63, 64);
      if (r == 0) m = v;
      if (lane == r) {
        my_id = id;
        my_x = v;
      }
    }
    const bool alive = m != -INFINITY;
    float e[V], z = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      e[j] = alive ? exp_neg(x[j] - m) : 0.f;
      z += e[j];
    }
    z = wave_sum(z);
    float g = my_id >= 0 ? exp_neg(my_x - m) : 0.f;
    const float zg = p.renorm ? wave_sum(g) : z;
    if (my_id >= 0) g /= zg;
    if (lane < p.k) {
      p.ids[t * p.k + lane] = my_id;
      p.gates[t * p.k + lane] = g;
    }
    if (balance && alive) {
      ++live;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += e[j] / z;
      if (my_id >= 0) atomicAdd(&cnt[my_id], 1);
    }
  }
  if (!balance) return;
  if (lane == 0) atomicAdd(&live_s, live);
#pragma unroll
  for (int j = 0; j < V; ++j) psum[wave][lane + 64 * j] = acc[j];
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kThreadsR) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += psum[w][e];
    p.part_sum[(int64_t)blockIdx.x * p.E + e] = s;
    p.part_cnt[(int64_t)blockIdx.x * p.E + e] = cnt[e];
  }
  if (threadIdx.x == 0) p.part_live[blockIdx.x] = live_s;
}

// Sums the workgroups' parts in order, kFinishExperts experts per workgroup;
// the last workgroup to finish adds the experts' shares of the loss.
__global__ __launch_bounds__(256) void route_finish_kernel(RouteKParams p, int nparts) {
  constexpr int kSlices = 256 / kFinishExperts;
  __shared__ double sums[kSlices][kFinishExperts];
  __shared__ int cnts[kSlices][kFinishExperts];
  __shared__ int last;
  const int x = threadIdx.x % kFinishExperts, slice = threadIdx.x / kFinishExperts;
  const int e = blockIdx.x * kFinishExperts + x;
  double s = 0.0;
  int c = 0;
  if (e < p.E)
    for (int b = slice; b < nparts; b += kSlices) {
      s += p.part_sum[(int64_t)b * p.E + e];
      c += p.part_cnt[(int64_t)b * p.E + e];
    }
  sums[slice][x] = s;
  cnts[slice][x] = c;
  __syncthreads();
  if (slice == 0) {
    for (int i = 1; i < kSlices; ++i) {
      s += sums[i][x];
      c += cnts[i][x];
    }
    if (e < p.E) {
      p.prob_sum[e] = (float)s;
      p.counts[e] = c;
    }
    sums[0][x] = e < p.E ? s * c : 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double share = 0.0;
    for (int i = 0; i < kFinishExperts; ++i) share += sums[0][i];
    __hip_atomic_store(p.shares + blockIdx.x, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  int n = 0;
  for (int b = threadIdx.x; b < nparts; b += 256) n += p.part_live[b];
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  atomicAdd(&total, n);
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int b = 0; b < (int)gridDim.x; ++b)
      sum += __hip_atomic_load(p.shares + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *p.tokens = total;
    *p.loss = total ? (float)((double)p.coef * p.E * sum / ((double)p.k * total * total)) : 0.f;
  }
}

template <class T, int V>
__global__ __launch_bounds__(kThreadsR) void route_backward_kernel(RouteBwdKParams p) {
  __shared__ float add[kWaves][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // counts, and what a probability's gradient is multiplied with
  float f[V], scale = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = 0.f;
  if (p.counts) {
    const double n = *p.tokens;
    if (n > 0) scale = (float)((double)p.coef * (p.dloss ? *p.dloss : 1.f) * p.E / ((double)p.k * n * n));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + 64 * j;
      if (e < p.E) f[j] = (float)p.counts[e];
    }
  }
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave; t < p.T; t += (int64_t)gridDim.x * kWaves) {
    T* out = static_cast<T*>(p.dlogits) + t * p.ld_out;
    auto store = [&](int e, float v) {
      if constexpr (sizeof(T) == 2) out[e] = __builtin_bit_cast(uint16_t, (__bf16)v);
      else out[e] = v;
    };
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    float x[V], m = -INFINITY;
    const bool on = !p.mask || p.mask[t];
    bool nan = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + 64 * j;
      x[j] = on && e < p.E ? load_logit(row + e) : -INFINITY;
      nan |= x[j] != x[j];
      m = fmaxf(m, x[j]);
    }
    m = __any(nan) ? NAN : wave_max(m);
    if (m == -INFINITY) {  // a token that does not count, or that no expert is left for
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (lane + 64 * j < p.E) store(lane + 64 * j, 0.f);
      continue;
    }
    float pr[V], z = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      pr[j] = exp_neg(x[j] - m);
      z += pr[j];
    }
    z = wave_sum(z);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      pr[j] /= z;
      s += pr[j] * f[j];
    }
    s = wave_sum(s);
    // the gates' part: lane i has choice i
    int id = -1;
    float dg = 0.f, v = 0.f, dense = 0.f;
    if (p.dgates) {
      if (lane < p.k) id = p.ids[t * p.k + lane];
      if (id >= p.E) id = -1;
      float xc = -INFINITY;
      if (id >= 0) {
        dg = p.dgates[t * p.k + lane];
        xc = load_logit(row + id);
      }
      if (p.renorm) {
        const float mc = wave_max(xc);
        float g = id >= 0 && mc != -INFINITY ? exp_neg(xc - mc) : 0.f;
        g /= fmaxf(wave_sum(g), 1e-30f);
        if (z != z) g = z;
        const float dot = wave_sum(id >= 0 ? g * dg : 0.f);
        v = id >= 0 ? g * (dg - dot) : 0.f;
      } else {
        const float g = id >= 0 ? exp_neg(xc - m) / z : 0.f;
        v = g * dg;
        dense = wave_sum(v);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) add[wave][lane + 64 * j] = 0.f;
      // an expert named twice: its first lane adds all, in lane order
      float all = 0.f;
      bool first = id >= 0;
      for (int i = 0; i < p.k; ++i) {
        const int oi = __shfl(id, i, 64);
        const float ov = __shfl(v, i, 64);
        if (oi == id) {
          all += ov;
          if (i < lane) first = false;
        }
      }
      __builtin_amdgcn_wave_barrier();
      if (first) add[wave][id] = all;
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + 64 * j;
      float d = pr[j] * (scale * (f[j] - s) - dense);
      if (p.dgates) d += add[wave][e];
      if (e < p.E) store(e, d);
    }
  }
}

int route_blocks(int64_t T, bool balance) {
  const int64_t all = (T + kWaves - 1) / kWaves;
  return (int)std::max<int64_t>(1, std::min<int64_t>(all, balance ? kMaxBlocks : 1 << 20));
}

template <class F>
void by_width(int E, F&& f) {
  if (E <= 64) f(std::integral_constant<int, 1>());
  else if (E <= 128) f(std::integral_constant<int, 2>());
  else if (E <= 256) f(std::integral_constant<int, 4>());
  else if (E <= 512) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

}  // namespace

int64_t route_workspace_bytes(int64_t T, int E) {
  const int64_t nb = route_blocks(T, true);
  const int64_t shares = (E + kFinishExperts - 1) / kFinishExperts;
  return (8 * shares + 8 + nb * (8 * (int64_t)E + 4) + 255) / 256 * 256;
}

hipError_t launch_route(RouteKParams p, void* ws, hipStream_t stream) {
  const bool balance = ws != nullptr;
  const int nb = route_blocks(p.T, balance);
  const int shares = (p.E + kFinishExperts - 1) / kFinishExperts;
  if (balance) {
    p.shares = static_cast<double*>(ws);
    p.ticket = reinterpret_cast<uint32_t*>(p.shares + shares);
    p.part_sum = reinterpret_cast<float*>(p.ticket + 2);
    p.part_cnt = reinterpret_cast<int*>(p.part_sum + (int64_t)nb * p.E);
    p.part_live = p.part_cnt + (int64_t)nb * p.E;
  } else if (p.T == 0) {
    return hipSuccess;
  }
  by_width(p.E, [&](auto v) {
    constexpr int V = decltype(v)::value;
    if (p.bf16) hipLaunchKernelGGL((route_kernel<uint16_t, V>), dim3(nb), dim3(kThreadsR), 0, stream, p);
    else hipLaunchKernelGGL((route_kernel<float, V>), dim3(nb), dim3(kThreadsR), 0, stream, p);
  });
  if (balance) hipLaunchKernelGGL(route_finish_kernel, dim3(shares), dim3(256), 0, stream, p, nb);
  return hipGetLastError();
}

hipError_t launch_route_backward(const RouteBwdKParams& p, hipStream_t stream) {
  if (p.T == 0) return hipSuccess;
  const int nb = route_blocks(p.T, false);
  by_width(p.E, [&](auto v) {
    constexpr int V = decltype(v)::value;
    if (p.bf16) hipLaunchKernelGGL((route_backward_kernel<uint16_t, V>), dim3(nb), dim3(kThreadsR), 0, stream, p);
    else hipLaunchKernelGGL((route_backward_kernel<float, V>), dim3(nb), dim3(kThreadsR), 0, stream, p);
  });
  return hipGetLastError();
}

}  // namespace mk
