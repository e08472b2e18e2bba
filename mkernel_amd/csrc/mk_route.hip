// mk_route.hip — the router of the MoE layer on gfx950: top-k choice, gates,
// per-expert counts and the balance loss in one pass over the logits, and the
// gradient of the logits.
//
// 16 logits per lane in registers, so 4 lanes (up to 64 experts) to 64 per token
// and 16 tokens to one per wavefront.  A choice is the maximum over (ordered
// bits of the logit, lowest index) as one number, so ids do not depend on how a
// sum is ordered, and ties go to the lowest index.
// The balance loss needs sums over all tokens: every workgroup writes its
// tokens' sums to the workspace and a second kernel adds them in a fixed order,
// so results do not depend on timing either.
//
// What bounds it: a small batch the chain of launch, loads, ranking and stores
// (1 x 256, 8 choices 3.2 us; 4096 x 256 fp32 with sums 8 to 9 and 6 us, gradient
// 8; its 128 workgroups leave half of the CUs idle).  A large one, 131001 x 60
// bf16, 4 choices, with sums, 13.9 us for 20 MB that a copy moves in 4: 477 vector
// instructions per 16 tokens, whose issue is 7 us and keeps the units busy for 73 %
// of the waves' life.  The sums over workgroups take 7.1 us, the gradient 14.3 (447
// instructions, 62 %; its waves wait for two thirds of their life, on the choices'
// logits, which are loaded after the choices).  fp32 logits take 134 to 138
// registers where bf16 takes 105, so a CU holds one workgroup of 8 waves with sums
// instead of two: 131001 x 60 fp32 26.5 us forward and 15.6 back, bf16 19.8 and
// 12.5 (calls back to back).  16384 x 256 bf16, 8 choices, without sums: 6.6 us.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "mk_device.h"
#include "mk_internal.h"

namespace mk {
namespace {

constexpr int kWaves = 4, kThreadsR = 64 * kWaves;
constexpr int kWavesSum = 8;        // with balance sums: fewer workgroups, so fewer parts to add
constexpr int kMaxBlocks = 2048;
constexpr int kMaxParts = 512;      // workgroups with balance sums
constexpr int kFinishExperts = 4;   // experts per workgroup of the second kernel

// exp(x - m) for every x of a token, m their maximum (and not -inf): 2^(x c - m c)
// with c = log2 e.  The product m c is rounded once, to `shift`; that error is
// one factor of all of a token's exponentials and cancels in their quotients.
// What is left is one rounding of the exponent: |x - m| half steps of the
// result, as much as the rounding of a difference x - m, and 0.3 as much from
// c.  The factor is 2 to the power of shift's error, up to |m| 2^-23: beyond
// kFar, where it would reach 2^(1/8) and later pass the range, the difference
// is taken first (the product then rounds once more).  Which form a token takes
// depends on its own logits only; the branch is taken where one of a wave does.
// A row with NaN or +inf gives NaN.
constexpr float kLog2e = 1.44269502162933349609375f, kFar = 0x1p20f;
struct ExpOf {
  float m, shift;
  bool far;
  __device__ __forceinline__ explicit ExpOf(float m_) : m(m_), shift(m_ * kLog2e), far(fabsf(m_) > kFar) {}
  template <int N>
  __device__ __forceinline__ void near_form(const float (&x)[N], float (&e)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = fmaf(x[i], kLog2e, -shift);
  }
  template <int N>
  __device__ __forceinline__ void far_form(const float (&x)[N], float (&e)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = far ? (x[i] - m) * kLog2e : e[i];
  }
};
// e = exp_a(x), g = exp_b(y), with one branch for both.
template <int N, int M>
__device__ __forceinline__ void exps(const ExpOf& a, const float (&x)[N], float (&e)[N], const ExpOf& b,
                                     const float (&y)[M], float (&g)[M]) {
  a.near_form(x, e);
  b.near_form(y, g);
  if (__builtin_expect(__any(a.far || b.far), 0)) {
    a.far_form(x, e);
    b.far_form(y, g);
    asm volatile("");  // keeps this a branch: as selects it is 3 instructions per value
  }
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = __builtin_amdgcn_exp2f(e[i]);
#pragma unroll
  for (int i = 0; i < M; ++i) g[i] = __builtin_amdgcn_exp2f(g[i]);
}

// A lane's V logits of a row as they lie in memory: a bf16 pair a word, or fp32.
template <class T, int V>
struct Raw {
  static constexpr int kWords = sizeof(T) == 2 ? V / 2 : V;
  uint32_t w[kWords];
  __device__ __forceinline__ void values(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 2) {
        x[2 * i] = bf16_lo(w[i]);
        x[2 * i + 1] = bf16_hi(w[i]);
      } else {
        x[i] = __uint_as_float(w[i]);
      }
    }
  }
};

// Keys: numbers whose order is that of (logit, lowest index): -0 equals +0, NaN
// above all.  A bf16 logit leaves room for its index in 32 bits: 16 bits in
// two's complement (two logits of a word at a time) above the inverted index.
// A float takes 44, as the fraction of a double in [1, 2), so that one
// v_max_f64 compares both at the rate of a 32-bit one.
template <class T>
struct Key;
template <>
struct Key<uint16_t> {
  using type = int32_t;
  static constexpr type kNone = INT32_MIN;  // (the least logit is -0x7fff)
  static constexpr uint32_t kCode = 0xffffu;  // less the index: a key's low bits
  typedef int16_t s16x2 __attribute__((ext_vector_type(2)));
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  template <int V>
  static __device__ __forceinline__ void make(const Raw<uint16_t, V>& raw, const uint32_t (&code)[V], type (&key)[V]) {
    s16x2 o[V / 2];
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const s16x2 sign = __builtin_bit_cast(s16x2, raw.w[i]) >> 15;
      o[i] = __builtin_bit_cast(s16x2, raw.w[i] ^ (__builtin_bit_cast(uint32_t, sign) & 0x7fff7fffu)) - sign;
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, raw.w[i] & 0x7fff7fffu));
    }
    if (__builtin_expect(__any(most[0] > 0x7f80 || most[1] > 0x7f80), 0)) {  // NaN of either sign: the greatest
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if ((raw.w[i] & 0x7fffu) > 0x7f80u) o[i][0] = 0x7fff;
        if ((raw.w[i] >> 16 & 0x7fffu) > 0x7f80u) o[i][1] = 0x7fff;
      }
      asm volatile("");  // (stays a branch)
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const uint32_t w = __builtin_bit_cast(uint32_t, o[i]);
      key[2 * i] = (int32_t)(w << 16 | code[2 * i]);
      key[2 * i + 1] = (int32_t)((w & 0xffff0000u) | code[2 * i + 1]);
    }
  }
  static __device__ __forceinline__ uint32_t index(type k) { return kCode - ((uint32_t)k & kCode); }
  static __device__ __forceinline__ float value(type k) {
    const int32_t o = k >> 16;
    return __uint_as_float((uint32_t)(o < 0 ? -o | 0x8000 : o) << 16);
  }
  static __device__ __forceinline__ type top(type a, type b) { return max(a, b); }
  static __device__ __forceinline__ type low(type a, type b) { return min(a, b); }
  template <int CTRL>
  static __device__ __forceinline__ type dpp(type k) {
    return __builtin_amdgcn_mov_dpp(k, CTRL, 0xf, 0xf, true);
  }
  static __device__ __forceinline__ type shuffle(type k, int mask) { return __shfl_xor(k, mask, 64); }
};
template <>
struct Key<float> {
  using type = double;
  static constexpr type kNone = 0.0;
  static constexpr uint32_t kCode = 0xfffffu;
  static __device__ __forceinline__ type pack(uint32_t hi, uint32_t lo) {
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  }
  template <int V>
  static __device__ __forceinline__ void make(const Raw<float, V>& raw, const uint32_t (&code)[V], type (&key)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float x = __uint_as_float(raw.w[j]);
      const uint32_t u = __float_as_uint(x + 0.f);
      const uint32_t o = x != x ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
      key[j] = pack(0x3ff00000u | o >> 12, o << 20 | code[j]);
    }
  }
  static __device__ __forceinline__ uint32_t index(type k) {
    return kCode - ((uint32_t)__builtin_bit_cast(uint64_t, k) & kCode);
  }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t o = (uint32_t)(__builtin_bit_cast(uint64_t, k) >> 20);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
  }
  static __device__ __forceinline__ type top(type a, type b) { return __builtin_fmax(a, b); }
  static __device__ __forceinline__ type low(type a, type b) { return __builtin_fmin(a, b); }
  template <int CTRL>
  static __device__ __forceinline__ type dpp(type k) {
    const uint64_t b = __builtin_bit_cast(uint64_t, k);
    return pack((uint32_t)__builtin_amdgcn_mov_dpp((int)(b >> 32), CTRL, 0xf, 0xf, true),
                (uint32_t)__builtin_amdgcn_mov_dpp((int)b, CTRL, 0xf, 0xf, true));
  }
  static __device__ __forceinline__ type shuffle(type k, int mask) {
    const uint64_t b = __builtin_bit_cast(uint64_t, k);
    return pack((uint32_t)__shfl_xor((int)(b >> 32), mask, 64), (uint32_t)__shfl_xor((int)b, mask, 64));
  }
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}

// All of the L neighbouring lanes of a token get op over their values.  Inside a
// row of 16 lanes the partner comes as a DPP operand: lane ^ 1, lane ^ 2, then
// mirrored halves (whose quads, and whose halves, hold one value by then).
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;
template <int L, class V, class Op, class Dpp, class Shuffle>
__device__ __forceinline__ V across(V v, Op op, Dpp d, Shuffle sh) {
  using std::integral_constant;
  v = op(v, d(v, integral_constant<int, kXor1>()));
  v = op(v, d(v, integral_constant<int, kXor2>()));
  if constexpr (L >= 8) v = op(v, d(v, integral_constant<int, kHalfMirror>()));
  if constexpr (L >= 16) v = op(v, d(v, integral_constant<int, kMirror>()));
  if constexpr (L >= 32) v = op(v, sh(v, 16));
  if constexpr (L >= 64) v = op(v, sh(v, 32));
  return v;
}

template <int L, class Op>
__device__ __forceinline__ float row_float(float v, Op op) {
  return across<L>(v, op, [](float x, auto c) { return dpp<decltype(c)::value>(x); },
                   [](float x, int m) { return __shfl_xor(x, m, 64); });
}
template <int L>
__device__ __forceinline__ float row_sum(float v) {
  return row_float<L>(v, [](float a, float b) { return a + b; });
}
template <int L>
__device__ __forceinline__ float row_max(float v) {
  return row_float<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L, class T>
__device__ __forceinline__ typename Key<T>::type row_top(typename Key<T>::type v) {
  using K = Key<T>;
  using V = typename K::type;
  return across<L>(v, [](V a, V b) { return K::top(a, b); },
                   [](V x, auto c) { return K::template dpp<decltype(c)::value>(x); },
                   [](V x, int m) { return K::shuffle(x, m); });
}

// The exchanges of a sorting network of V (a power of two) by odd-even merges,
// made by the compiler: every index is a constant, so keys stay in registers.
template <int V>
struct Network {
  int n = 0, a[V * V / 2 + 1] = {}, b[V * V / 2 + 1] = {};
  constexpr Network() {
    for (int p = 1; p < V; p *= 2)
      for (int k = p; k >= 1; k /= 2)
        for (int j = k % p; j + k < V; j += 2 * k)
          for (int i = 0; i < k; ++i)
            if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
              a[n] = i + j;
              b[n++] = i + j + k;
            }
  }
};

template <class T, int V, int N, size_t... I>
__device__ __forceinline__ void exchange(typename Key<T>::type (&a)[N], int at, std::index_sequence<I...>) {
  constexpr Network<V> net;
  auto one = [&](int hi, int lo) {
    const auto x = a[at + hi], y = a[at + lo];
    a[at + hi] = Key<T>::top(x, y);
    a[at + lo] = Key<T>::low(x, y);
  };
  (one(net.a[I], net.b[I]), ...);
}

// The D largest of a lane's V keys in falling order, in a[0 .. D): runs of D are
// sorted, then two runs at a time become one (the larger of each pair of a run
// and the other one reversed, put in order by halves).  V = 16: 126 minima and
// maxima for D = 16, 108 for 8, 76 for 4.
template <class T, int D, int V>
__device__ __forceinline__ void sort_keys(typename Key<T>::type (&a)[V]) {
  using K = Key<T>;
  constexpr Network<D> net;
#pragma unroll
  for (int g = 0; g < V; g += D) exchange<T, D>(a, g, std::make_index_sequence<net.n>());
#pragma unroll
  for (int runs = V / D; runs > 1; runs /= 2) {
#pragma unroll
    for (int g = 0; g < runs / 2; ++g) {
      typename K::type c[D];
#pragma unroll
      for (int i = 0; i < D; ++i) c[i] = K::top(a[2 * g * D + i], a[2 * g * D + 2 * D - 1 - i]);
#pragma unroll
      for (int d = D / 2; d >= 1; d /= 2)
#pragma unroll
        for (int i = 0; i < D; ++i)
          if ((i & d) == 0) {
            const auto x = c[i], y = c[i + d];
            c[i] = K::top(x, y);
            c[i + d] = K::low(x, y);
          }
#pragma unroll
      for (int i = 0; i < D; ++i) a[g * D + i] = c[i];
    }
  }
}

// Where a lane's values lie: V of them in pieces of C neighbours.
template <int L, int C>
__device__ __forceinline__ int expert_of(int lane, int j) {
  return (j / C) * (L * C) + lane * C + j % C;
}

template <class T>
__device__ __forceinline__ float load_one(const T* p) {
  if constexpr (sizeof(T) == 2) return __uint_as_float((uint32_t)*p << 16);
  else return *p;
}

template <int V, int L, int C, class T>
__device__ __forceinline__ void load_row(Raw<T, V>& x, const T* row, int E, int lane, bool on) {
  constexpr uint32_t kNothing = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
  constexpr int kEach = sizeof(T) == 2 ? 2 : 1;                              // values of a word
#pragma unroll
  for (int i = 0; i < x.kWords; ++i) x.w[i] = kNothing;
#pragma unroll
  for (int j = 0; j < V; j += C) {
    const int e = expert_of<L, C>(lane, j);
    if (on && e < E) {  // (C > 1: E is a multiple of it)
      if constexpr (C == 1 && sizeof(T) == 2) {
        x.w[j / 2] = j % 2 ? (x.w[j / 2] & 0xffffu) | (uint32_t)row[e] << 16 : (x.w[j / 2] & 0xffff0000u) | row[e];
      } else if constexpr (C == 1) {
        x.w[j] = __float_as_uint(row[e]);
      } else {
        typedef uint32_t words __attribute__((ext_vector_type(C / kEach)));
        const words v = *reinterpret_cast<const words*>(row + e);
#pragma unroll
        for (int i = 0; i < C / kEach; ++i) x.w[j / kEach + i] = v[i];
      }
    }
  }
}

// V values per lane, L lanes per token, KM the most choices (a lane keeps its
// KM largest, sorted; the winner of a round of maxima leaves its lane's list).
template <class T, int V, int L, int C, int KM>
__global__ __launch_bounds__(64 * kWavesSum) void route_kernel(RouteKParams p) {
  using K = Key<T>;
  using KeyT = typename K::type;
  constexpr int R = 64 / L, S = (KM + L - 1) / L, D = V < KM ? V : KM;
  extern __shared__ float psum[];  // [waves][L * V], with balance sums
  __shared__ int cnt[L * V];
  __shared__ int live_s;
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & (L - 1), sub = (threadIdx.x & 63) / L;
  const bool balance = p.part_sum != nullptr;
  if (balance) {
    for (int e = threadIdx.x; e < L * V; e += blockDim.x) cnt[e] = 0;
    if (threadIdx.x == 0) live_s = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
    __syncthreads();
  }
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int live = 0;
  const int64_t stride = (int64_t)gridDim.x * waves * R;
  int64_t t = ((int64_t)blockIdx.x * waves + wave) * R + sub;
  auto present = [&](int64_t u) { return u < p.T && (!p.mask || p.mask[u]); };
  // (in registers of their own: worked out anew they are one more instruction per key)
  uint32_t code[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    code[j] = K::kCode - expert_of<L, C>(lane, j);
    asm volatile("" : "+v"(code[j]));
  }
  Raw<T, V> next;
  load_row<V, L, C>(next, static_cast<const T*>(p.logits) + t * p.ld, p.E, lane, present(t));
  for (; t - sub < p.T; t += stride) {
    float x[V];
    next.values(x);
    KeyT key[V], kept[S];
    K::make(next, code, key);
    // the next token's logits are on their way while this one's are ranked
    if (t - sub + stride < p.T)
      load_row<V, L, C>(next, static_cast<const T*>(p.logits) + (t + stride) * p.ld, p.E, lane, present(t + stride));
    sort_keys<T, D>(key);
#pragma unroll
    for (int s = 0; s < S; ++s) kept[s] = K::kNone;
    KeyT best = row_top<L, T>(key[0]);
    const float m = K::value(best);
    for (int r = 0;;) {
      const bool won = key[0] == best;
#pragma unroll
      for (int i = 0; i < D; ++i) {
        // (by value: a choice between two elements would index the array)
        const KeyT here = key[i], then = i + 1 < D ? +key[i + 1 < D ? i + 1 : i] : K::kNone;
        key[i] = won ? then : here;
      }
#pragma unroll
      for (int s = 0; s < S; ++s) kept[s] = lane + s * L == r ? best : +kept[s];
      if (++r == p.k) break;
      best = row_top<L, T>(key[0]);
    }
    int id[S];
    float top[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const float v = K::value(kept[s]);
      const bool chosen = kept[s] != K::kNone && v != -INFINITY;
      id[s] = chosen ? (int)K::index(kept[s]) : -1;
      top[s] = chosen ? v : -INFINITY;
    }
    const bool alive = m != -INFINITY;
    const ExpOf exp_of(alive ? m : 0.f);
    // (top is -inf where there is no choice: 0, but NaN beside a NaN or +inf)
    float e[V], z = 1.f, g[S];
    if (balance || !p.renorm) {
      exps(exp_of, x, e, exp_of, top, g);
      z = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) z += e[j];
      z = row_sum<L>(z);
    } else {
      float none[1] = {0.f}, unused[1];
      exps(exp_of, none, unused, exp_of, top, g);
    }
    float zg = z;
#pragma unroll
    for (int s = 0; s < S; ++s) g[s] = id[s] >= 0 ? g[s] : 0.f;
    if (p.renorm) {
      zg = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) zg += g[s];
      zg = row_sum<L>(zg);
    }
    if (t < p.T) {
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (lane + s * L < p.k) {
          p.ids[t * p.k + lane + s * L] = id[s];
          p.gates[t * p.k + lane + s * L] = id[s] >= 0 ? g[s] / zg : 0.f;
        }
    }
    if (balance && alive) {
      live += lane == 0;
      const float inv = 1.f / z;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += e[j] * inv;
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (id[s] >= 0) atomicAdd(&cnt[id[s]], 1);
    }
  }
  if (!balance) return;
  if (live) atomicAdd(&live_s, live);
#pragma unroll
  for (int j = 0; j < V; ++j) {
#pragma unroll
    for (int d = L; d < 64; d *= 2) acc[j] += __shfl_xor(acc[j], d, 64);
    if (sub == 0) psum[wave * (L * V) + expert_of<L, C>(lane, j)] = acc[j];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < waves; ++w) s += psum[w * (L * V) + e];
    p.part_sum[(int64_t)blockIdx.x * p.E + e] = s;
    p.part_cnt[(int64_t)blockIdx.x * p.E + e] = cnt[e];
  }
  if (threadIdx.x == 0) p.part_live[blockIdx.x] = live_s;
}

// Sums the workgroups' parts, kFinishExperts experts per workgroup, in an order
// that the launch's size alone decides; the last workgroup to finish adds the
// experts' shares of the loss.  All latency: two loads' worth of memory, the
// store and ticket, and the shares (131001 x 60, 512 parts 7.2 us, one workgroup
// for everything 15; the sums in LDS one after another 9.5).
__global__ __launch_bounds__(256) void route_finish_kernel(RouteKParams p, int nparts) {
  constexpr int kSlices = 256 / kFinishExperts, kAhead = 16;
  __shared__ double sums[4][kFinishExperts];
  __shared__ int cnts[4][kFinishExperts], lives[4];
  __shared__ int last;
  const int x = threadIdx.x % kFinishExperts, slice = threadIdx.x / kFinishExperts;
  const int e = blockIdx.x * kFinishExperts + x;
  double s = 0.0;
  int c = 0, n = 0;
  for (int b0 = slice; b0 < nparts; b0 += kAhead * kSlices) {
    float ps[kAhead];
    int pc[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = b0 + i * kSlices;
      const bool in = e < p.E && b < nparts;
      ps[i] = in ? p.part_sum[(int64_t)b * p.E + e] : 0.f;
      pc[i] = in ? p.part_cnt[(int64_t)b * p.E + e] : 0;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      s += ps[i];
      c += pc[i];
    }
  }
  for (int b = threadIdx.x; b < nparts; b += 256) n += p.part_live[b];
#pragma unroll
  for (int d = kFinishExperts; d < 64; d *= 2) {
    s += __shfl_xor(s, d, 64);
    c += __shfl_xor(c, d, 64);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) n += __shfl_xor(n, d, 64);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < kFinishExperts) {
    sums[wave][x] = s;
    cnts[wave][x] = c;
    if (x == 0) lives[wave] = n;
  }
  __syncthreads();
  if (slice == 0) {
    for (int i = 1; i < 4; ++i) {
      s += sums[i][x];
      c += cnts[i][x];
    }
    if (e < p.E) {
      p.prob_sum[e] = (float)s;
      p.counts[e] = c;
    }
    double share = e < p.E ? s * c : 0.0;
#pragma unroll
    for (int d = 1; d < kFinishExperts; d *= 2) share += __shfl_xor(share, d, 64);
    sums[0][x] = share;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double share = sums[0][0];
    // written through to agent scope and waited for: a plain ticket orders it
    __hip_atomic_store(p.shares + blockIdx.x, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_vmem_all();
    last = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last || threadIdx.x >= 64) return;
  double sum = 0.0;  // one share per kFinishExperts experts
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 64)
    sum += __hip_atomic_load(p.shares + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if (threadIdx.x != 0) return;
  const int total = lives[0] + lives[1] + lives[2] + lives[3];
  *p.tokens = total;
  *p.loss = total ? (float)((double)p.coef * p.E * sum / ((double)p.k * total * total)) : 0.f;
}

template <class T, int V, int L, int C, int KM>
__global__ __launch_bounds__(kThreadsR) void route_backward_kernel(RouteBwdKParams p) {
  constexpr int R = 64 / L, S = (KM + L - 1) / L;
  // the gates' part of the gradient, by expert; zero but between a token's writes and reads
  __shared__ __align__(16) float add_s[kWaves * R][L * V];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & (L - 1), sub = (threadIdx.x & 63) / L;
  float* add = add_s[wave * R + sub];
  const int64_t stride = (int64_t)gridDim.x * kWaves * R;
  int64_t t = ((int64_t)blockIdx.x * kWaves + wave) * R + sub;
  auto present = [&](int64_t u) { return u < p.T && (!p.mask || p.mask[u]); };
  // a token's logits, choices and their gates' gradients
  struct Token {
    Raw<T, V> x;
    float dg[S];
    int id[S];
    bool on;
  } next;
  auto fetch = [&](int64_t u) {
    next.on = present(u);
    load_row<V, L, C>(next.x, static_cast<const T*>(p.logits) + u * p.ld, p.E, lane, next.on);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int i = lane + s * L;
      const bool in = p.dgates && next.on && i < p.k;
      next.id[s] = in ? p.ids[u * p.k + i] : -1;
      next.dg[s] = in ? p.dgates[u * p.k + i] : 0.f;
    }
  };
  fetch(t);
  // counts, and what a probability's gradient is multiplied with
  float f[V], scale = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = expert_of<L, C>(lane, j);
    f[j] = p.counts && e < p.E ? (float)p.counts[e] : 0.f;
    add[e] = 0.f;
  }
  if (p.counts) {
    const double n = *p.tokens;
    if (n > 0) scale = (float)((double)p.coef * (p.dloss ? *p.dloss : 1.f) * p.E / ((double)p.k * n * n));
  }
  for (; t - sub < p.T; t += stride) {
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    float x[V], dg[S], xc[S];
    int id[S];
    next.x.values(x);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      id[s] = next.id[s] < p.E ? next.id[s] : -1;
      dg[s] = id[s] >= 0 ? next.dg[s] : 0.f;
      xc[s] = id[s] >= 0 ? load_one(row + id[s]) : -INFINITY;
    }
    // the next token's are on their way meanwhile (an output over the logits
    // does not reach them: every row is read and written by the same lanes)
    if (t - sub + stride < p.T) fetch(t + stride);
    float m = -INFINITY;
    int odd = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      m = fmaxf(m, x[j]);
      odd |= x[j] != x[j];
    }
    m = row_max<L>(m);
    odd = row_max<L>(odd ? 1.f : 0.f) != 0.f || m == INFINITY;  // a NaN or +inf: the whole row is NaN
    const bool alive = m != -INFINITY || odd;  // else the token does not count, or no expert is left for it
    // the gates: softmax over the choices, or over all
    float mc = xc[0];
#pragma unroll
    for (int s = 1; s < S; ++s) mc = fmaxf(mc, xc[s]);
    mc = row_max<L>(mc);
    if (!p.renorm) mc = m;
    float pr[V], g[S], z = 0.f, s0 = 0.f;
    exps(ExpOf(alive ? m : 0.f), x, pr, ExpOf(mc != -INFINITY ? mc : 0.f), xc, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      z += pr[j];
      s0 += pr[j] * f[j];
    }
    z = row_sum<L>(z);
    const float inv = odd ? NAN : alive ? 1.f / z : 0.f;
    s0 = row_sum<L>(s0) * inv;
    float v[S], dense = 0.f;
    if (p.dgates) {
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        g[s] = id[s] >= 0 && xc[s] != -INFINITY ? g[s] : 0.f;
        sum += g[s];
      }
      if (p.renorm) {
        sum = row_sum<L>(sum);
        sum = sum > 0.f ? 1.f / sum : 0.f;
      } else {
        sum = inv;
      }
#pragma unroll
      for (int s = 0; s < S; ++s) {
        g[s] *= sum;
        dot += g[s] * dg[s];
      }
      dot = row_sum<L>(dot);
      if (!p.renorm) dense = dot;
#pragma unroll
      for (int s = 0; s < S; ++s) v[s] = g[s] * (p.renorm ? dg[s] - dot : dg[s]);
      // An expert named twice gets the sum, in the order of the choices: every
      // choice leaves its number at its expert's place, and only where one does
      // not find its own there again are they added one after another.
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (id[s] >= 0) add[id[s]] = __int_as_float(lane + s * L);
      __builtin_amdgcn_wave_barrier();
      bool twice = false;
#pragma unroll
      for (int s = 0; s < S; ++s) twice |= id[s] >= 0 && __float_as_int(add[id[s]]) != lane + s * L;
      __builtin_amdgcn_wave_barrier();
      if (!__any(twice)) {
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (id[s] >= 0) add[id[s]] = v[s];
      } else {
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (id[s] >= 0) add[id[s]] = 0.f;
        for (int i = 0; i < p.k; ++i) {
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int s = 0; s < S; ++s)
            if (id[s] >= 0 && lane + s * L == i) add[id[s]] += v[s];
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      d[j] = alive ? pr[j] * inv * (scale * (f[j] - s0) - dense) : 0.f;
      if (p.dgates) d[j] += add[expert_of<L, C>(lane, j)];
      if (odd) d[j] = NAN;
    }
    if (p.dgates) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (id[s] >= 0) add[id[s]] = 0.f;
    }
    if (t >= p.T) continue;
    T* out = static_cast<T*>(p.dlogits) + t * p.ld_out;
#pragma unroll
    for (int j = 0; j < V; j += C) {
      const int e = expert_of<L, C>(lane, j);
      if (e >= p.E) continue;
      if constexpr (C == 1) {
        if constexpr (sizeof(T) == 2) out[e] = __builtin_bit_cast(uint16_t, (__bf16)d[j]);
        else out[e] = d[j];
      } else if constexpr (sizeof(T) == 2) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        *reinterpret_cast<u32x2*>(out + e) = u32x2{pack_bf16x2(d[j], d[j + 1]), pack_bf16x2(d[j + 2], d[j + 3])};
      } else {
        *reinterpret_cast<f32x4*>(out + e) = f32x4{d[j], d[j + 1], d[j + 2], d[j + 3]};
      }
    }
  }
}

// Lanes and values per lane for E experts, pieces of C, and at most 4, 8 or
// kMaxTopk choices.
template <class F>
void by_shape(int E, bool vector, int k, F&& f) {
  using std::integral_constant;
  auto choices = [&](auto v, auto l, auto c) {
    if (k <= 4) f(v, l, c, integral_constant<int, 4>());
    else if (k <= 8) f(v, l, c, integral_constant<int, 8>());
    else f(v, l, c, integral_constant<int, kMaxTopk>());
  };
  auto pieces = [&](auto v, auto l) {
    if (vector) choices(v, l, integral_constant<int, 4>());
    else choices(v, l, integral_constant<int, 1>());
  };
  constexpr integral_constant<int, 16> v;
  if (E <= 64) pieces(v, integral_constant<int, 4>());
  else if (E <= 128) pieces(v, integral_constant<int, 8>());
  else if (E <= 256) pieces(v, integral_constant<int, 16>());
  else if (E <= 512) pieces(v, integral_constant<int, 32>());
  else pieces(v, integral_constant<int, 64>());
}

int tokens_per_wave(int E) { return E <= 64 ? 16 : E <= 128 ? 8 : E <= 256 ? 4 : E <= 512 ? 2 : 1; }

// Workgroups of `waves` waves, one token group per wave where that many are allowed.
int route_blocks(int64_t T, int E, int waves, int most) {
  const int64_t each = tokens_per_wave(E) * waves;
  return (int)std::max<int64_t>(1, std::min<int64_t>((T + each - 1) / each, most));
}

// Whether rows can be read (written) in pieces of four neighbours.
bool pieces_of_four(const void* rows, int64_t ld, int E, int bf16) {
  const int size = bf16 ? 2 : 4;
  return E % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(rows) % (4 * size) == 0;
}

}  // namespace

int64_t route_workspace_bytes(int64_t T, int E) {
  const int64_t nb = route_blocks(T, E, kWavesSum, kMaxParts);
  const int64_t shares = (E + kFinishExperts - 1) / kFinishExperts;
  return (8 * shares + 8 + nb * (8 * (int64_t)E + 4) + 255) / 256 * 256;
}

hipError_t launch_route(RouteKParams p, void* ws, hipStream_t stream) {
  const bool balance = ws != nullptr;
  const int waves = balance ? kWavesSum : kWaves;
  const int64_t nb = route_blocks(p.T, p.E, waves, balance ? kMaxParts : kMaxBlocks);
  const int shares = (p.E + kFinishExperts - 1) / kFinishExperts;
  if (balance) {
    p.shares = static_cast<double*>(ws);
    p.ticket = reinterpret_cast<uint32_t*>(p.shares + shares);
    p.part_sum = reinterpret_cast<float*>(p.ticket + 2);
    p.part_cnt = reinterpret_cast<int*>(p.part_sum + nb * p.E);
    p.part_live = p.part_cnt + nb * p.E;
  } else if (p.T == 0) {
    return hipSuccess;
  }
  by_shape(p.E, pieces_of_four(p.logits, p.ld, p.E, p.bf16), p.k, [&](auto v, auto l, auto c, auto km) {
    constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value, KM = decltype(km)::value;
    const unsigned lds = balance ? waves * L * V * sizeof(float) : 0;
    if (p.bf16)
      hipLaunchKernelGGL((route_kernel<uint16_t, V, L, C, KM>), dim3((unsigned)nb), dim3(64 * waves), lds, stream, p);
    else
      hipLaunchKernelGGL((route_kernel<float, V, L, C, KM>), dim3((unsigned)nb), dim3(64 * waves), lds, stream, p);
  });
  if (balance) hipLaunchKernelGGL(route_finish_kernel, dim3(shares), dim3(256), 0, stream, p, (int)nb);
  return hipGetLastError();
}

hipError_t launch_route_backward(const RouteBwdKParams& p, hipStream_t stream) {
  if (p.T == 0) return hipSuccess;
  const int nb = route_blocks(p.T, p.E, kWaves, kMaxBlocks / 2);
  const bool vector = pieces_of_four(p.logits, p.ld, p.E, p.bf16) && pieces_of_four(p.dlogits, p.ld_out, p.E, p.bf16);
  by_shape(p.E, vector, p.k, [&](auto v, auto l, auto c, auto km) {
    constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value, KM = decltype(km)::value;
    if (p.bf16)
      hipLaunchKernelGGL((route_backward_kernel<uint16_t, V, L, C, KM>), dim3(nb), dim3(kThreadsR), 0, stream, p);
    else
      hipLaunchKernelGGL((route_backward_kernel<float, V, L, C, KM>), dim3(nb), dim3(kThreadsR), 0, stream, p);
  });
  return hipGetLastError();
}

}  // namespace mk
