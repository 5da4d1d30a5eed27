// Mixture of experts around the experts' products: routing of tokens to experts (with its gradient),
// the expert order of the chosen rows, and the weighted sum that brings the experts' rows back to
// their tokens (with its gradients).  No counterpart in the reference; routing stands beside the
// top-k of topk.cu and keeps its order (greatest first, lowest index among equals, NaN greatest).
#include <limits.h>

#include <type_traits>

#include "early_launch.cuh"
#include "kmb_common.cuh"
#include "row_types.cuh"

namespace kmb {

constexpr unsigned FULL = 0xffffffffu;
constexpr int64_t MAX_CHOICES = INT32_MAX - 4096;    // n * k: places are 32-bit numbers, grids a little longer

// ================================================================================== routing
// L lanes of a warp per token (8, 16 or 32).  Lane l of them holds the V consecutive experts l * V ..
// l * V + V - 1 in registers, so that the lowest lane among equals is the lowest index.  k rounds take the
// greatest key each: a maximum in the lane, one over the lanes, a ballot for the lowest of them.
// Bound by the rounds, each a chain of shuffles behind the one before: neither HBM (1.0 TB/s) nor issue (0.55 to 0.65
// a scheduler and cycle) is full.  16 384 x 128 float32, k = 8, takes 9.4 us, 65 521 x 64 bfloat16, k = 6, 13 us; with
// a whole warp per token, whatever the number of experts, 17 and 41 us.
constexpr int RT_WARPS = 4;
constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_K = 32;       // the choices of a token live one to a lane
constexpr int RT_MAX_GROUPS = 32;  // and so do its groups

struct RouteParams {
  const void* logits;
  const float* bias;        // or NULL
  float* weights;
  int32_t* experts;
  int64_t n;
  int n_experts, k, groups, topk_groups, group_best, group_size;
  int sigmoid, renormalize, vec;
  float scale;
};

// Whole numbers in the order of the values, NaN on top; 0 is below everything, -inf among it.
__device__ __forceinline__ uint32_t order_bits(float v) {
  uint32_t b = __float_as_uint(v + 0.f);      // -0 and 0 are one value
  b ^= (b >> 31) ? 0xffffffffu : 0x80000000u;
  b = b == 0x007fffffu ? 0u : b;              // -inf: never chosen
  return v != v ? 0xffffffffu : b;
}
__device__ __forceinline__ unsigned long long order_bits(double v) {
  if (v != v) return 0xffffffffffffffffull;
  unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  b ^= (b >> 63) ? 0xffffffffffffffffull : 0x8000000000000000ull;
  return b == 0x000fffffffffffffull ? 0ull : b;
}
__device__ __forceinline__ float from_order_bits(uint32_t b) {
  if (b == 0u) return __int_as_float(0xff800000);
  return __uint_as_float((b >> 31) ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ double from_order_bits(unsigned long long b) {
  if (b == 0ull) return __longlong_as_double(0xfff0000000000000LL);
  return __longlong_as_double((long long)((b >> 63) ? b ^ 0x8000000000000000ull : ~b));
}
template <typename K>
struct OrderBits;
template <>
struct OrderBits<float> { typedef uint32_t type; };
template <>
struct OrderBits<double> { typedef unsigned long long type; };

// Greatest value and sum over the L lanes of a token.
template <int L, typename B>
__device__ __forceinline__ B lanes_max(B v) {
  if constexpr (L == 32 && sizeof(B) == 4) {
    return __reduce_max_sync(FULL, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      const B u = __shfl_xor_sync(FULL, v, o);
      v = u > v ? u : v;
    }
    return v;
  }
}
template <int L, typename K>
__device__ __forceinline__ K lanes_sum(K v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
template <typename K>
__device__ __forceinline__ K warp_sum_of(K v) { return lanes_sum<32>(v); }

// The bits of a ballot that belong to this token's lanes.
template <int L>
__device__ __forceinline__ unsigned lanes_of(unsigned ballot, int lane) {
  if constexpr (L == 32) return ballot;
  else return (ballot >> (lane & ~(L - 1))) & ((1u << L) - 1u);
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// What a pass over one token finds: lane j < k of its lanes holds choice j.
struct Chosen {
  int expert;      // or -1
  bool unsure;     // (32 bits) two values that the choice hangs on lie closer than they are exact
};

// Scores, keys, groups and choice of one token in arithmetic of type K.
//
// In 32 bits the keys carry rounding errors, and two keys closer than `margin` may be in the wrong
// order.  The errors, in 2^-24 of the largest score and key: the exponentials in the sum of the scores 4 and its
// V + 5 additions, which move both keys of a pair alike; for each of the two the exponential 4, its argument's
// rounding |x - top| against a factor exp(x - top) 1, the quotient 1 and the bias's addition 1; the margin's own
// subtraction 1.  That makes V + 24.  A token with such a pair (about one in a hundred) is done again in 64
// bits, which is what the definition says.  Equal logits with equal biases have equal keys and need no second
// look; so each choice is compared with the next, and the last one with all that was not chosen and is not its
// equal.
template <typename K, int L, int V, bool PLAIN, typename T>
__device__ __forceinline__ Chosen route_token(const RouteParams& p, const T* row, const float (&x)[V], int lane,
                                              bool by_logit, float* s_keys) {
  typedef typename OrderBits<K>::type B;
  constexpr bool narrow = sizeof(K) == 4;
  const int sub = lane & (L - 1), e0 = sub * V;
  const K ninf = -(K)INFINITY;
  K key[V];
  K margin = 0;
  if (PLAIN || by_logit) {
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = (K)x[i];
  } else {
    K top_score = 1;
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = (K)1 / ((K)1 + exp_of(-(K)x[i]));
    } else {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) t = max(t, order_bits(x[i]));
      t = lanes_max<L>(t);
      const K top = t == 0xffffffffu ? (K)NAN : t == 0u ? (K)0 : (K)from_order_bits(t);
      K sum = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        key[i] = exp_of((K)x[i] - top);
        sum += key[i];
      }
      sum = lanes_sum<L>(sum);
      sum = sum == (K)0 ? (K)1 : sum;
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = key[i] / sum;
      top_score = (K)1 / sum;
    }
    K most = 0;
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = e0 + i;
        if (e < p.n_experts) key[i] += (K)p.bias[e];
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (x[i] == -INFINITY) key[i] = ninf;
      if (narrow && key[i] > ninf) most = fmaxf((float)most, fabsf((float)key[i]));
    }
    if (narrow) {
      const uint32_t m = lanes_max<L>(__float_as_uint((float)most));
      margin = (K)((float)(V + 24) * 0x1p-24f) * (top_score + (K)__uint_as_float(m));
    }
  }
  bool unsure = false;

  if (!PLAIN && L == 32 && p.groups > 1) {
    // lane g works out the score of group g from the keys in shared memory
    K* keys = reinterpret_cast<K*>(s_keys);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e0 + i < p.n_experts) keys[e0 + i] = key[i];
    __syncwarp();
    K score = ninf;
    B bits = 0;
    if (lane < p.groups) {
      const K* mine = keys + lane * p.group_size;
      B b1 = 0, b2 = 0;      // the two greatest of the group
      K v1 = ninf, v2 = ninf;
      for (int i = 0; i < p.group_size; ++i) {
        const K v = mine[i];
        const B b = order_bits(v);
        if (b > b1) {
          b2 = b1; v2 = v1;
          b1 = b; v1 = v;
        } else if (b > b2) {
          b2 = b; v2 = v;
        }
      }
      score = p.group_best == 2 ? v1 + v2 : v1;
      bits = order_bits(score);
    }
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const B other = __shfl_sync(FULL, bits, g);
      if (other > bits || (other == bits && g < lane)) ++rank;
    }
    const bool kept = lane < p.groups && rank < p.topk_groups;
    if (narrow && !by_logit) {
      const unsigned last_m = __ballot_sync(FULL, lane < p.groups && rank == p.topk_groups - 1);
      const unsigned next_m = __ballot_sync(FULL, lane < p.groups && rank == p.topk_groups);
      if (next_m) {
        const K a = __shfl_sync(FULL, score, __ffs(last_m) - 1), b = __shfl_sync(FULL, score, __ffs(next_m) - 1);
        if (a > ninf && !(a - b > 3 * margin)) unsure = true;
      }
    }
    const unsigned mask = __ballot_sync(FULL, kept);
    int g = e0 / p.group_size, left = (g + 1) * p.group_size - e0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // without a bias the order of the scores is the logits' own, and that is exact
      if (!((mask >> (g & 31)) & 1u)) key[i] = ninf;
      else if (!p.bias) key[i] = (K)x[i];
      if (--left == 0) {
        ++g;
        left = p.group_size;
      }
    }
  }

  B bits[V];
#pragma unroll
  for (int i = 0; i < V; ++i) bits[i] = e0 + i < p.n_experts ? order_bits(key[i]) : (B)0;
  Chosen c = {-1, false};
  B mine = 0, next = 0;
  int next_e = -1;
  for (int j = 0; j < p.k; ++j) {
    B best = bits[0];
#pragma unroll
    for (int i = 1; i < V; ++i) best = best > bits[i] ? best : bits[i];
    const B top = lanes_max<L>(best);
    const unsigned won = lanes_of<L>(__ballot_sync(FULL, best == top), lane);
    const int w = __ffs(won) - 1;
    int at = V - 1;
#pragma unroll
    for (int i = V - 2; i >= 0; --i) at = bits[i] == best ? i : at;
    if (sub == w) {
#pragma unroll
      for (int i = 0; i < V; ++i) bits[i] = i == at ? (B)0 : bits[i];
    }
    const int at_w = __shfl_sync(FULL, at, (lane & ~(L - 1)) + w);
    const int e = top == 0 ? -1 : at_w + w * V;
    if (sub == j) {
      c.expert = e;
      mine = top;
    }
    if (sub == j - 1) {
      next = top;
      next_e = e;
    }
  }
  if constexpr (!PLAIN && narrow) {
    if (p.bias) {
      const auto same = [&](int a, int b) { return p.bias[a] == p.bias[b] && to_float(row[a]) == to_float(row[b]); };
      bool close = c.expert >= 0 && next_e >= 0 && !(from_order_bits(mine) - from_order_bits(next) > margin);
      if (close && same(c.expert, next_e)) close = false;
      // what was not chosen: its key is still there
      const int last_lane = (lane & ~(L - 1)) + p.k - 1;
      const B least = order_bits(from_order_bits(__shfl_sync(FULL, mine, last_lane)) - margin);
      const int last = __shfl_sync(FULL, c.expert, last_lane);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (bits[i] != 0 && bits[i] >= least && !same(last, e0 + i)) close = true;
      unsure = unsure || lanes_of<L>(__ballot_sync(FULL, close), lane) != 0;
    }
  }
  c.unsure = unsure;
  return c;
}

// Choice by logits alone.  A key holds the upper bits of a logit's order and below them the expert, counted
// down, so that all keys of a token differ: a round is one maximum, and what it found is struck out wherever it
// lies.  The low bits that the expert takes are empty in logits of 16 bits.  Of two float32 logits that differ
// in nothing else the order may be wrong.  Equal upper bits lie side by side in the order of the keys, so it is
// right if the chosen of equal upper bits are equal each to the next, and no expert behind them that shares the
// last one's upper bits is greater than that one; else the token is done again with whole keys (`unsure`: about
// one in two hundred).  65 521 x 64 bfloat16, k = 6, took 17 us with whole keys; float32 logits gain nothing
// (16 384 x 128, k = 8: 10 us with whole keys, 9.4 with these), but lose nothing either.
template <typename T, int L, int V>
__device__ __forceinline__ Chosen route_by_logit(const RouteParams& p, const T* row, const float (&x)[V], int lane) {
  constexpr bool exact = sizeof(T) == 2;
  constexpr uint32_t LOW = L * V - 1;
  static_assert((L * V & (L * V - 1)) == 0 && L * V <= 1024, "an expert takes whole bits, ten at most");
  const int sub = lane & (L - 1), e0 = sub * V;
  uint32_t bits[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t b = order_bits(x[i]);       // behind the last expert x is -inf
    bits[i] = b == 0u ? 0u : (b & ~LOW) | (LOW - (uint32_t)(e0 + i));
  }
  uint32_t mine = 0, next = 0;
  for (int j = 0; j < p.k; ++j) {
    uint32_t top = bits[0];
#pragma unroll
    for (int i = 1; i < V; ++i) top = max(top, bits[i]);
    top = lanes_max<L>(top);
#pragma unroll
    for (int i = 0; i < V; ++i) bits[i] = bits[i] == top ? 0u : bits[i];
    if (sub == j) mine = top;
    if (!exact && sub == j - 1) next = top;
  }
  Chosen c = {mine ? (int)(LOW - (mine & LOW)) : -1, false};
  if (!exact) {
    bool close = mine != 0u && next != 0u && (mine & ~LOW) == (next & ~LOW);
    if (close)
      close = order_bits(to_float(row[LOW - (mine & LOW)])) != order_bits(to_float(row[LOW - (next & LOW)]));
    // what was not chosen: its key is still there
    const uint32_t last = __shfl_sync(FULL, mine, (lane & ~(L - 1)) + p.k - 1);
    bool cut = false;
#pragma unroll
    for (int i = 0; i < V; ++i) cut = cut || (bits[i] != 0u && (bits[i] & ~LOW) == (last & ~LOW));
    if (cut) {
      const uint32_t least = order_bits(to_float(row[LOW - (last & LOW)]));
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (bits[i] != 0u && (bits[i] & ~LOW) == (last & ~LOW)) close = close || order_bits(to_float(row[e0 + i])) > least;
    }
    c.unsure = lanes_of<L>(__ballot_sync(FULL, close), lane) != 0;
  }
  return c;
}

template <typename T, int V>
__device__ __forceinline__ void route_load(const T* row, int sub, int n_experts, int vec, float (&x)[V]) {
  const int e0 = sub * V;
  constexpr int BYTES = V * (int)sizeof(T);
  if (vec && e0 + V <= n_experts) {
    if constexpr (BYTES >= 16) {
      union { uint4 u[BYTES / 16]; T t[V]; } r;
#pragma unroll
      for (int j = 0; j < BYTES / 16; ++j) r.u[j] = reinterpret_cast<const uint4*>(row + e0)[j];
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = to_float(r.t[i]);
    } else {
      union { uint2 u; T t[V]; } r;
      r.u = *reinterpret_cast<const uint2*>(row + e0);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = to_float(r.t[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = e0 + i < n_experts ? to_float(row[e0 + i]) : -INFINITY;
}

// The pass with whole keys (PLAIN: the logits; else 64 bits), for the tokens that asked for it; all lanes of
// the warp take part.
template <typename T, int L, int V, bool PLAIN>
__device__ __noinline__ int route_again(const RouteParams& p, const T* row, int lane, float* s_keys) {
  float x[V];
  route_load<T, V>(row, lane & (L - 1), p.n_experts, p.vec, x);
  if constexpr (PLAIN) return route_token<float, L, V, true>(p, row, x, lane, true, s_keys).expert;
  else return route_token<double, L, V, false>(p, row, x, lane, false, s_keys).expert;
}

__device__ __forceinline__ float sigmoid_of(float x) {
  // exp(-|x|) never leaves the range, and keeps the small scores of negative logits
  const float t = expf(-fabsf(x));
  return (x < 0.f ? t : 1.f) / (1.f + t);
}

// Share of each lane's choice among the choices of its token (sum 1), 0 where there is none.
// Softmax: exp(x - top of the chosen) over its sum.  Sigmoid: s over its sum, with exp(x) for s
// where all chosen logits lie below -60 (there s = exp(x) to 2^-80, and s itself runs out of range).
template <int L>
__device__ __forceinline__ float share_of(bool there, float x, bool sigmoid) {
  const uint32_t t = lanes_max<L>(there ? order_bits(x) : 0u);
  const float top = from_order_bits(t);
  float s;
  if (sigmoid && !(top < -60.f)) s = sigmoid_of(x);
  else s = expf(x - top);
  if (t == 0xffffffffu) s = __uint_as_float(0x7fffffffu);
  if (!there) s = 0.f;
  const float sum = lanes_sum<L>(s);
  return there ? s / sum : 0.f;
}

// (top, sum of exp(x - top)) of a token's logits; top 0 where nothing but -inf is there.
template <int L, int V>
__device__ __forceinline__ void softmax_stats(const float (&x)[V], float& top, float& sum) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) t = max(t, order_bits(x[i]));
  t = lanes_max<L>(t);
  top = t == 0u ? 0.f : t == 0xffffffffu ? __uint_as_float(0x7fffffffu) : from_order_bits(t);
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) sum += expf(x[i] - top);
  sum = lanes_sum<L>(sum);
  if (sum == 0.f) sum = 1.f;
}

// PLAIN: experts ordered by their logits, no groups: nothing is left of the keys, and half the registers.
template <typename T, int L, int V, bool PLAIN>
__global__ void __launch_bounds__(RT_WARPS * 32)
route_topk_kernel(const __grid_constant__ RouteParams p) {
  // groups: one row of keys per warp, wide enough for 64-bit keys
  extern __shared__ __align__(16) float s_route[];
  next_grid_may_start();
  grid_dependency_wait();
  constexpr int PER = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (L - 1);
  float* s_keys = s_route + (size_t)warp * 2 * p.n_experts;
  const bool by_logit = PLAIN || (p.bias == nullptr && (p.groups == 1 || p.group_best == 1));
  const int64_t step = (int64_t)gridDim.x * RT_WARPS * PER;
  for (int64_t i0 = ((int64_t)blockIdx.x * RT_WARPS + warp) * PER; i0 < p.n; i0 += step) {
    const int64_t mine = i0 + lane / L;
    const int64_t i = mine < p.n ? mine : p.n - 1;       // lanes without a token repeat the last one
    const T* row = (const T*)p.logits + i * p.n_experts;
    float x[V];
    route_load<T, V>(row, sub, p.n_experts, p.vec, x);
    Chosen c;
    if constexpr (PLAIN) c = route_by_logit<T, L, V>(p, row, x, lane);
    else c = route_token<float, L, V, false>(p, row, x, lane, by_logit, s_keys);
    if (__any_sync(FULL, c.unsure)) {
      const int e = route_again<T, L, V, PLAIN>(p, row, lane, s_keys);
      if (c.unsure) c.expert = e;
    }
    const bool there = c.expert >= 0;
    const float xe = there ? to_float(row[c.expert]) : 0.f;
    float w;
    float top = 0.f, sum = 1.f;
    const bool stats = !p.sigmoid && (!p.renormalize || !by_logit);
    if (stats) softmax_stats<L, V>(x, top, sum);
    if (p.renormalize) {
      w = share_of<L>(there, xe, p.sigmoid != 0);
      if (stats && sum != sum) w = sum;            // a NaN that was not chosen still is in every score
    } else {
      w = p.sigmoid ? sigmoid_of(xe) : expf(xe - top) / sum;
    }
    if (sub < p.k && mine < p.n) {
      p.weights[i * p.k + sub] = there ? w * p.scale : 0.f;
      p.experts[i * p.k + sub] = c.expert;
    }
  }
}

struct RouteGradParams {
  const void* logits;
  const int32_t* experts;
  const float* grad_weights;
  void* grad_logits;
  int64_t n;
  int n_experts, k;
  int sigmoid, renormalize, vec;
  float scale;
};

// Gradient of the weights to the logits.  With p the shares and g = scale * grad of the chosen:
//   softmax, renormalised   p_j (g_j - sum p g)                 on the chosen, 0 elsewhere
//   sigmoid, renormalised   p_j (g_j - sum p g) (1 - s_j)       on the chosen
//   sigmoid                 g_j s_j (1 - s_j)                   on the chosen
//   softmax                 s_e ([e chosen] g_e - sum s g)      everywhere
// 1 - s is the sigmoid of the negative logit: the difference of 1 and s would lose it bit by bit (0.9 % off at
// a logit of 12, nothing left at 17).
// A token's lanes write the row's dense part and then, ordered by __syncwarp, the chosen places.
template <typename T, int L, int V>
__global__ void __launch_bounds__(RT_WARPS * 32)
route_topk_grad_kernel(const __grid_constant__ RouteGradParams p) {
  next_grid_may_start();
  grid_dependency_wait();
  constexpr int PER = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (L - 1), e0 = sub * V;
  const bool dense = !p.sigmoid && !p.renormalize;
  const int64_t step = (int64_t)gridDim.x * RT_WARPS * PER;
  for (int64_t i0 = ((int64_t)blockIdx.x * RT_WARPS + warp) * PER; i0 < p.n; i0 += step) {
    const int64_t mine = i0 + lane / L;
    const bool live = mine < p.n;
    const int64_t i = live ? mine : p.n - 1;
    const T* row = (const T*)p.logits + i * p.n_experts;
    T* out = (T*)p.grad_logits + i * p.n_experts;
    int e = -1;
    float g = 0.f, xe = -INFINITY;
    if (sub < p.k) {
      e = p.experts[i * p.k + sub];
      if (e >= p.n_experts) e = -1;
      if (e >= 0) {
        g = p.grad_weights[i * p.k + sub] * p.scale;
        xe = to_float(row[e]);
      }
    }
    const bool there = e >= 0;
    float d = 0.f;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (dense) {
      float x[V], top, sum;
      route_load<T, V>(row, sub, p.n_experts, p.vec, x);
      softmax_stats<L, V>(x, top, sum);
      const float s = there ? expf(xe - top) / sum : 0.f;
      const float dot = lanes_sum<L>(s * g);
      const float inv = 1.f / sum;
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = -(expf(x[j] - top) * inv) * dot;
      d = s * (g - dot);
    } else if (p.renormalize) {
      const float share = share_of<L>(there, xe, p.sigmoid != 0);
      const float dot = lanes_sum<L>(share * g);
      d = share * (g - dot);
      if (p.sigmoid) d *= sigmoid_of(-xe);
    } else {
      d = g * sigmoid_of(xe) * sigmoid_of(-xe);
    }
    constexpr int BYTES = V * (int)sizeof(T);
    if (!live) {
    } else if (p.vec && e0 + V <= p.n_experts) {
      union { uint4 u4[(BYTES + 15) / 16]; uint2 u2; T t[V]; } r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.t[j] = from_float<T>(v[j]);
      if constexpr (BYTES >= 16) {
#pragma unroll
        for (int j = 0; j < BYTES / 16; ++j) reinterpret_cast<uint4*>(out + e0)[j] = r.u4[j];
      } else {
        *reinterpret_cast<uint2*>(out + e0) = r.u2;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j < p.n_experts) out[e0 + j] = from_float<T>(v[j]);
    }
    __syncwarp();
    if (there && live) out[e] = from_float<T>(d);
    __syncwarp();
  }
}

template <typename T>
bool route_rows_are_vec(const void* a, const void* b, int n_experts, int v) {
  const int64_t bytes = (int64_t)v * sizeof(T) < 16 ? (int64_t)v * sizeof(T) : 16;
  return (((uintptr_t)a | (uintptr_t)b) % bytes) == 0 && (n_experts * (int64_t)sizeof(T)) % bytes == 0;
}

// Lanes and experts per lane: eight experts in registers, and as few lanes as hold the token's experts
// and its choices, so that a reduction serves several tokens.
#define KMB_ROUTE_WIDTHS(wide, RUN)                                                             \
  do {                                                                                          \
    if (!(wide) && p.n_experts <= 32 && p.k <= 8) { RUN(8, 4); }                                \
    else if (!(wide) && p.n_experts <= 64 && p.k <= 8) { RUN(8, 8); }                           \
    else if (!(wide) && p.n_experts <= 128 && p.k <= 16) { RUN(16, 8); }                        \
    else if (p.n_experts <= 128) { RUN(32, 4); }                                                \
    else if (p.n_experts <= 256) { RUN(32, 8); }                                                \
    else if (p.n_experts <= 512) { RUN(32, 16); }                                               \
    else { RUN(32, 32); }                                                                       \
  } while (0)

static unsigned route_grid(int64_t n, int lanes) {
  const int64_t blocks = ceil_div(n, RT_WARPS * (32 / lanes)), cap = (int64_t)sm_count() * 16;
  return (unsigned)(blocks < cap ? blocks : cap);
}

template <typename T>
int route_run(RouteParams p, cudaStream_t s) {
  const size_t smem = p.groups > 1 ? (size_t)RT_WARPS * 2 * p.n_experts * sizeof(float) : 0;
#define KMB_RUN(L, V)                                                                           \
  p.vec = route_rows_are_vec<T>(p.logits, nullptr, p.n_experts, V);                             \
  return launch_early(p.bias == nullptr && p.groups == 1 ? route_topk_kernel<T, L, V, true>     \
                                                         : route_topk_kernel<T, L, V, false>,   \
                      route_grid(p.n, L), RT_WARPS * 32, smem, 1, s, p)
  KMB_ROUTE_WIDTHS(p.groups > 1, KMB_RUN);
#undef KMB_RUN
}

template <typename T>
int route_grad_run(RouteGradParams p, cudaStream_t s) {
#define KMB_RUN(L, V)                                                                           \
  p.vec = route_rows_are_vec<T>(p.logits, p.grad_logits, p.n_experts, V);                       \
  return launch_early(route_topk_grad_kernel<T, L, V>, route_grid(p.n, L), RT_WARPS * 32, 0, 1, s, p)
  KMB_ROUTE_WIDTHS(false, KMB_RUN);
#undef KMB_RUN
}

// ============================================================================= expert order
// A stable counting sort of the choices by expert.  A block takes SL_CHUNK consecutive choices, a warp
// of it SL_ROUNDS * 32 of them; one ballot for each bit of the expert finds the equal ones of 32 choices
// (match_any, which walks the distinct values, took twice as long), the warp's own counters carry the
// rank from round to round, and the counters of the warps before it, the chunks before it and the
// experts before it make the place.  1 048 568 choices of 256 experts take 15.6 us in three launches: 3.5
// counting, 2.8 scanning, 10 placing: 170 instructions for 32 choices at 0.55 a scheduler and cycle, in 256 blocks of
// which some SMs get two and some one; the 12.6 MB that it moves would take 1.9.
constexpr int SL_WARPS = 16, SL_ROUNDS = 8;
constexpr int SL_THREADS = SL_WARPS * 32;
constexpr int SL_CHUNK = SL_THREADS * SL_ROUNDS;
constexpr int SL_MAX_EXPERTS = 1024;

// counts[chunk][e] for every chunk
__global__ void __launch_bounds__(SL_THREADS)
slots_count_kernel(const int32_t* experts, int64_t total, int n_experts,
                   int32_t* __restrict__ counts) {
  __shared__ int32_t s_cnt[SL_MAX_EXPERTS];
  next_grid_may_start();
  grid_dependency_wait();
  for (int e = threadIdx.x; e < n_experts; e += SL_THREADS) s_cnt[e] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * SL_CHUNK;
#pragma unroll
  for (int r = 0; r < SL_ROUNDS; ++r) {
    const int64_t c = first + r * SL_THREADS + threadIdx.x;
    const int e = c < total ? experts[c] : -1;
    if (e >= 0 && e < n_experts) atomicAdd(&s_cnt[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_experts; e += SL_THREADS)
    counts[(int64_t)blockIdx.x * n_experts + e] = s_cnt[e];
}

// counts[chunk][e] -> choices of expert e in the chunks before; totals[e].  A block takes 32 experts; each
// of its 32 warps sums (and then rewrites) a run of SC_RUN chunks, its lanes one expert each.
constexpr int SC_RUN = 8;
__global__ void __launch_bounds__(1024)
slots_scan_kernel(int32_t* __restrict__ counts, int chunks, int n_experts, int32_t* __restrict__ totals) {
  __shared__ int32_t s_sum[32][33];
  next_grid_may_start();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = blockIdx.x * 32 + lane;
  const bool mine = e < n_experts;
  int carry = 0;
  for (int c0 = 0; c0 < chunks; c0 += 32 * SC_RUN) {
    int v[SC_RUN], sum = 0;
#pragma unroll
    for (int r = 0; r < SC_RUN; ++r) {
      const int c = c0 + warp * SC_RUN + r;
      v[r] = mine && c < chunks ? counts[(int64_t)c * n_experts + e] : 0;
    }
#pragma unroll
    for (int r = 0; r < SC_RUN; ++r) sum += v[r];
    s_sum[warp][lane] = sum;
    __syncthreads();
    // warp w scans the 32 runs of expert w of the block
    const int x = s_sum[lane][warp];
    int inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(FULL, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    s_sum[lane][warp] = inc;
    __syncthreads();
    int base = carry + s_sum[warp][lane] - sum;
    carry += s_sum[31][lane];
#pragma unroll
    for (int r = 0; r < SC_RUN; ++r) {
      const int c = c0 + warp * SC_RUN + r;
      if (mine && c < chunks) counts[(int64_t)c * n_experts + e] = base;
      base += v[r];
    }
    __syncthreads();
  }
  if (warp == 0 && mine) totals[e] = carry;
}

constexpr size_t slots_place_smem(int n_experts) {
  return (size_t)n_experts * (2 * sizeof(int32_t) + SL_WARPS * sizeof(uint16_t));
}

// ONE: a single chunk, whose counts are the totals.
template <bool ONE>
__global__ void __launch_bounds__(SL_THREADS)
slots_place_kernel(const int32_t* experts, int64_t total, int k, int n_experts,
                   const int32_t* counts, const int32_t* totals,
                   int32_t* __restrict__ slots, int32_t* __restrict__ rows, int32_t* __restrict__ offsets) {
  extern __shared__ int32_t s_dyn[];
  int32_t* s_base = s_dyn;                            // first place of each expert in this chunk
  int32_t* s_local = s_dyn + n_experts;               // and among the chunk's own choices
  uint16_t* s_warp = (uint16_t*)(s_dyn + 2 * n_experts);  // [SL_WARPS][n_experts] choices in the warp
  // the chunk's choices in expert order: (place, row), so that the rows of an expert leave side by side
  __shared__ int2 s_out[SL_CHUNK];
  __shared__ int32_t s_count;
  __shared__ int2 s_scan[SL_WARPS];
  __shared__ int32_t s_end;
  next_grid_may_start();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t first = (int64_t)blockIdx.x * SL_CHUNK + warp * (SL_ROUNDS * 32);

  int32_t e_r[SL_ROUNDS];
#pragma unroll
  for (int r = 0; r < SL_ROUNDS; ++r) {
    const int64_t c = first + r * 32 + lane;
    const int e = c < total ? experts[c] : -1;
    e_r[r] = e >= 0 && e < n_experts ? e : -1;
  }
  uint16_t* mine = s_warp + warp * n_experts;
  for (int e = lane; e < n_experts; e += 32) mine[e] = 0;
  __syncwarp();
  uint32_t rank[SL_ROUNDS];
#pragma unroll
  for (int r = 0; r < SL_ROUNDS; ++r) {
    const bool valid = e_r[r] >= 0;
    unsigned same = __ballot_sync(FULL, valid);
#pragma unroll
    for (int b = 0; b < 10; ++b) {
      if (b == 8 && n_experts <= 256) break;       // no expert has these bits
      const bool one = (e_r[r] >> b) & 1;
      const unsigned m = __ballot_sync(FULL, one);
      same &= one ? m : ~m;
    }
    const int before = __popc(same & ((1u << lane) - 1u));
    const uint32_t seen = valid ? mine[e_r[r]] : 0u;
    rank[r] = seen + before;
    __syncwarp();
    if (valid && before == 0) mine[e_r[r]] = (uint16_t)(seen + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  // warps' counts -> choices in the warps before; then the experts' first places
  int carry = 0, carry_local = 0;
  for (int e0 = 0; e0 < n_experts; e0 += SL_THREADS) {
    const int e = e0 + threadIdx.x;
    int in_chunk = 0;
    if (e < n_experts) {
#pragma unroll
      for (int w = 0; w < SL_WARPS; ++w) {
        const int v = s_warp[w * n_experts + e];
        s_warp[w * n_experts + e] = (uint16_t)in_chunk;
        in_chunk += v;
      }
    }
    const int tot = e < n_experts ? (ONE ? in_chunk : totals[e]) : 0;
    const int before = e < n_experts && !ONE ? counts[(int64_t)blockIdx.x * n_experts + e] : 0;
    int inc = tot, inc_local = in_chunk;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(FULL, inc, o), ul = __shfl_up_sync(FULL, inc_local, o);
      if (lane >= o) {
        inc += u;
        inc_local += ul;
      }
    }
    if (lane == 31) s_scan[warp] = make_int2(inc, inc_local);
    __syncthreads();
    int base = carry, base_local = carry_local;
#pragma unroll
    for (int w = 0; w < SL_WARPS; ++w) {
      const int2 v = s_scan[w];
      if (w < warp) {
        base += v.x;
        base_local += v.y;
      }
      carry += v.x;
      carry_local += v.y;
    }
    if (e < n_experts) {
      const int start = base + inc - tot;
      s_base[e] = start + before;
      s_local[e] = base_local + inc_local - in_chunk;
      if (blockIdx.x == 0) offsets[e] = start;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    s_end = carry;
    s_count = carry_local;
    if (blockIdx.x == 0) offsets[n_experts] = carry;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SL_ROUNDS; ++r) {
    const int64_t c = first + r * 32 + lane;
    if (c >= total) continue;
    const int e = e_r[r];
    int place = -1;
    if (e >= 0) {
      const int in_chunk = mine[e] + (int)rank[r];
      place = s_base[e] + in_chunk;
      s_out[s_local[e] + in_chunk] = make_int2(place, (int32_t)((uint32_t)c / (uint32_t)k));
    }
    slots[c] = place;
    if (c >= s_end) rows[c] = -1;      // places behind the last chosen row
  }
  __syncthreads();
  for (int i = threadIdx.x; i < s_count; i += SL_THREADS) rows[s_out[i].x] = s_out[i].y;
}

// ============================================================================= weighted sums
// out[t] = sum_j w[t, j] values[slots[t, j]]; a slot outside [0, n_values) counts as none.
constexpr int CB_THREADS = 256;   // at most; the launch takes as many as a row needs (combine_threads)
constexpr int CB_MAX_D = 1 << 30; // places in a row, a block's pass behind its end among them, fit 32 bits
constexpr int CB_K = 8;           // rows that a thread asks for before it adds the first
constexpr int CG_THREADS = 128, CG_K = 4;   // the gradients', which hold twice as much per row

// Eight elements of a row as they lie in memory.  VEC: consecutive ones of a row of whole 16-byte pieces
// (eight floats are two of them, the second of which may lie behind the row); else one in
// blockDim.x, so that neighbouring threads read neighbouring elements of a row that starts anywhere.
template <typename T, bool VEC>
struct RowPiece {
  alignas(16) T t[8];
  __device__ __forceinline__ static int span() { return blockDim.x * 8; }     // elements of a block's pass
  static constexpr int PER_QUAD = 16 / (int)sizeof(T), QUADS = 8 / PER_QUAD;
  __device__ __forceinline__ static int at(int f0, int j) {
    return VEC ? f0 + threadIdx.x * 8 + j : f0 + threadIdx.x + j * blockDim.x;
  }
  __device__ __forceinline__ void load(const T* row, int f0, int d) {
    if constexpr (VEC) {
      uint4* dst = reinterpret_cast<uint4*>(t);
#pragma unroll
      for (int q = 0; q < QUADS; ++q)
        if (at(f0, q * PER_QUAD) < d) dst[q] = *reinterpret_cast<const uint4*>(row + at(f0, q * PER_QUAD));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(f0, j) < d) t[j] = row[at(f0, j)];
    }
  }
  __device__ __forceinline__ void store(T* __restrict__ row, int f0, int d) const {
    if constexpr (VEC) {
      const uint4* src = reinterpret_cast<const uint4*>(t);
#pragma unroll
      for (int q = 0; q < QUADS; ++q)
        if (at(f0, q * PER_QUAD) < d) *reinterpret_cast<uint4*>(row + at(f0, q * PER_QUAD)) = src[q];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(f0, j) < d) row[at(f0, j)] = t[j];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_float<T>(0.f);
  }
};

// Bound by HBM: each thread asks for the pieces of up to CB_K rows before it adds the first.  8192 tokens of
// eight rows of 2048 bfloat16 take 50 to 55 us (302 MB, 5.5 to 6.0 TB/s), 8191 of six rows of 1031 float32,
// which start anywhere and of which one in nine is not there, 46 us (214 MB, 4.6 TB/s).  (Copying rows ahead into shared memory with cp.async was no
// faster, 54 and 64 us.)
template <typename T, bool VEC>
__global__ void __maxnreg__(96)      // four blocks of 160 threads on an SM
combine_kernel(const T* values, int64_t n_values, const int32_t* slots,
               const float* weights, int k, int d, T* __restrict__ out, int parts) {
  typedef RowPiece<T, VEC> Piece;
  next_grid_may_start();
  grid_dependency_wait();
  const int64_t t = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - t * parts);
  for (int f0 = part * Piece::span(); f0 < d; f0 += parts * Piece::span()) {
    if (Piece::at(f0, 0) >= d) continue;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < k; j0 += CB_K) {
      Piece v[CB_K];
      float w[CB_K];
#pragma unroll
      for (int j = 0; j < CB_K; ++j) {
        const int slot = j0 + j < k ? slots[t * k + j0 + j] : -1;
        w[j] = 0.f;
        v[j].clear();
        if (slot >= 0 && slot < n_values) {
          w[j] = weights[t * k + j0 + j];
          v[j].load(values + (int64_t)slot * d, f0, d);
        }
      }
#pragma unroll
      for (int j = 0; j < CB_K; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(w[j], to_float(v[j].t[i]), acc[i]);
    }
    Piece o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.t[i] = from_float<T>(acc[i]);
    o.store(out + t * d, f0, d);
  }
}

// Gradients.  Bound by HBM: the same 8192 x 8 rows of 2048 bfloat16 take 92.5 us with the two small kernels ahead (571 MB
// read and written, of which 528 reach DRAM at 6.0 TB/s, the rest being found in L2).  A block takes CG_K choices of
// a token, 128 threads (with 256 threads the large kernel alone took 111 us, with 128 85).  A row of values that several choices share needs the sum of their gradients, in a fixed
// order.  `users` counts the choices of each row; where the workspace has room for `next`, one number for each choice,
// `head` and `next` chain them in the order in which they came, and else `head` is the lowest of them.  The
// blocks of the tokens write the rows with one user, the last blocks of the grid all others.
__device__ __forceinline__ void combine_clear_row(int64_t r, int32_t* users, int32_t* head, const int32_t* next) {
  users[r] = 0;
  head[r] = next ? -1 : INT_MAX;
}
// Returns the choice that came before in the chain (or -1).
__device__ __forceinline__ int32_t combine_note_user(int32_t c, int32_t slot, int32_t* users, int32_t* head,
                                                     const int32_t* next) {
  atomicAdd(&users[slot], 1);
  if (next) return atomicExch(&head[slot], c);
  atomicMin(&head[slot], c);
  return -1;
}

__global__ void combine_clear_kernel(int64_t n_values, int32_t* users, int32_t* head, const int32_t* next) {
  next_grid_may_start();
  grid_dependency_wait();
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r < n_values) combine_clear_row(r, users, head, next);
}

__global__ void combine_users_kernel(const int32_t* slots, int64_t total, int64_t n_values, int32_t* users, int32_t* head,
                                     int32_t* next) {
  next_grid_may_start();
  grid_dependency_wait();
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= total) return;
  const int slot = slots[c];
  if (slot < 0 || slot >= n_values) return;
  const int32_t before = combine_note_user((int32_t)c, slot, users, head, next);
  if (next) next[c] = before;
}

// Both for few rows and choices, in one launch and in shared memory.
constexpr int CG_FEW = 8192, CG_FEW_THREADS = 1024;
__global__ void __launch_bounds__(CG_FEW_THREADS)
combine_few_users_kernel(const int32_t* slots, int total, int n_values, int32_t* users, int32_t* head, int32_t* next) {
  extern __shared__ int32_t s_few[];
  int32_t* s_users = s_few;
  int32_t* s_head = s_few + n_values;
  next_grid_may_start();
  for (int r = threadIdx.x; r < n_values; r += CG_FEW_THREADS) combine_clear_row(r, s_users, s_head, next);
  __syncthreads();
  grid_dependency_wait();
  for (int c = threadIdx.x; c < total; c += CG_FEW_THREADS) {
    const int slot = slots[c];
    if (slot < 0 || slot >= n_values) continue;
    const int32_t before = combine_note_user(c, slot, s_users, s_head, next);
    if (next) next[c] = before;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < n_values; r += CG_FEW_THREADS) {
    users[r] = s_users[r];
    head[r] = s_head[r];
  }
}

// acc += the gradients of the `found` choices in `list`, in its order.
template <typename T, bool VEC>
__device__ __forceinline__ void combine_add_users(const int32_t* list, int found, const float* weights, const T* grad_out,
                                                  int k, int f0, int d, float (&acc)[8]) {
  for (int q = 0; q < found; ++q) {
    const uint32_t c = (uint32_t)list[q];
    const float w = weights[c];
    RowPiece<T, VEC> g;
    g.clear();
    g.load(grad_out + (int64_t)(c / (uint32_t)k) * d, f0, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, to_float(g.t[i]), acc[i]);
  }
}

// The rows that have no user or several: zeros, or the sum over the users in ascending order.  A row's users come
// from its chain, which one thread follows (0.6 us a user) and the block sorts; or, without chains and for rows of
// more than `most_chained` users, from a walk over the choices, CG_WALK of them to a thread at a time (1 us for each
// 1024).  The walk alone costs rows times choices: 4096 rows of 64 users and 64 floats took 189 ms with it, 0.31 with
// chains; one row of 65 536 users takes 8.4 ms.  Block `block` of `blocks` looks at `batch` rows at once.
constexpr int CG_LIST = 2048, CG_WALK = 8;
static_assert(CG_LIST >= CG_THREADS * CG_WALK, "the choices of one step of the walk may all be users");
template <typename T, bool VEC>
__device__ __noinline__ void combine_other_rows(int64_t block, int64_t blocks, int batch, int64_t n_values,
                                                const int32_t* slots, const float* weights,
                                                const T* grad_out, int64_t choices, int k, int d,
                                                const int32_t* users, const int32_t* head, const int32_t* next,
                                                int most_chained, T* __restrict__ grad_values) {
  typedef RowPiece<T, VEC> Piece;
  __shared__ int32_t list[CG_LIST], other[CG_THREADS];
  __shared__ int list_n[CG_WALK][CG_THREADS / 32], other_n[CG_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x / 32;
  const unsigned below = (1u << lane) - 1u;
  for (int64_t base = block * batch; base < n_values; base += blocks * batch) {
    const int64_t mine = base + threadIdx.x;
    const bool odd = (int)threadIdx.x < batch && mine < n_values && users[mine] != 1;
    if (!__syncthreads_or(odd)) continue;
    const unsigned odd_m = __ballot_sync(FULL, odd);
    if (lane == 0) other_n[warp] = __popc(odd_m);
    __syncthreads();
    int place = 0, others = 0;
    for (int q = 0; q < warps; ++q) {
      if (q < warp) place += other_n[q];
      others += other_n[q];
    }
    if (odd) other[place + __popc(odd_m & below)] = (int32_t)threadIdx.x;
    __syncthreads();
    for (int o = 0; o < others; ++o) {
      const int64_t r = base + other[o];
      const int count = users[r];
      const bool chained = next != nullptr && count <= most_chained;
      if (chained && count > 0) {
        int size = 1;
        while (size < count) size *= 2;
        if (threadIdx.x == 0)
          for (int q = 0, c = head[r]; q < count; ++q, c = next[c]) list[q] = c;
        for (int q = count + threadIdx.x; q < size; q += blockDim.x) list[q] = INT_MAX;
        __syncthreads();
        // bitonic: runs of `run` places are sorted, up and down in turn
        for (int run = 2; run <= size; run *= 2)
          for (int gap = run / 2; gap > 0; gap /= 2) {
            for (int q = threadIdx.x; q < size; q += blockDim.x)
              if (!(q & gap)) {
                const int a = list[q], b = list[q + gap];
                if ((a > b) == ((q & run) == 0)) {
                  list[q] = b;
                  list[q + gap] = a;
                }
              }
            __syncthreads();
          }
      }
      for (int f0 = 0; f0 < d; f0 += Piece::span()) {
        const bool in = Piece::at(f0, 0) < d;
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.f;
        if (chained) {
          if (in) combine_add_users<T, VEC>(list, count, weights, grad_out, k, f0, d, acc);
        } else {
          int left = count;
          for (int64_t cb = next ? 0 : count ? head[r] : choices; left > 0 && cb < choices; cb += CG_WALK * blockDim.x) {
            unsigned m[CG_WALK];
#pragma unroll
            for (int u = 0; u < CG_WALK; ++u) {
              const int64_t c = cb + u * blockDim.x + threadIdx.x;
              m[u] = __ballot_sync(FULL, c < choices && slots[c] == r);
            }
            if (lane == 0) {
#pragma unroll
              for (int u = 0; u < CG_WALK; ++u) list_n[u][warp] = __popc(m[u]);
            }
            __syncthreads();
            int found = 0;
#pragma unroll
            for (int u = 0; u < CG_WALK; ++u)
              for (int q = 0; q < warps; ++q) {
                if (q == warp && ((m[u] >> lane) & 1u))
                  list[found + __popc(m[u] & below)] = (int32_t)(cb + u * blockDim.x + threadIdx.x);
                found += list_n[u][q];
              }
            __syncthreads();
            if (in) combine_add_users<T, VEC>(list, found, weights, grad_out, k, f0, d, acc);
            left -= found;
            __syncthreads();
          }
        }
        Piece out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out.t[i] = from_float<T>(acc[i]);
        if (in) out.store(grad_values + r * d, f0, d);
      }
      __syncthreads();       // the list is free again
    }
  }
}

// Nine blocks on an SM where the registers of the token's part allow it, eight else; the other rows' part
// takes what that leaves (64 registers for both, and so eight blocks, took 94 us where nine take 92).
template <typename T, bool VEC>
constexpr int combine_grad_blocks() { return VEC && std::is_same<T, __nv_bfloat16>::value ? 9 : 8; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(CG_THREADS, (combine_grad_blocks<T, VEC>()))
combine_grad_kernel(const T* values, int64_t n_values, const int32_t* slots,
                    const float* weights, const T* grad_out, int64_t n, int k, int d,
                    const int32_t* users, const int32_t* head, const int32_t* next, int most_chained, int batch,
                    T* __restrict__ grad_values, float* __restrict__ grad_weights, int64_t token_blocks) {
  typedef RowPiece<T, VEC> Piece;
  __shared__ float red[CG_THREADS / 32][CG_K];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  next_grid_may_start();
  grid_dependency_wait();
  if ((int64_t)blockIdx.x >= token_blocks) {
    combine_other_rows<T, VEC>((int64_t)blockIdx.x - token_blocks, (int64_t)gridDim.x - token_blocks, batch, n_values,
                               slots, weights, grad_out, n * k, k, d, users, head, next, most_chained, grad_values);
    return;
  }
  // a block takes CG_K choices of a token
  const int parts = (k + CG_K - 1) / CG_K;
  const int64_t t = blockIdx.x / (unsigned)parts;
  const int j0 = (int)(blockIdx.x - t * parts) * CG_K;
  int slot[CG_K], used[CG_K];
  bool there[CG_K];
  float w[CG_K], dot[CG_K];
#pragma unroll
  for (int j = 0; j < CG_K; ++j) {
    const int64_t c = t * k + (j0 + j < k ? j0 + j : k - 1);
    slot[j] = slots[c];
    w[j] = weights[c];
    dot[j] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < CG_K; ++j) {
    there[j] = j0 + j < k && slot[j] >= 0 && slot[j] < n_values;
    slot[j] = there[j] ? slot[j] : 0;
    used[j] = n_values > 0 ? users[slot[j]] : 0;      // looked at when the first gradients are stored
  }
  for (int f0 = 0; f0 < d && n_values > 0; f0 += Piece::span()) {
    if (Piece::at(f0, 0) >= d) continue;
    Piece g, v[CG_K];
    g.clear();
    g.load(grad_out + t * d, f0, d);
#pragma unroll
    for (int j = 0; j < CG_K; ++j) {
      v[j].clear();
      if (there[j]) v[j].load(values + (int64_t)slot[j] * d, f0, d);
    }
#pragma unroll
    for (int j = 0; j < CG_K; ++j) {
      Piece o;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float gi = to_float(g.t[i]);
        dot[j] = fmaf(to_float(v[j].t[i]), gi, dot[j]);
        o.t[i] = from_float<T>(w[j] * gi);
      }
      if (there[j] && used[j] == 1) o.store(grad_values + (int64_t)slot[j] * d, f0, d);
    }
  }
#pragma unroll
  for (int j = 0; j < CG_K; ++j) {
    dot[j] = warp_sum_of(dot[j]);
    // 0 where there is no row, whatever the gradient holds
    if (lane == 0) red[warp][j] = there[j] ? dot[j] : 0.f;
  }
  __syncthreads();
  if (threadIdx.x < CG_K && j0 + threadIdx.x < k) {
    float sum = 0.f;
    for (int q = 0; q < (int)blockDim.x / 32; ++q) sum += red[q][threadIdx.x];
    grad_weights[t * k + j0 + threadIdx.x] = sum;     // 0 where there is no row
  }
}

// Threads for a row of d elements, eight to a thread: as few as do it in the fewest passes, so that a row a
// little longer than a round number leaves no block nearly idle.
static unsigned combine_threads(int d, int most) {
  const int64_t passes = ceil_div(d, most * 8);
  return (unsigned)(ceil_div(ceil_div(d, 8 * passes), 32) * 32);
}

static int check_route(const char* who, int n_experts, int k) {
  KMB_REQUIRE(n_experts >= 1 && n_experts <= RT_MAX_EXPERTS, "%s: the number of experts must be in [1, %d], got %d",
              who, RT_MAX_EXPERTS, n_experts);
  KMB_REQUIRE(k >= 1 && k <= RT_MAX_K && k <= n_experts,
              "%s: k must be in [1, %d] and at most the number of experts, got %d", who, RT_MAX_K, k);
  return KMB_OK;
}

}  // namespace kmb

using namespace kmb;

extern "C" {

int kmb_route_topk(int dtype, const void* logits, const float* bias, int64_t n, int n_experts, int k,
                   int flags, int groups, int topk_groups, int group_best, float scale, float* weights,
                   int32_t* experts, void* stream) {
  int rc = check_route("kmb_route_topk", n_experts, k);
  if (rc != KMB_OK) return rc;
  KMB_REQUIRE(n >= 0, "kmb_route_topk: bad sizes");
  KMB_REQUIRE((flags & ~(KMB_ROUTE_SIGMOID | KMB_ROUTE_RENORMALIZE)) == 0, "kmb_route_topk: unknown flag bits");
  KMB_REQUIRE(groups >= 1 && groups <= RT_MAX_GROUPS && n_experts % groups == 0,
              "kmb_route_topk: the number of groups must be in [1, %d] and divide the number of experts, got %d",
              RT_MAX_GROUPS, groups);
  KMB_REQUIRE(topk_groups >= 1 && topk_groups <= groups,
              "kmb_route_topk: topk_groups must be in [1, groups], got %d", topk_groups);
  KMB_REQUIRE((int64_t)topk_groups * (n_experts / groups) >= k,
              "Expected k to be greater than or equal to the number of items in the search space, but got "
              "k=%d and %d items in the search space.", k, topk_groups * (n_experts / groups));
  KMB_REQUIRE((group_best == 1 || group_best == 2) && group_best <= n_experts / groups,
              "kmb_route_topk: group_best must be 1 or 2 and at most the size of a group, got %d", group_best);
  if (n == 0) return KMB_OK;
  KMB_REQUIRE(logits && weights && experts, "kmb_route_topk: NULL argument");
  RouteParams p;
  p.logits = logits;
  p.bias = bias;
  p.weights = weights;
  p.experts = experts;
  p.n = n;
  p.n_experts = n_experts;
  p.k = k;
  p.groups = topk_groups == groups ? 1 : groups;     // every group stays: no groups
  p.topk_groups = topk_groups;
  p.group_best = group_best;
  p.group_size = n_experts / groups;
  p.sigmoid = (flags & KMB_ROUTE_SIGMOID) != 0;
  p.renormalize = (flags & KMB_ROUTE_RENORMALIZE) != 0;
  p.scale = scale;
  KMB_DISPATCH_ROWS(dtype, { return route_run<T>(p, (cudaStream_t)stream); });
}

int kmb_route_topk_grad(int dtype, const void* logits, const int32_t* experts, const float* grad_weights,
                        int64_t n, int n_experts, int k, int flags, float scale, void* grad_logits,
                        void* stream) {
  int rc = check_route("kmb_route_topk_grad", n_experts, k);
  if (rc != KMB_OK) return rc;
  KMB_REQUIRE(n >= 0, "kmb_route_topk_grad: bad sizes");
  KMB_REQUIRE((flags & ~(KMB_ROUTE_SIGMOID | KMB_ROUTE_RENORMALIZE)) == 0,
              "kmb_route_topk_grad: unknown flag bits");
  if (n == 0) return KMB_OK;
  KMB_REQUIRE(logits && experts && grad_weights && grad_logits, "kmb_route_topk_grad: NULL argument");
  RouteGradParams p;
  p.logits = logits;
  p.experts = experts;
  p.grad_weights = grad_weights;
  p.grad_logits = grad_logits;
  p.n = n;
  p.n_experts = n_experts;
  p.k = k;
  p.sigmoid = (flags & KMB_ROUTE_SIGMOID) != 0;
  p.renormalize = (flags & KMB_ROUTE_RENORMALIZE) != 0;
  p.scale = scale;
  KMB_DISPATCH_ROWS(dtype, { return route_grad_run<T>(p, (cudaStream_t)stream); });
}

size_t kmb_expert_slots_workspace_bytes(int64_t n, int k, int n_experts) {
  if (n < 0 || k < 1 || n_experts < 1) return 0;
  const int64_t chunks = ceil_div(n * k, SL_CHUNK);
  return chunks <= 1 ? 0 : (size_t)(chunks + 1) * n_experts * sizeof(int32_t);
}

int kmb_expert_slots(const int32_t* experts, int64_t n, int k, int n_experts, int32_t* slots, int32_t* rows,
                     int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  KMB_REQUIRE(n >= 0 && k >= 1, "kmb_expert_slots: bad sizes");
  KMB_REQUIRE(n_experts >= 1 && n_experts <= SL_MAX_EXPERTS,
              "kmb_expert_slots: the number of experts must be in [1, %d], got %d", SL_MAX_EXPERTS, n_experts);
  KMB_REQUIRE(n <= MAX_CHOICES / k, "kmb_expert_slots: n * k must be below 2^31 - 4096");
  KMB_REQUIRE(offsets && (n == 0 || (experts && slots && rows)), "kmb_expert_slots: NULL argument");
  const size_t need = kmb_expert_slots_workspace_bytes(n, k, n_experts);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("kmb_expert_slots: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return KMB_ERR_WORKSPACE;
  }
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t total = n * k;
  const int chunks = (int)ceil_div(total, SL_CHUNK);
  const size_t smem = slots_place_smem(n_experts);
  // The counters of 16 warps and the ordered chunk may pass the 48 KB that need no asking.  The limit belongs to
  // the kernel, not to the call: every call that needs one sets the same, so that none lowers it under another's
  // launch.
  const auto place = chunks <= 1 ? slots_place_kernel<true> : slots_place_kernel<false>;
  if (smem > 8 * 1024)
    KMB_CHECK_CUDA(cudaFuncSetAttribute(place, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)slots_place_smem(SL_MAX_EXPERTS)));
  if (chunks <= 1)
    return launch_early(place, 1, SL_THREADS, smem, 1, s, experts, total, k, n_experts, nullptr, nullptr, slots, rows,
                        offsets);
  int32_t* counts = (int32_t*)workspace;
  int32_t* totals = counts + (int64_t)chunks * n_experts;
  int rc = launch_early(slots_count_kernel, chunks, SL_THREADS, 0, 1, s, experts, total, n_experts, counts);
  if (rc == KMB_OK)
    rc = launch_early(slots_scan_kernel, (unsigned)ceil_div(n_experts, 32), 1024, 0, 1, s, counts, chunks, n_experts,
                      totals);
  if (rc == KMB_OK)
    rc = launch_early(place, chunks, SL_THREADS, smem, 1, s, experts, total, k, n_experts, counts, totals, slots, rows,
                      offsets);
  return rc;
}

int kmb_combine_experts(int dtype, const void* values, int64_t n_values, const int32_t* slots,
                        const float* weights, int64_t n, int k, int d, void* out, void* stream) {
  KMB_REQUIRE(n >= 0 && n < (1ll << 31) - 1 && n_values >= 0 && k >= 1 && d >= 1, "kmb_combine_experts: bad sizes");
  KMB_REQUIRE(d < CB_MAX_D, "kmb_combine_experts: d must be below 2^30");
  if (n == 0) return KMB_OK;
  KMB_REQUIRE((values || n_values == 0) && slots && weights && out, "kmb_combine_experts: NULL argument");
  KMB_DISPATCH_ROWS(dtype, {
    const int vec = rows_are_vec((const T*)values, d) && rows_are_vec((const T*)out, d);
    const unsigned threads = combine_threads(d, CB_THREADS);
    // long rows of few tokens are shared between blocks
    const int64_t passes = ceil_div(d, threads * 8);
    const int parts = n * passes <= (int64_t)sm_count() * 4 ? (int)passes : 1;
    return launch_early(vec ? combine_kernel<T, true> : combine_kernel<T, false>, (unsigned)(n * parts), (int)threads, 0,
                        1, (cudaStream_t)stream, (const T*)values, n_values, slots, weights, k, d, (T*)out, parts);
  });
}

size_t kmb_combine_experts_grad_workspace_bytes(int64_t n_values) {
  return n_values < 0 ? 0 : (size_t)n_values * 2 * sizeof(int32_t);
}

size_t kmb_combine_experts_grad_workspace_bytes_for(int64_t n_values, int64_t n, int k) {
  if (n < 0 || k < 1 || n > MAX_CHOICES / k) return 0;
  return n_values <= 0 ? 0 : kmb_combine_experts_grad_workspace_bytes(n_values) + (size_t)(n * k) * sizeof(int32_t);
}

int kmb_combine_experts_grad(int dtype, const void* values, int64_t n_values, const int32_t* slots,
                             const float* weights, const void* grad_out, int64_t n, int k, int d,
                             void* grad_values, float* grad_weights, void* workspace, size_t workspace_bytes,
                             void* stream) {
  KMB_REQUIRE(n >= 0 && n_values >= 0 && k >= 1 && d >= 1, "kmb_combine_experts_grad: bad sizes");
  KMB_REQUIRE(d < CB_MAX_D, "kmb_combine_experts_grad: d must be below 2^30");
  KMB_REQUIRE(n <= MAX_CHOICES / k, "kmb_combine_experts_grad: n * k must be below 2^31 - 4096");
  if (n == 0 && n_values == 0) return KMB_OK;
  KMB_REQUIRE((n_values == 0 || (values && grad_values)) && (n == 0 || (slots && weights && grad_out && grad_weights)),
              "kmb_combine_experts_grad: NULL argument");
  const size_t need = kmb_combine_experts_grad_workspace_bytes(n_values);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("kmb_combine_experts_grad: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return KMB_ERR_WORKSPACE;
  }
  cudaStream_t s = (cudaStream_t)stream;
  int32_t* users = (int32_t*)workspace;
  int32_t* head = users + n_values;
  int32_t* next = n > 0 && workspace_bytes >= kmb_combine_experts_grad_workspace_bytes_for(n_values, n, k)
                      ? head + n_values : nullptr;
  if (n_values > 0 && n_values <= CG_FEW && n * k <= CG_FEW) {
    const size_t smem = (size_t)n_values * 2 * sizeof(int32_t);
    if (smem > 48 * 1024)      // every call that needs a limit sets the same one
      KMB_CHECK_CUDA(cudaFuncSetAttribute(combine_few_users_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          CG_FEW * 2 * (int)sizeof(int32_t)));
    const int rc = launch_early(combine_few_users_kernel, 1, CG_FEW_THREADS, smem, 1, s, slots, n * k, n_values, users,
                                head, next);
    if (rc != KMB_OK) return rc;
  } else {
    if (n_values > 0) {
      const int rc = launch_early(combine_clear_kernel, (unsigned)ceil_div(n_values, 256), 256, 0, 1, s, n_values, users,
                                  head, next);
      if (rc != KMB_OK) return rc;
    }
    if (n > 0) {
      const int rc = launch_early(combine_users_kernel, (unsigned)ceil_div(n * k, 256), 256, 0, 1, s, slots, n * k,
                                  n_values, users, head, next);
      if (rc != KMB_OK) return rc;
    }
  }
  // a user found by its chain costs as much as 512 choices walked over
  const int64_t chained = n * k / 512 > 32 ? n * k / 512 : 32;
  const int most_chained = (int)(chained < CG_LIST ? chained : CG_LIST);
  KMB_DISPATCH_ROWS(dtype, {
    const int vec = rows_are_vec((const T*)values, d) && rows_are_vec((const T*)grad_out, d) &&
                    rows_are_vec((const T*)grad_values, d);
    const unsigned threads = combine_threads(d, CG_THREADS);
    // Blocks for the rows without a user or with several: up to four to an SM, each with as few rows at a time as that
    // gives, but sixteen where rows have few users (1000 rows, one user each: 500 such blocks cost 0.5 us more than 63).
    const int64_t most = (int64_t)sm_count() * 4;
    int64_t rows = ceil_div(n_values, most);
    if (rows < 16 && n * k <= n_values * 4) rows = 16;
    if (rows > (int64_t)threads) rows = threads;
    const int64_t fill = n_values == 0 ? 0 : (ceil_div(n_values, rows) < most ? ceil_div(n_values, rows) : most);
    const int64_t token_blocks = n * ceil_div(k, CG_K);
    return launch_early(vec ? combine_grad_kernel<T, true> : combine_grad_kernel<T, false>,
                        (unsigned)(token_blocks + fill), (int)threads, 0, 1, s, (const T*)values, n_values, slots,
                        weights, (const T*)grad_out, n, k, d, users, head, next, most_chained, (int)rows,
                        (T*)grad_values, grad_weights, token_blocks);
  });
}

}  // extern "C"
