// A mixture's router: from logits to experts and weights, the balance loss, and the gradients of both.
//
// A row of logits is shared out to kLanes lanes, kVals neighbouring experts each, in registers, so that a wave has
// 64 / kLanes rows and every row is read once. What a row needs as a whole (its largest logit, sums) is reduced
// among its lanes by DPP moves. All sums are FP32 in a fixed order, those over tokens FP64 at their end.
//
// Route: `top` times the row's largest key is found and taken out. Keys are the logits themselves, compared exactly,
// or with a bias score + bias in FP64: in FP32 two experts near the border could change places by rounding.
// Balance: p = softmax or normalized sigmoids, of which a lane adds up its experts' over its rows; a second launch
// of one workgroup adds up the workgroups' sums.
#include <type_traits>

#include "mxfp4_common.h"

namespace mps {
namespace {

constexpr float kNone = -__builtin_inff();  // a masked expert's logit; a key that is never taken

struct RouteArgs {
  const void *logits;
  int64_t stride, tokens;  // elements from row to row
  const float *bias;
  int32_t *ids;
  float *weights, *shares;  // shares: weights before the factor `scale`, if asked for
  const float *dweights;
  void *dlogits;
  float scale;
  int32_t experts, top, normalize;
};

// `op` over the L lanes of a row; all of them get the result. Every step joins two halves that already agree.
template <int kControl>
__device__ inline float moved(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), kControl, 0xf, 0xf, true));
}
template <int kControl>
__device__ inline double moved(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, kControl, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), kControl, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int kRows>  // 16: the other row of 16 lanes of a pair, 32: the other half of the wave
__device__ inline void halves(float v, float &a, float &b) {
  const uint32_t u = __float_as_uint(v);
  const auto r = kRows == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
  a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
}
template <int kRows>
__device__ inline void halves(double v, double &a, double &b) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
  const auto lo = kRows == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false) : __builtin_amdgcn_permlane32_swap(l, l, false, false);
  const auto hi = kRows == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false) : __builtin_amdgcn_permlane32_swap(h, h, false, false);
  a = __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]), b = __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
template <int L, typename T, typename Op>
__device__ inline T over_row(T v, Op op) {
  static_assert(L == 4 || L == 8 || L == 16 || L == 32 || L == 64, "");
  v = op(v, moved<0xB1>(v));                        // lane ^ 1
  v = op(v, moved<0x4E>(v));                        // lane ^ 2
  if constexpr (L >= 8) v = op(v, moved<0x141>(v));  // 7 - lane within eight
  if constexpr (L >= 16) v = op(v, moved<0x140>(v));  // 15 - lane within sixteen
  if constexpr (L >= 32) {
    T a, b;
    halves<16>(v, a, b);
    v = op(a, b);
  }
  if constexpr (L >= 64) {
    T a, b;
    halves<32>(v, a, b);
    v = op(a, b);
  }
  return v;
}
struct Max {
  template <typename T>
  __device__ T operator()(T a, T b) const {
    return __builtin_elementwise_max(a, b);
  }
};
struct Sum {
  template <typename T>
  __device__ T operator()(T a, T b) const {
    return a + b;
  }
};

// kVals neighbouring logits of a row from `col` on, -inf past the last; 16-byte accesses take any alignment.
template <int T, int V>
__device__ inline void load_vals(const typename Elem<T>::raw *row, int32_t col, int32_t experts, float (&v)[V]) {
  typedef typename Elem<T>::raw raw;
  constexpr int kWords = V * (int)sizeof(raw) / 4;
  if (col + V <= experts) {
    typedef uint32_t words __attribute__((ext_vector_type(kWords < 4 ? kWords : 4), aligned(2)));
    constexpr int kEach = kWords < 4 ? kWords : 4;
#pragma unroll
    for (int w = 0; w < kWords; w += kEach) {
      const words b = *reinterpret_cast<const words *>(reinterpret_cast<const char *>(row + col) + w * 4);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if constexpr (T == MPS_TYPE_F32) {
          v[w + i] = __uint_as_float(b[i]);
        } else {
          v[2 * (w + i)] = Elem<T>::get((uint16_t)b[i]);
          v[2 * (w + i) + 1] = Elem<T>::get((uint16_t)(b[i] >> 16));
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = col + i < experts ? Elem<T>::get(row[col + i]) : kNone;
  }
}
template <int T, int V>
__device__ inline void store_vals(typename Elem<T>::raw *row, int32_t col, int32_t experts, const float (&v)[V]) {
  typedef typename Elem<T>::raw raw;
  constexpr int kWords = V * (int)sizeof(raw) / 4;
  if (col + V <= experts) {
    typedef uint32_t words __attribute__((ext_vector_type(kWords < 4 ? kWords : 4), aligned(2)));
    constexpr int kEach = kWords < 4 ? kWords : 4;
#pragma unroll
    for (int w = 0; w < kWords; w += kEach) {
      words b;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if constexpr (T == MPS_TYPE_F32)
          b[i] = __float_as_uint(v[w + i]);
        else
          b[i] = (uint32_t)Elem<T>::put(v[2 * (w + i)]) | (uint32_t)Elem<T>::put(v[2 * (w + i) + 1]) << 16;
      }
      *reinterpret_cast<words *>(reinterpret_cast<char *>(row + col) + w * 4) = b;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (col + i < experts) row[col + i] = Elem<T>::put(v[i]);
  }
}

constexpr int kRouteThreads = 256;

// LDS that lanes of one wave share: what they wrote is there for the others.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// kBias: keys are scores and a bias in FP64 (its scores by kSigmoid).
template <int T, int L, int V, bool kSigmoid, bool kBias>
__global__ __launch_bounds__(kRouteThreads) void expert_route_kernel(RouteArgs a) {
  typedef std::conditional_t<kBias, double, float> Key;
  typedef typename Elem<T>::raw raw;
  constexpr int kRows = 64 / L, kWaves = kRouteThreads / 64;
  __shared__ int32_t chosen[kWaves * kRows * L * V];
  const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  int32_t *const mine = chosen + (wave * kRows + row_in_wave) * L * V;
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    const int64_t t = token ? t0 + row_in_wave : a.tokens - 1;
    const raw *const row = static_cast<const raw *>(a.logits) + t * a.stride;
    float logit[V];
    load_vals<T, V>(row, in_row * V, a.experts, logit);
    float most = kNone;
#pragma unroll
    for (int j = 0; j < V; ++j) most = __builtin_elementwise_max(most, logit[j]);
    most = over_row<L>(most, Max());
    float nan = 0;  // softmax: a NaN or an infinity makes all of the row's scores NaN
    if constexpr (!kSigmoid) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < V; ++j) any |= !(logit[j] < __builtin_inff());
      const uint64_t rows = __ballot(any);
      const uint64_t own = L == 64 ? rows : rows >> (row_in_wave * L) & ((1ull << (L & 63)) - 1);
      if (own) nan = __builtin_nanf("");
    }
    Key key[V];
    if constexpr (kBias) {
      double sum = 1.0;
      if constexpr (!kSigmoid) {
        sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          key[j] = logit[j] > kNone ? exp((double)logit[j] - (double)most) : 0.0;
          sum += key[j];
        }
        sum = over_row<L>(sum, Sum());
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int32_t e = in_row * V + j;
        const double b = e < a.experts ? (double)a.bias[e] : 0.0;
        const double k = (kSigmoid ? 1.0 / (1.0 + exp(-(double)logit[j])) : key[j] / sum) + b;
        key[j] = logit[j] > kNone && k == k ? k : (double)kNone;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = logit[j] > kNone ? logit[j] : kNone;  // a NaN's, too
    }
    for (int32_t i = in_row; i < a.top; i += L) mine[i] = -1;
    wave_sync();
    for (int32_t i = 0; i < a.top; ++i) {
      Key best = key[0];
#pragma unroll
      for (int j = 1; j < V; ++j) best = __builtin_elementwise_max(best, key[j]);
      best = over_row<L>(best, Max());
      const bool some = best > (Key)kNone;
      int32_t at = V;  // the first of this lane's that has it
#pragma unroll
      for (int j = V - 1; j >= 0; --j) at = key[j] == best ? j : at;
      const uint64_t hits = __ballot(some && at < V);
      const uint64_t own = L == 64 ? hits : hits >> (row_in_wave * L) & ((1ull << (L & 63)) - 1);
      if (hits == 0) break;  // no row of this wave has any left
      const bool won = some && at < V && __ffsll((unsigned long long)own) - 1 == in_row;  // ties: the lowest expert
      if (won) mine[i] = in_row * V + at;
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = won && j == at ? (Key)kNone : key[j];
    }
    wave_sync();
    // Weights: those of a row's choice relative to its largest chosen logit, where they are divided by their sum.
    float top_logit = kNone;
    if (a.normalize) {
      for (int32_t i = in_row; i < a.top; i += L)
        if (mine[i] >= 0) top_logit = __builtin_elementwise_max(top_logit, Elem<T>::get(row[mine[i]]));
      top_logit = over_row<L>(top_logit, Max());
    }
    const float base = a.normalize ? top_logit : most;
    auto value = [&](int32_t e) -> float {
      if (e < 0) return 0.0f;
      const float l = Elem<T>::get(row[e]);
      if constexpr (kSigmoid) {  // sigmoids that are all small, as multiples of exp(base)
        return a.normalize && base < 0 ? expf(l - base) / (1.0f + expf(l)) : 1.0f / (1.0f + expf(-l));
      } else {
        return expf(l - base) + nan;
      }
    };
    float total = 0;
    if (a.normalize) {
      for (int32_t i = in_row; i < a.top; i += L) total += value(mine[i]);
      total = over_row<L>(total, Sum());
    } else if constexpr (kSigmoid) {
      total = 1.0f;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) total += logit[j] > kNone ? expf(logit[j] - base) : 0.0f;
      total = over_row<L>(total, Sum());
    }
    if (token)
      for (int32_t i = in_row; i < a.top; i += L) {
        const int32_t e = mine[i];
        const float share = e >= 0 ? value(e) / total : 0.0f;
        a.ids[t * a.top + i] = e;
        a.weights[t * a.top + i] = share * a.scale;
        if (a.shares) a.shares[t * a.top + i] = share;
      }
    wave_sync();
  }
}

// dlogit[e] = share (dw - c) (1 - sigmoid, for sigmoids) for the chosen experts, with c = sum over these of share dw if
// weights are divided by their sum, else 0; softmax without that division gives all experts -share c too.
template <int T, int L, int V, bool kSigmoid>
__global__ __launch_bounds__(kRouteThreads) void expert_route_grad_kernel(RouteArgs a) {
  typedef typename Elem<T>::raw raw;
  constexpr int kRows = 64 / L, kWaves = kRouteThreads / 64;
  __shared__ __attribute__((aligned(16))) float sums[kWaves * kRows * L * V];
  const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  float *const mine = sums + (wave * kRows + row_in_wave) * L * V;
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    const int64_t t = token ? t0 + row_in_wave : a.tokens - 1;
    const raw *const row = static_cast<const raw *>(a.logits) + t * a.stride;
#pragma unroll
    for (int j = 0; j < V; ++j) mine[in_row * V + j] = 0.0f;
    wave_sync();
    float c = 0;
    if (a.normalize || !kSigmoid)
      for (int32_t i = in_row; i < a.top; i += L)
        if (a.ids[t * a.top + i] >= 0) c = __builtin_fmaf(a.shares[t * a.top + i], a.dweights[t * a.top + i], c);
    c = over_row<L>(c, Sum());
    const float back = a.normalize ? c : 0.0f;
    for (int32_t i = in_row; i < a.top; i += L) {
      const int32_t e = a.ids[t * a.top + i];
      if (e < 0 || e >= a.experts) continue;
      float d = a.shares[t * a.top + i] * (a.dweights[t * a.top + i] - back);
      if constexpr (kSigmoid) d *= 1.0f / (1.0f + expf(Elem<T>::get(row[e])));
      mine[e] = d * a.scale;
    }
    wave_sync();
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = mine[in_row * V + j];
    if constexpr (!kSigmoid) {
      if (!a.normalize) {
        float logit[V], most = kNone, total = 0;
        load_vals<T, V>(row, in_row * V, a.experts, logit);
#pragma unroll
        for (int j = 0; j < V; ++j) most = __builtin_elementwise_max(most, logit[j]);
        most = over_row<L>(most, Max());
        float e[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          e[j] = logit[j] > kNone ? expf(logit[j] - most) : logit[j] == kNone ? 0.0f : logit[j];
          total += e[j];
        }
        total = over_row<L>(total, Sum());
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] -= logit[j] == kNone ? 0.0f : e[j] / total * c * a.scale;
      }
    }
    if (token) store_vals<T, V>(static_cast<raw *>(a.dlogits) + t * a.experts, in_row * V, a.experts, d);
    wave_sync();
  }
}

// ------------------------------------------------------------------ balance
// loss = experts * sum_e counts[e] / N * (1 / T) sum_t p[t, e], N pairs that have an expert, T tokens that have a
// logit above -inf; 0 if there are none.
struct BalanceArgs {
  const void *logits, *ids;
  int64_t stride, tokens, pairs;
  int32_t experts, ids_64;
  float *sums;        // [workgroups, experts]: of p
  int32_t *parts;     // [workgroups, experts + 1]: counts, and tokens
  float *loss;
  int32_t *counts;    // [experts], if asked for
  int32_t *kept;      // [experts + 1]: counts, and T, if asked for
  const float *dloss;
  void *dlogits;
};
constexpr int kBalanceThreads = 512;

// p of a row's kVals experts (of a row of -inf throughout: zeros, and `empty`), and for sigmoids 1 - sigmoid.
template <int L, int V, bool kSigmoid>
__device__ inline bool shares_of(const float (&logit)[V], float (&p)[V], float (&rest)[V]) {
  float most = kNone, total = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) most = __builtin_elementwise_max(most, logit[j]);
  most = over_row<L>(most, Max());
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if constexpr (kSigmoid) {  // sigmoids that are all small, as multiples of exp(most)
      const float e = expf(-logit[j]);  // infinite for small logits: the sigmoid is 0, and 1 - it 1
      rest[j] = 1.0f / (1.0f + expf(logit[j]));
      p[j] = most < 0 ? expf(logit[j] - most) * rest[j] : 1.0f / (1.0f + e);
    } else {
      p[j] = expf(logit[j] - most);
    }
    if (logit[j] == kNone) p[j] = 0.0f;
    total += p[j];
  }
  total = over_row<L>(total, Sum());
  const bool empty = total == 0.0f;  // no: some p is 1, or at least 1/2, or NaN
  const float by = empty ? 0.0f : 1.0f / total;
#pragma unroll
  for (int j = 0; j < V; ++j) p[j] *= by;
  return empty;
}

template <typename Id>
__device__ inline void count_ids(const BalanceArgs &a, int32_t *counts) {
  const Id *const ids = static_cast<const Id *>(a.ids);
  for (int64_t i = (int64_t)blockIdx.x * kBalanceThreads + threadIdx.x; i < a.pairs; i += (int64_t)gridDim.x * kBalanceThreads) {
    const Id e = ids[i];
    if (e >= 0 && e < a.experts) atomicAdd(&counts[e], 1);
  }
}

// The last step, by one workgroup, from `blocks` workgroups' sums: work-items share out first the blocks of an expert, then
// the experts.
struct FinishWork {
  double p[kBalanceThreads], all[kBalanceThreads];
  int32_t count[kBalanceThreads];
  double pairs[kBalanceThreads];
};
__device__ inline void finish_balance(const BalanceArgs &a, int32_t blocks, const float *sums, const int32_t *parts, FinishWork &work) {
  const int tid = threadIdx.x;
  int32_t width = 1;
  while (width < a.experts && width < kBalanceThreads) width *= 2;
  const int32_t shares = kBalanceThreads / width, keys = a.experts + 1;
  double pairs = 0.0, all = 0.0;
  for (int32_t e0 = 0; e0 < a.experts; e0 += width) {
    const int32_t e = e0 + tid % width;
    int32_t count = 0;
    double p = 0.0;
    if (e < a.experts) {
#pragma unroll 8
      for (int32_t b = tid / width; b < blocks; b += shares) {
        count += parts[(int64_t)b * keys + e];
        p += (double)sums[(int64_t)b * a.experts + e];
      }
    }
    work.p[tid] = p, work.count[tid] = count;
    __syncthreads();
    if (tid < width && e < a.experts) {
      for (int32_t i = 1; i < shares; ++i) p += work.p[i * width + tid], count += work.count[i * width + tid];
      if (a.counts) a.counts[e] = count;
      if (a.kept) a.kept[e] = count;
      pairs += count, all += (double)count * p;
    }
    __syncthreads();
  }
  int32_t tokens = 0;
  for (int32_t b = tid; b < blocks; b += kBalanceThreads) tokens += parts[(int64_t)b * keys + a.experts];
  work.pairs[tid] = pairs, work.all[tid] = all, work.count[tid] = tokens;
  __syncthreads();
  for (int d = kBalanceThreads / 2; d > 0; d /= 2) {
    if (tid < d) work.pairs[tid] += work.pairs[tid + d], work.all[tid] += work.all[tid + d], work.count[tid] += work.count[tid + d];
    __syncthreads();
  }
  if (tid == 0) {
    const double n = work.pairs[0], t = work.count[0];
    if (a.kept) a.kept[a.experts] = work.count[0];
    *a.loss = n > 0 && t > 0 ? (float)(a.experts * work.all[0] / (n * t)) : 0.0f;
  }
}

template <int T, int L, int V, bool kSigmoid>
__global__ __launch_bounds__(kBalanceThreads) void expert_balance_kernel(BalanceArgs a) {
  typedef typename Elem<T>::raw raw;
  constexpr int kRows = 64 / L, kWaves = kBalanceThreads / 64, kE = L * V;
  __shared__ float sums[kWaves][kE];
  __shared__ int32_t counts[kE + 1];
  __shared__ FinishWork work;
  const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  for (int32_t i = threadIdx.x; i <= kE; i += kBalanceThreads) counts[i] = 0;
  __syncthreads();
  if (a.ids_64)
    count_ids<int64_t>(a, counts);
  else
    count_ids<int32_t>(a, counts);
  float sum[V] = {};
  int32_t rows = 0;
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    const int64_t t = token ? t0 + row_in_wave : a.tokens - 1;
    float logit[V], p[V], rest[V];
    load_vals<T, V>(static_cast<const raw *>(a.logits) + t * a.stride, in_row * V, a.experts, logit);
    const bool empty = shares_of<L, V, kSigmoid>(logit, p, rest);
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] += token ? p[j] : 0.0f;
    rows += token && !empty && in_row == 0;
  }
  if (rows) atomicAdd(&counts[a.experts], rows);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    for (int d = L; d < 64; d *= 2) sum[j] += __shfl_xor(sum[j], d);
    if (row_in_wave == 0) sums[wave][in_row * V + j] = sum[j];
  }
  __syncthreads();
  for (int32_t e = threadIdx.x; e < a.experts; e += kBalanceThreads) {
    float s = 0;
    for (int w = 0; w < kWaves; ++w) s += sums[w][e];
    if (gridDim.x == 1)
      sums[0][e] = s;
    else
      a.sums[(int64_t)blockIdx.x * a.experts + e] = s;
  }
  if (gridDim.x == 1) {
    __syncthreads();
    finish_balance(a, 1, sums[0], counts, work);
  } else {
    for (int32_t e = threadIdx.x; e <= a.experts; e += kBalanceThreads) a.parts[(int64_t)blockIdx.x * (a.experts + 1) + e] = counts[e];
  }
}

__global__ __launch_bounds__(kBalanceThreads) void expert_balance_sum_kernel(BalanceArgs a, int32_t blocks) {
  __shared__ FinishWork work;
  finish_balance(a, blocks, a.sums, a.parts, work);
}

// dlogit[t, e] = dloss experts / (N T) p (counts[e] - sum_j counts[j] p[t, j]) (1 - sigmoid, for sigmoids).
template <int T, int L, int V, bool kSigmoid>
__global__ __launch_bounds__(kRouteThreads) void expert_balance_grad_kernel(BalanceArgs a) {
  typedef typename Elem<T>::raw raw;
  constexpr int kRows = 64 / L, kWaves = kRouteThreads / 64;
  const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  float count[V];
  double n = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int32_t e = in_row * V + j, c = e < a.experts ? a.kept[e] : 0;
    count[j] = (float)c, n += c;
  }
  n = over_row<L>(n, Sum());
  const double tokens = a.kept[a.experts];
  const float factor = n > 0 && tokens > 0 ? (float)((double)*a.dloss * a.experts / (n * tokens)) : 0.0f;
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    const int64_t t = token ? t0 + row_in_wave : a.tokens - 1;
    float logit[V], p[V], rest[V], c = 0;
    load_vals<T, V>(static_cast<const raw *>(a.logits) + t * a.stride, in_row * V, a.experts, logit);
    shares_of<L, V, kSigmoid>(logit, p, rest);
#pragma unroll
    for (int j = 0; j < V; ++j) c = __builtin_fmaf(count[j], p[j], c);
    c = over_row<L>(c, Sum());
#pragma unroll
    for (int j = 0; j < V; ++j) {
      p[j] = logit[j] == kNone ? 0.0f : p[j] * (count[j] - c) * factor;
      if constexpr (kSigmoid) p[j] *= rest[j];
    }
    if (token) store_vals<T, V>(static_cast<raw *>(a.dlogits) + t * a.experts, in_row * V, a.experts, p);
  }
}

// Workgroups of the first launch: one up to 64 rows of waves' rows, else as many as leave the second launch little to add up.
int32_t balance_blocks(int64_t tokens, int64_t experts, int64_t pairs) {
  const int64_t work = tokens * experts + pairs;
  if (work <= 16384) return 1;
  const int64_t most = 32768 / experts < 256 ? 32768 / experts : 256, wanted = (work + 16383) / 16384;
  return (int32_t)(wanted < most ? wanted : most);
}
inline int64_t balance_bytes(int32_t blocks, int64_t experts) { return blocks > 1 ? blocks * (2 * experts + 1) * 4 : 0; }

int check_route(const char *what, int32_t type, int64_t tokens, int64_t experts, int64_t top, int64_t stride, int32_t scores) {
  if (!is_float_type(type)) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: unknown type of logits", what);
  if (scores != MPS_SCORES_SOFTMAX && scores != MPS_SCORES_SIGMOID) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: unknown scores", what);
  if (experts < 1 || experts > MPS_MAX_EXPERTS)
    return fail(MPS_ERR_INVALID_ARGUMENT, "%s: experts must be in [1, %d]", what, MPS_MAX_EXPERTS);
  if (tokens < 0 || top < 0 || stride < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (top > 0 && tokens > (INT32_MAX - 1024) / top)
    return fail(MPS_ERR_INVALID_ARGUMENT, "%s: over 2^31 - 1025 pairs of tokens and experts", what);
  if (tokens > INT32_MAX - 1024) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: over 2^31 - 1025 tokens", what);
  return MPS_OK;
}

// How a row is shared out: lanes, and experts a lane.
#define MPS_BY_EXPERTS(experts, T, CALL)          \
  do {                                            \
    if ((experts) <= 16) { CALL(T, 4, 4); }       \
    else if ((experts) <= 32) { CALL(T, 8, 4); }  \
    else if ((experts) <= 64) { CALL(T, 16, 4); } \
    else if ((experts) <= 128) { CALL(T, 16, 8); }\
    else if ((experts) <= 256) { CALL(T, 32, 8); }\
    else if ((experts) <= 512) { CALL(T, 64, 8); }\
    else { CALL(T, 64, 16); }                     \
  } while (0)
#define MPS_BY_LOGITS(type, experts, CALL)                                        \
  do {                                                                            \
    if ((type) == MPS_TYPE_F32) { MPS_BY_EXPERTS(experts, MPS_TYPE_F32, CALL); }  \
    else if ((type) == MPS_TYPE_BF16) { MPS_BY_EXPERTS(experts, MPS_TYPE_BF16, CALL); } \
    else { MPS_BY_EXPERTS(experts, MPS_TYPE_F16, CALL); }                         \
  } while (0)

template <int L>
unsigned route_grid(int64_t tokens) {
  constexpr int64_t per = kRouteThreads / L;
  return workgroups((tokens + per - 1) / per);
}

}  // namespace
}  // namespace mps

using namespace mps;

extern "C" {

int mps_expert_route(const void *logits, int32_t type, int64_t tokens, int64_t experts, int64_t stride, int64_t top,
                     int32_t scores, const float *bias, int32_t normalize, float scale, int32_t *ids, float *weights,
                     float *shares, void *stream) {
  last_error().clear();
  const int rc = check_route("expert_route", type, tokens, experts, top, stride, scores);
  if (rc != MPS_OK) return rc;
  if (top > experts) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_route: top is over the experts");
  if (tokens == 0 || top == 0) return MPS_OK;
  if (!logits || !ids || !weights) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_route: null pointer");
  RouteArgs a = {};
  a.logits = logits, a.stride = stride, a.tokens = tokens, a.bias = bias, a.ids = ids, a.weights = weights, a.shares = shares;
  a.scale = scale, a.experts = (int32_t)experts, a.top = (int32_t)top, a.normalize = normalize;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define LAUNCH(T, L, V, S, B) \
  hipLaunchKernelGGL((expert_route_kernel<T, L, V, S, B>), dim3(route_grid<L>(tokens)), dim3(kRouteThreads), 0, s, a)
#define CALL(T, L, V)                                                                            \
  if (scores == MPS_SCORES_SIGMOID) {                                                            \
    if (bias) { LAUNCH(T, L, V, true, true); } else { LAUNCH(T, L, V, true, false); }            \
  } else {                                                                                       \
    if (bias) { LAUNCH(T, L, V, false, true); } else { LAUNCH(T, L, V, false, false); }          \
  }
  MPS_BY_LOGITS(type, experts, CALL);
#undef CALL
#undef LAUNCH
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_route_grad(const void *logits, int32_t type, int64_t tokens, int64_t experts, int64_t stride, int64_t top,
                          int32_t scores, int32_t normalize, float scale, const int32_t *ids, const float *shares,
                          const float *dweights, void *dlogits, void *stream) {
  last_error().clear();
  const int rc = check_route("expert_route_grad", type, tokens, experts, top, stride, scores);
  if (rc != MPS_OK) return rc;
  if (top > experts) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_route_grad: top is over the experts");
  if (tokens == 0) return MPS_OK;
  if (!logits || !dlogits || (top > 0 && (!ids || !shares || !dweights)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_route_grad: null pointer");
  RouteArgs a = {};
  a.logits = logits, a.stride = stride, a.tokens = tokens, a.ids = const_cast<int32_t *>(ids), a.shares = const_cast<float *>(shares);
  a.dweights = dweights, a.dlogits = dlogits, a.scale = scale;
  a.experts = (int32_t)experts, a.top = (int32_t)top, a.normalize = normalize;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define LAUNCH(T, L, V, S) \
  hipLaunchKernelGGL((expert_route_grad_kernel<T, L, V, S>), dim3(route_grid<L>(tokens)), dim3(kRouteThreads), 0, s, a)
#define CALL(T, L, V) \
  if (scores == MPS_SCORES_SIGMOID) { LAUNCH(T, L, V, true); } else { LAUNCH(T, L, V, false); }
  MPS_BY_LOGITS(type, experts, CALL);
#undef CALL
#undef LAUNCH
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_balance_workspace(int64_t tokens, int64_t experts, int64_t top, int64_t *bytes) {
  last_error().clear();
  const int rc = check_route("expert_balance", MPS_TYPE_F32, tokens, experts, top, 0, MPS_SCORES_SOFTMAX);
  if (rc != MPS_OK) return rc;
  if (!bytes) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_balance: null pointer");
  *bytes = balance_bytes(balance_blocks(tokens, experts, tokens * top), experts);
  return MPS_OK;
}

int mps_expert_balance(const void *logits, int32_t type, int64_t tokens, int64_t experts, int64_t stride, int32_t scores,
                       const void *ids, int32_t ids_64, int64_t top, float *loss, int32_t *counts, int32_t *kept, void *workspace,
                       int64_t workspace_bytes, void *stream) {
  last_error().clear();
  const int rc = check_route("expert_balance", type, tokens, experts, top, stride, scores);
  if (rc != MPS_OK) return rc;
  if (!loss || (tokens > 0 && (!logits || (top > 0 && !ids))))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_balance: null pointer");
  const int32_t blocks = balance_blocks(tokens, experts, tokens * top);
  const int64_t need = balance_bytes(blocks, experts);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_balance: %lld bytes of workspace are needed", (long long)need);
  BalanceArgs a = {};
  a.logits = logits, a.ids = ids, a.stride = stride, a.tokens = tokens, a.pairs = tokens * top;
  a.experts = (int32_t)experts, a.ids_64 = ids_64, a.loss = loss, a.counts = counts, a.kept = kept;
  a.sums = static_cast<float *>(workspace), a.parts = reinterpret_cast<int32_t *>(a.sums + (need > 0 ? blocks * experts : 0));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define LAUNCH(T, L, V, S) hipLaunchKernelGGL((expert_balance_kernel<T, L, V, S>), dim3(blocks), dim3(kBalanceThreads), 0, s, a)
#define CALL(T, L, V) \
  if (scores == MPS_SCORES_SIGMOID) { LAUNCH(T, L, V, true); } else { LAUNCH(T, L, V, false); }
  MPS_BY_LOGITS(type, experts, CALL);
#undef CALL
#undef LAUNCH
  if (blocks > 1) hipLaunchKernelGGL(expert_balance_sum_kernel, dim3(1), dim3(kBalanceThreads), 0, s, a, blocks);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_balance_grad(const void *logits, int32_t type, int64_t tokens, int64_t experts, int64_t stride, int32_t scores,
                            const int32_t *kept, const float *dloss, void *dlogits, void *stream) {
  last_error().clear();
  const int rc = check_route("expert_balance_grad", type, tokens, experts, 0, stride, scores);
  if (rc != MPS_OK) return rc;
  if (tokens == 0) return MPS_OK;
  if (!logits || !kept || !dloss || !dlogits) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_balance_grad: null pointer");
  BalanceArgs a = {};
  a.logits = logits, a.stride = stride, a.tokens = tokens, a.experts = (int32_t)experts;
  a.kept = const_cast<int32_t *>(kept), a.dloss = dloss, a.dlogits = dlogits;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define LAUNCH(T, L, V, S) \
  hipLaunchKernelGGL((expert_balance_grad_kernel<T, L, V, S>), dim3(route_grid<L>(tokens)), dim3(kRouteThreads), 0, s, a)
#define CALL(T, L, V) \
  if (scores == MPS_SCORES_SIGMOID) { LAUNCH(T, L, V, true); } else { LAUNCH(T, L, V, false); }
  MPS_BY_LOGITS(type, experts, CALL);
#undef CALL
#undef LAUNCH
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
