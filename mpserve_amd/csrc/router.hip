// A mixture's router: from logits to experts and weights, the balance loss, and the gradients of both.
//
// A row of logits is shared out to kLanes lanes, kVals neighbouring experts each, in registers, so that a wave has
// 64 / kLanes rows and every row is read once. What a row needs as a whole (its largest logit, sums) is reduced
// among its lanes by DPP moves. All sums are FP32 in a fixed order, those over tokens FP64 at their end.
//
// Route: `top` times the row's largest key is found and taken out. Keys are the logits themselves, compared exactly,
// or with a bias score + bias, which are compared in FP64 where FP32 cannot tell two of them apart.
// Balance: p = softmax or normalized sigmoids, of which a lane adds up its experts' over its rows; a second launch
// of one workgroup adds up the workgroups' sums.
#include <algorithm>
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
template <int kControl, typename T>
__device__ inline T moved(T v) {
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int32_t, v), kControl, 0xf, 0xf, true));
}
template <int kControl>
__device__ inline double moved(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, kControl, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), kControl, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int kRows, typename T>  // 16: the other row of 16 lanes of a pair, 32: the other half of the wave
__device__ inline void halves(T v, T &a, T &b) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = kRows == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
  a = __builtin_bit_cast(T, (uint32_t)r[0]), b = __builtin_bit_cast(T, (uint32_t)r[1]);
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

// exp(x) = 2^t (1 + rest ln 2), where t = x log2(e) rounded, and rest what that lost and what log2(e) has behind FP32: two steps
// of FP32 off at most, where expf takes twice the instructions. Below x = -150, of masks too, 0; a NaN stays one.
__device__ inline float exp_of(float x) {
  constexpr float kLog2e = 1.44269502e+0f, kLog2eRest = 1.92596303e-8f, kLn2 = 0.693147181f;
  x = x < -150.0f ? -150.0f : x;
  const float t = x * kLog2e, rest = __builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, -t)), e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, rest * kLn2, e);
}
__device__ inline float one_over(float d) {  // for finite d
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}
// 1 / (1 + exp(-x)): below x = -88 less than 2^-126.
__device__ inline float sigmoid_of(float x) { return one_over(1.0f + exp_of(x < -88.0f ? 88.0f : -x)); }

// The largest of a row's logits that is no NaN; 0 in a row of none but -inf, of which all differences are -inf then.
template <int L, int V>
__device__ inline float largest(const float (&logit)[V]) {
  float most = logit[0] > kNone ? logit[0] : kNone;
#pragma unroll
  for (int j = 1; j < V; ++j) most = logit[j] > most ? logit[j] : most;
  int32_t k = __builtin_bit_cast(int32_t, most + 0.0f);
  k = over_row<L>(k ^ (k >> 31 & 0x7fffffff), Max());
  most = __builtin_bit_cast(float, k ^ (k >> 31 & 0x7fffffff));
  return most > kNone ? most : 0.0f;
}

constexpr int kRouteThreads = 256;

// LDS that lanes of one wave share: what they wrote is there for the others.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Keys in the order of FP32 numbers, as whole numbers: their maxima need no care for NaN and go with DPP moves in one instruction.
constexpr int32_t kNoKey = INT32_MIN;
__device__ inline int32_t key_of(float f) {  // the two zeros are alike; -inf and NaN have no key
  const int32_t b = __builtin_bit_cast(int32_t, f + 0.0f);
  return f > kNone ? b ^ (b >> 31 & 0x7fffffff) : kNoKey;
}
__device__ inline float of_key(int32_t k) { return __builtin_bit_cast(float, k ^ (k >> 31 & 0x7fffffff)); }

// One after the other the row's largest keys, ties to the lowest expert, into `mine`: the first `top`. With keys that are not
// exact, as many more as do not follow the last of these by enough (`apart`), so that the true ones are among them; how many, alike
// for all rows of the wave, and whether any are too near. Mostly each row has one key that is the largest: the masks of who has it tell, and
// the tie's longer way is left out (65536 x 128 FP32, one row in twenty of -inf alone, eight of them: 20.6 us where those rows
// take it too, 17.8 us so).
struct Chosen {
  int32_t count;
  bool sure;
};
template <bool kNear, int L, int V, typename Apart>
__device__ inline Chosen choose(int32_t (&key)[V], int32_t top, int32_t *mine, Apart apart) {
  const int in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  int32_t last = INT32_MAX, i = 0;
  bool sure = true;
  for (;; ++i) {
    int32_t best = key[0];
#pragma unroll
    for (int j = 1; j < V; ++j) best = __builtin_elementwise_max(best, key[j]);
    best = __builtin_elementwise_max(over_row<L>(best, Max()), kNoKey + 1);  // no key is that: a row without any finds none
    const bool some = best != kNoKey + 1;
    if constexpr (kNear) {
      const bool far = apart(last, best);
      if (__all(!some || (i >= top && far))) break;
      sure &= !some || far;
      last = i < top ? best : last;
    } else if (i == top) {
      break;
    }
    uint64_t who[V];
    int32_t at = V, hits = 0;
#pragma unroll
    for (int j = V - 1; j >= 0; --j) {
      const bool has = key[j] == best;
      who[j] = __ballot(has);
      hits += __popcll(who[j]);
      at = has ? j : at;  // the first of this lane's
      key[j] = has ? kNoKey : key[j];
    }
    bool won = at < V;
    if (hits * L != __popcll(__ballot(some))) {
      const uint64_t lanes = __ballot(won), own = L == 64 ? lanes : lanes >> (row_in_wave * L) & ((1ull << (L & 63)) - 1);
      won = __ffsll((unsigned long long)own) - 1 == in_row;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((who[j] >> in_wave & 1) && !(won && j == at)) key[j] = best;
    }
    if (won) mine[i] = in_row * V + at;
  }
  return {i, (bool)__all(sure)};
}

// kBias: keys are scores and a bias. In FP32 they are off by less than 37 u of the row's largest score, u = 2^-24, and u of themselves, by the
// sum with the bias. For the largest shape, 16 experts a lane and 64 lanes: a softmax's sum 15 + 6 additions, its exponentials 4 u and their
// arguments' rounding |x| u, at most 4.5 u of the sum for up to 1024 terms exp(x); a score's own exponential 4 u; the reciprocal 2 u and
// the product u. (Sigmoids: 7 u of 1.) Two keys are off by less than 74 u: where two that follow each other are not 2^-17, 128 u, and 2^-22 of
// themselves apart, those chosen and all that are near the last of them are put in order by keys in FP64. In a row whose
// experts are all alike (a router that starts from zeros) the order is that of FP32, ties. (All keys in FP64: 8192 x 256 15.3 us, 12.9 us so.)
template <int T, int L, int V, bool kSigmoid, bool kBias>
__global__ __launch_bounds__(kRouteThreads) void expert_route_kernel(RouteArgs a) {
  typedef typename Elem<T>::raw raw;
  constexpr int kRows = 64 / L, kWaves = kRouteThreads / 64;
  __shared__ int32_t chosen[kWaves * kRows * L * V], sorted[kBias ? kWaves * kRows * L * V : 1];
  const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  int32_t *const mine = chosen + (wave * kRows + row_in_wave) * L * V;
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    const int64_t t = token ? t0 + row_in_wave : a.tokens - 1;
    const raw *const row = static_cast<const raw *>(a.logits) + t * a.stride;
    float logit[V];
    load_vals<T, V>(row, in_row * V, a.experts, logit);
    for (int32_t i = in_row; i < (kBias ? L * V : a.top); i += L) mine[i] = -1;
    wave_sync();
    // Softmax without a division by the chosen ones' sum, or as part of keys: its largest logit and its sum. A NaN or an
    // infinity makes all of the row's scores NaN; as parts of keys these count as 0, so that experts are taken, with NaN for weights.
    float most = 0, total = 1.0f, nan = 0, score[V];
    if constexpr (!kSigmoid) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < V; ++j) any |= !(logit[j] < __builtin_inff());
      const uint64_t rows = __ballot(any);
      const uint64_t own = L == 64 ? rows : rows >> (row_in_wave * L) & ((1ull << (L & 63)) - 1);
      if (own) nan = __builtin_nanf("");
      if (kBias || !a.normalize) {
        most = largest<L>(logit);
        total = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) score[j] = exp_of(logit[j] - most), total += score[j];
        total = over_row<L>(total, Sum());
      }
    }
    int32_t key[V];
    if constexpr (kBias) {
      float bias[V];
      bool alike = true;
      const float first_logit = Elem<T>::get(row[0]), first_bias = a.bias[0];
      const float by = kSigmoid ? 1.0f : one_over(total);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        bias[j] = a.bias[min(in_row * V + j, a.experts - 1)];
        alike &= in_row * V + j >= a.experts || (logit[j] == first_logit && bias[j] == first_bias);
        const float k = (kSigmoid ? sigmoid_of(logit[j]) : nan == 0.0f ? score[j] * by : 0.0f) + bias[j];
        key[j] = logit[j] > kNone ? key_of(k) : kNoKey;
      }
      const uint64_t others = __ballot(!alike);
      const bool ties = (L == 64 ? others : others >> (row_in_wave * L) & ((1ull << (L & 63)) - 1)) == 0;
      const float score_error = 0x1p-17f * (nan == 0.0f ? by : 0.0f);
      const Chosen c = choose<true, L, V>(key, a.top, mine, [&](int32_t last, int32_t best) {
        const float f = of_key(best);
        return ties || last == INT32_MAX || of_key(last) - f > __builtin_fmaf(0x1p-22f, __builtin_fabsf(f), score_error);
      });
      if (__builtin_expect(!c.sure, 0)) {
        wave_sync();
        double sum = 1.0;
        if constexpr (!kSigmoid) {
          sum = 0.0;
#pragma unroll 1
          for (int j = 0; j < V; ++j) sum += exp((double)Elem<T>::get(row[min(in_row * V + j, a.experts - 1)]) - (double)most) * (in_row * V + j < a.experts ? 1.0 : 0.0);
          sum = over_row<L>(sum, Sum());
        }
        // An expert's place: how many of the others have a larger key, or the same and a lower number. One a lane and turn.
        for (int32_t i0 = 0; i0 < c.count; i0 += L) {
          const int32_t e = i0 + in_row < c.count ? mine[i0 + in_row] : -1;
          auto exact = [&](int32_t of) -> double {
            const double l = (double)Elem<T>::get(row[max(of, 0)]);
            return (kSigmoid ? 1.0 / (1.0 + exp(-l)) : nan == 0.0f ? exp(l - (double)most) / sum : 0.0) + (double)a.bias[max(of, 0)];
          };
          const double own = exact(e);
          int32_t place = 0;
          for (int32_t j0 = 0; j0 < c.count; j0 += L) {
            const int32_t their = j0 + in_row < c.count ? mine[j0 + in_row] : -1;
            const double their_key = i0 == j0 ? own : exact(their);
            for (int32_t j = 0; j < L && j0 + j < c.count; ++j) {
              const double k = __shfl(their_key, j, L);
              const int32_t o = __shfl(their, j, L);
              place += o >= 0 && (k > own || (k == own && o < e));
            }
          }
          wave_sync();
          if (e >= 0) sorted[(wave * kRows + row_in_wave) * L * V + place] = e;
        }
        wave_sync();
        for (int32_t i = in_row; i < c.count; i += L)
          if (mine[i] >= 0) mine[i] = sorted[(wave * kRows + row_in_wave) * L * V + i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = key_of(logit[j]);
      choose<false, L, V>(key, a.top, mine, [](int32_t, int32_t) { return true; });
    }
    wave_sync();
    // Weights: those of a row's choice relative to its largest chosen logit, where they are divided by their sum.
    const int32_t first = in_row < a.top ? mine[in_row] : -1;
    const float first_logit = Elem<T>::get(row[max(first, 0)]);
    auto chosen_logit = [&](int32_t i, int32_t e) -> float { return i == in_row ? first_logit : Elem<T>::get(row[max(e, 0)]); };
    float base = most;
    if (a.normalize) {
      int32_t top_key = first >= 0 ? key_of(first_logit) : kNoKey;
      for (int32_t i = in_row + L; i < a.top; i += L)
        if (mine[i] >= 0) top_key = __builtin_elementwise_max(top_key, key_of(Elem<T>::get(row[mine[i]])));
      base = of_key(over_row<L>(top_key, Max()));
    }
    auto value = [&](int32_t i, int32_t e) -> float {
      const float l = chosen_logit(i, e);
      float v;
      if constexpr (kSigmoid)  // sigmoids that are all small, as multiples of exp(base)
        v = a.normalize && base < 0 ? exp_of(l - base) * sigmoid_of(-l) : sigmoid_of(l);
      else
        v = exp_of(l - base) + nan;
      return e >= 0 ? v : 0.0f;
    };
    const float first_value = value(in_row, first);
    if (a.normalize) {
      total = first_value;
      for (int32_t i = in_row + L; i < a.top; i += L) total += value(i, mine[i]);
      total = over_row<L>(total, Sum());
    }
    if (token)
      for (int32_t i = in_row; i < a.top; i += L) {
        const int32_t e = mine[i];
        const float share = e >= 0 ? (i == in_row ? first_value : value(i, e)) / total : 0.0f;
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
      if constexpr (kSigmoid) d *= sigmoid_of(-Elem<T>::get(row[e]));
      mine[e] = d * a.scale;
    }
    wave_sync();
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = mine[in_row * V + j];
    if constexpr (!kSigmoid) {
      if (!a.normalize) {
        float logit[V], e[V], total = 0;
        load_vals<T, V>(row, in_row * V, a.experts, logit);
        const float most = largest<L>(logit);
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = exp_of(logit[j] - most), total += e[j];
        total = over_row<L>(total, Sum());
        const float by = total == 0.0f ? 0.0f : one_over(total) * c * a.scale;
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] -= logit[j] == kNone ? 0.0f : e[j] * by;
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
  const float most = largest<L>(logit);
  float total = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if constexpr (kSigmoid) {  // sigmoids that are all small, as multiples of exp(most)
      rest[j] = sigmoid_of(-logit[j]);
      p[j] = most < 0 ? exp_of(logit[j] - most) * rest[j] : sigmoid_of(logit[j]);
    } else {
      p[j] = exp_of(logit[j] - most);
    }
    if (kSigmoid && logit[j] == kNone) p[j] = 0.0f;
    total += p[j];
  }
  total = over_row<L>(total, Sum());
  const bool empty = total == 0.0f;  // no: some p is 1, or at least 1/2, or NaN
  const float by = empty ? 0.0f : one_over(total);
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

// The last step, by one workgroup, from `blocks` workgroups' sums: work-items share out first the blocks of an expert, of which each
// has kFlight under way at a time, then the experts. (65536 x 128, 256 blocks: 26 us with 512 work-items and loads as they come.)
template <int kThreads>
struct FinishWork {
  double p[kThreads], all[kThreads], pairs[kThreads];
  int32_t count[kThreads];
};
template <int kThreads, int kFlight>
__device__ inline void finish_balance(const BalanceArgs &a, int32_t blocks, const float *sums, const int32_t *parts, FinishWork<kThreads> &work) {
  const int tid = threadIdx.x;
  int32_t width = 1;
  while (width < a.experts && width < kThreads) width *= 2;
  const int32_t shares = kThreads / width, keys = a.experts + 1;
  int32_t tokens = 0;
  for (int32_t b = tid; b < blocks; b += kThreads) tokens += parts[(int64_t)b * keys + a.experts];
  double pairs = 0.0, all = 0.0;
  for (int32_t e0 = 0; e0 < a.experts; e0 += width) {
    const int32_t e = e0 + tid % width, from = min(e, a.experts - 1);
    int32_t count = 0;
    double p = 0.0;
    for (int32_t b = tid / width; b < blocks; b += shares * kFlight) {
      float f[kFlight];
      int32_t c[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const int32_t at = min(b + i * shares, blocks - 1);
        f[i] = sums[(int64_t)at * a.experts + from], c[i] = parts[(int64_t)at * keys + from];
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i)
        if (b + i * shares < blocks) p += (double)f[i], count += c[i];
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
  work.pairs[tid] = pairs, work.all[tid] = all, work.count[tid] = tokens;
  __syncthreads();
  for (int d = kThreads / 2; d > 0; d /= 2) {
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
  __shared__ FinishWork<kBalanceThreads> work;
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
  auto load = [&](int64_t t0, float (&logit)[V]) {
    load_vals<T, V>(static_cast<const raw *>(a.logits) + min(t0 + row_in_wave, a.tokens - 1) * a.stride, in_row * V, a.experts, logit);
  };
  int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows;
  float now[V], soon[V];  // a row's logits, and the next one's, which are loaded meanwhile
  if (t0 < a.tokens) load(t0, now);
  for (; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    float p[V], rest[V];
    if (t0 + step < a.tokens) load(t0 + step, soon);
    const bool empty = shares_of<L, V, kSigmoid>(now, p, rest);
#pragma unroll
    for (int j = 0; j < V; ++j) now[j] = soon[j];
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
    finish_balance<kBalanceThreads, 1>(a, 1, sums[0], counts, work);
  } else {
    for (int32_t e = threadIdx.x; e <= a.experts; e += kBalanceThreads) a.parts[(int64_t)blockIdx.x * (a.experts + 1) + e] = counts[e];
  }
}

constexpr unsigned kGradBlocks = 1024;  // 65536 x 128 BF16: a workgroup for every 16 rows 20.3 us, these 14.3 us
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void expert_balance_sum_kernel(BalanceArgs a, int32_t blocks) {
  __shared__ FinishWork<kSumThreads> work;
  finish_balance<kSumThreads, 16>(a, blocks, a.sums, a.parts, work);
}

// dlogit[t, e] = dloss experts / (N T) p (counts[e] - sum_j counts[j] p[t, j]) (1 - sigmoid, for sigmoids). The p of a row add up to 1, so
// that counts serve less their mean, too: loads that are nearly alike, which the loss is for, would else lose the digits that they share.
template <int T, int L, int V, bool kSigmoid>
__global__ __launch_bounds__(kRouteThreads) void expert_balance_grad_kernel(BalanceArgs a) {
  typedef typename Elem<T>::raw raw;
  constexpr int kRows = 64 / L, kWaves = kRouteThreads / 64;
  const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63, in_row = in_wave & (L - 1), row_in_wave = in_wave / L;
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  auto load = [&](int64_t t0, float (&logit)[V]) {
    load_vals<T, V>(static_cast<const raw *>(a.logits) + min(t0 + row_in_wave, a.tokens - 1) * a.stride, in_row * V, a.experts, logit);
  };
  int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows;
  float soon[V];  // the next row's logits, which are loaded meanwhile
  if (t0 < a.tokens) load(t0, soon);
  float count[V];
  int32_t whole[V];
  double n = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) whole[j] = in_row * V + j < a.experts ? a.kept[in_row * V + j] : 0, n += whole[j];
  n = over_row<L>(n, Sum());
#pragma unroll
  for (int j = 0; j < V; ++j) count[j] = (float)(whole[j] - n / a.experts);
  const double tokens = a.kept[a.experts];
  const float factor = n > 0 && tokens > 0 ? (float)((double)*a.dloss * a.experts / (n * tokens)) : 0.0f;
  for (; t0 < a.tokens; t0 += step) {
    const bool token = t0 + row_in_wave < a.tokens;
    const int64_t t = token ? t0 + row_in_wave : a.tokens - 1;
    float logit[V], p[V], rest[V], c = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) logit[j] = soon[j];
    if (t0 + step < a.tokens) load(t0 + step, soon);
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

// Workgroups of the first launch: one for up to 16384 logits and ids, which then makes the loss too; else one for every 16384, up to 256
// and, lest the second launch has much to add up, up to 32768 experts' sums.
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
  if (blocks > 1) hipLaunchKernelGGL(expert_balance_sum_kernel, dim3(1), dim3(kSumThreads), 0, s, a, blocks);
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
  hipLaunchKernelGGL((expert_balance_grad_kernel<T, L, V, S>), dim3(std::min(route_grid<L>(tokens), kGradBlocks)), dim3(kRouteThreads), 0, s, a)
#define CALL(T, L, V) \
  if (scores == MPS_SCORES_SIGMOID) { LAUNCH(T, L, V, true); } else { LAUNCH(T, L, V, false); }
  MPS_BY_LOGITS(type, experts, CALL);
#undef CALL
#undef LAUNCH
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
