// Tokens to their experts and back: a stable counting sort of (token, expert) pairs, the gather of
// their rows, the weighted sum of the experts' rows, and its gradients.
//
// Sort: place(pair) = number of pairs of lower experts + number of earlier pairs of its own; the
// counts need no order, the places come from counts alone, so the result does not depend on the
// order in which anything ran. Gather, sum and gradients read each row that they need once and
// are bound by memory; sums are FP32, over a token's pairs in their order.
#include "mxfp4_common.h"

namespace mps {
namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

// The expert of pair i, or `experts` for a pair of none.
template <typename Id>
__device__ inline int32_t expert_of(const Id *ids, int64_t i, int32_t experts) {
  const Id e = ids[i];
  return e >= 0 && e < experts ? (int32_t)e : experts;
}

// Up to kOneWorkgroup pairs are sorted by one workgroup; more in chunks, a workgroup each, of which
// each counts its pairs first, in a launch of its own. (65536 pairs of 128 experts: 78 us by one
// workgroup, @CHUNKS@ in chunks.)
constexpr int32_t kOneWorkgroup = 4096, kMostChunks = 64;
inline int32_t sort_chunk(int64_t pairs) {
  const int64_t chunk = (pairs + kMostChunks - 1) / kMostChunks;
  return pairs <= kOneWorkgroup ? kOneWorkgroup : (int32_t)(chunk < 2048 ? 2048 : (chunk + 1023) / 1024 * 1024);
}

template <typename Id>
__global__ __launch_bounds__(kSortThreads) void expert_count_kernel(const Id *__restrict__ ids, int32_t pairs,
                                                                    int32_t chunk, int32_t experts,
                                                                    int32_t *__restrict__ chunk_counts) {
  __shared__ int32_t counts[MPS_MAX_EXPERTS + 1];
  for (int32_t i = threadIdx.x; i <= experts; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * chunk, last = min(first + chunk, (int64_t)pairs);
  for (int64_t i = first + threadIdx.x; i < last; i += kSortThreads) atomicAdd(&counts[expert_of(ids, i, experts)], 1);
  __syncthreads();
  for (int32_t i = threadIdx.x; i <= experts; i += kSortThreads) chunk_counts[(int64_t)blockIdx.x * (experts + 1) + i] = counts[i];
}

// A workgroup sorts its chunk: each wave counts a stretch of it, the counts become the places where
// each (expert, wave) starts, and each wave goes over its stretch again, 64 pairs at a time.
// Lanes of one expert find each other by ballots over the expert's bits.
template <typename Id>
__global__ __launch_bounds__(kSortThreads) void expert_sort_kernel(const Id *__restrict__ ids, int32_t pairs,
                                                                   int32_t chunk, int32_t experts, int32_t bits,
                                                                   const int32_t *__restrict__ chunk_counts,
                                                                   int32_t *__restrict__ order,
                                                                   int32_t *__restrict__ positions,
                                                                   int32_t *__restrict__ offsets) {
  __shared__ int32_t counts[kSortWaves * (MPS_MAX_EXPERTS + 1)];  // [kSortWaves][experts + 1]
  __shared__ int32_t totals[MPS_MAX_EXPERTS + 1], before[MPS_MAX_EXPERTS + 1], wave_sums[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t keys = experts + 1;
  for (int32_t i = tid; i < kSortWaves * keys; i += kSortThreads) counts[i] = 0;
  for (int32_t i = tid; i < keys; i += kSortThreads) totals[i] = before[i] = 0;
  __syncthreads();
  const int32_t stretch = (chunk / kSortWaves + 63) / 64 * 64;
  const int64_t begin = (int64_t)blockIdx.x * chunk + wave * stretch, end = min(((int64_t)blockIdx.x + 1) * chunk, (int64_t)pairs);
  const int32_t first = (int32_t)min(begin, end), last = (int32_t)min(begin + stretch, end);
  for (int32_t i = first + lane; i < last; i += 64) atomicAdd(&counts[wave * keys + expert_of(ids, i, experts)], 1);
  if (chunk_counts) {  // this chunk's pairs come after those of the chunks before it
    const int32_t chunks = gridDim.x;
    for (int32_t i = tid; i < chunks * keys; i += kSortThreads) {
      const int32_t c = i / keys, e = i - c * keys, n = chunk_counts[i];
      if (n > 0) {
        atomicAdd(&totals[e], n);
        if (c < (int32_t)blockIdx.x) atomicAdd(&before[e], n);
      }
    }
  }
  __syncthreads();
  // Exclusive sums over experts: kSortThreads >= MPS_MAX_EXPERTS, so a work-item has one expert, and
  // work-item 0 the pairs of none too, which come after all others.
  int32_t mine = 0;
  if (tid < experts) {
    if (chunk_counts)
      mine = totals[tid];
    else
      for (int w = 0; w < kSortWaves; ++w) mine += counts[w * keys + tid];
  }
  int32_t upto = mine;
  for (int d = 1; d < 64; d *= 2) {
    const int32_t v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) wave_sums[wave] = upto;
  __syncthreads();
  int32_t start = upto - mine, total = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < wave) start += wave_sums[w];
    total += wave_sums[w];
  }
  if (blockIdx.x == 0) {
    if (tid < experts) offsets[tid] = start;
    if (tid == 0) offsets[experts] = total;
  }
  auto spread = [&](int32_t e, int32_t at) {
    at += before[e];
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t c = counts[w * keys + e];
      counts[w * keys + e] = at;
      at += c;
    }
  };
  if (tid < experts) spread(tid, start);
  if (tid == 0) spread(experts, total);
  __syncthreads();
  for (int32_t i0 = first; i0 < last; i0 += 64) {
    const int32_t i = i0 + lane;
    const bool in = i < last;
    const int32_t e = in ? expert_of(ids, i, experts) : -1;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    if (in) {
      int32_t *at = &counts[wave * keys + e];
      const int32_t place = *at + __popcll(same & ((1ull << lane) - 1));
      __builtin_amdgcn_wave_barrier();  // all lanes have read before the last of each expert writes
      if (same >> lane == 1) *at = place + 1;
      order[place] = i;
      positions[i] = e < experts ? place : -1;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

constexpr int kRowThreads = 256;

// kVec elements at a time: 16 bytes where rows are whole 16-byte pieces, else one.
template <int T, int kVec>
struct Piece {
  typename Elem<T>::raw v[kVec];
};

template <int T, int kVec>
__global__ __launch_bounds__(kRowThreads) void expert_gather_kernel(const typename Elem<T>::raw *__restrict__ x,
                                                                    int32_t tokens, int32_t top, int64_t pairs,
                                                                    int32_t experts, int64_t width,
                                                                    const int32_t *__restrict__ order,
                                                                    const int32_t *__restrict__ offsets,
                                                                    typename Elem<T>::raw *__restrict__ rows) {
  typedef Piece<T, kVec> P;
  const int64_t j = blockIdx.x;
  const bool there = j < offsets[experts];
  const int32_t token = min((uint32_t)order[j] / (uint32_t)top, (uint32_t)tokens - 1);
  const P *src = reinterpret_cast<const P *>(x + (int64_t)token * width);
  P *dst = reinterpret_cast<P *>(rows + j * width);
  const P zero = {};
  for (int64_t c = threadIdx.x; c < width / kVec; c += kRowThreads) dst[c] = there ? src[c] : zero;
}

template <int T, int kVec>
__global__ __launch_bounds__(kRowThreads) void expert_combine_kernel(const typename Elem<T>::raw *__restrict__ y,
                                                                     const void *__restrict__ weights, int32_t wtype,
                                                                     int32_t top, int64_t pairs, int64_t width,
                                                                     const int32_t *__restrict__ positions,
                                                                     typename Elem<T>::raw *__restrict__ out) {
  typedef Piece<T, kVec> P;
  const int64_t t = blockIdx.x;
  for (int64_t c = threadIdx.x; c < width / kVec; c += kRowThreads) {
    float sum[kVec] = {};
    for (int32_t i = 0; i < top; ++i) {
      const int64_t pair = t * top + i;
      const int32_t at = positions[pair];
      if (at < 0 || at >= pairs) continue;
      const float w = weights ? load_as_float(weights, wtype, pair) : 1.0f;
      const P p = reinterpret_cast<const P *>(y + (int64_t)at * width)[c];
      for (int v = 0; v < kVec; ++v) sum[v] += w * Elem<T>::get(p.v[v]);
    }
    P o;
    for (int v = 0; v < kVec; ++v) o.v[v] = Elem<T>::put(sum[v]);
    reinterpret_cast<P *>(out + t * width)[c] = o;
  }
}

// A workgroup a sorted row; the lanes' products are added up by a tree, whose order is fixed.
template <int T, int kVec>
__global__ __launch_bounds__(kRowThreads) void expert_combine_grad_kernel(
    const typename Elem<T>::raw *__restrict__ y, const typename Elem<T>::raw *__restrict__ dout,
    const void *__restrict__ weights, int32_t wtype, int32_t tokens, int32_t top, int64_t pairs, int32_t experts,
    int64_t width, const int32_t *__restrict__ order, const int32_t *__restrict__ offsets,
    typename Elem<T>::raw *__restrict__ dy, void *__restrict__ dweights) {
  typedef Piece<T, kVec> P;
  __shared__ float parts[kRowThreads / 64];
  const int64_t j = blockIdx.x;
  const bool there = j < offsets[experts];
  const uint32_t pair = min((uint32_t)order[j], (uint32_t)(pairs - 1)), token = pair / (uint32_t)top;
  const float w = load_as_float(weights, wtype, pair);
  float dot = 0;
  for (int64_t c = threadIdx.x; c < width / kVec; c += kRowThreads) {
    P o = {};
    if (there) {
      const P g = reinterpret_cast<const P *>(dout + (int64_t)token * width)[c];
      const P p = reinterpret_cast<const P *>(y + j * width)[c];
      for (int v = 0; v < kVec; ++v) {
        const float gv = Elem<T>::get(g.v[v]);
        dot += gv * Elem<T>::get(p.v[v]);
        o.v[v] = Elem<T>::put(w * gv);
      }
    }
    reinterpret_cast<P *>(dy + j * width)[c] = o;
  }
  for (int d = 32; d > 0; d /= 2) dot += __shfl_xor(dot, d);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0;
    for (int i = 0; i < kRowThreads / 64; ++i) sum += parts[i];
    store_as(dweights, wtype, pair, there ? sum : 0.0f);
  }
}

template <typename Id>
void launch_sort(const Id *ids, int32_t pairs, int32_t chunk, int32_t chunks, int32_t experts, int32_t *counts,
                 int32_t *order, int32_t *positions, int32_t *offsets, hipStream_t stream) {
  int32_t bits = 1;
  while ((1 << bits) <= experts) ++bits;
  if (counts)
    hipLaunchKernelGGL((expert_count_kernel<Id>), dim3(chunks), dim3(kSortThreads), 0, stream, ids, pairs, chunk,
                       experts, counts);
  hipLaunchKernelGGL((expert_sort_kernel<Id>), dim3(chunks), dim3(kSortThreads), 0, stream, ids, pairs, chunk, experts,
                     bits, counts, order, positions, offsets);
}

int check_sizes(const char *what, int64_t tokens, int64_t top, int64_t experts) {
  if (tokens < 0 || top < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (experts < 1 || experts > MPS_MAX_EXPERTS)
    return fail(MPS_ERR_INVALID_ARGUMENT, "%s: experts must be in [1, %d]", what, MPS_MAX_EXPERTS);
  if (top > 0 && tokens > (INT32_MAX - 1024) / top)
    return fail(MPS_ERR_INVALID_ARGUMENT, "%s: over 2^31 - 1025 pairs of tokens and experts", what);
  return MPS_OK;
}

// 16-byte pieces where every row starts at a 16-byte address.
template <typename... Ptr>
bool whole_rows(int64_t width, int32_t type, Ptr... p) {
  return width * type_bytes(type) % 16 == 0 && (aligned16(p) && ...);
}

#define MPS_BY_TYPE(type, whole, CALL)                                  \
  do {                                                                  \
    if ((type) == MPS_TYPE_F32) {                                       \
      if (whole) { CALL(MPS_TYPE_F32, 4); } else { CALL(MPS_TYPE_F32, 1); }     \
    } else if ((type) == MPS_TYPE_BF16) {                               \
      if (whole) { CALL(MPS_TYPE_BF16, 8); } else { CALL(MPS_TYPE_BF16, 1); }   \
    } else {                                                            \
      if (whole) { CALL(MPS_TYPE_F16, 8); } else { CALL(MPS_TYPE_F16, 1); }     \
    }                                                                   \
  } while (0)

}  // namespace
}  // namespace mps

using namespace mps;

extern "C" {

int mps_expert_sort_workspace(int64_t tokens, int64_t top, int64_t experts, int64_t *bytes) {
  last_error().clear();
  const int rc = check_sizes("expert_sort", tokens, top, experts);
  if (rc != MPS_OK) return rc;
  if (!bytes) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_sort: null pointer");
  const int64_t pairs = tokens * top, chunk = sort_chunk(pairs), chunks = (pairs + chunk - 1) / chunk;
  *bytes = chunks > 1 ? chunks * (experts + 1) * 4 : 0;
  return MPS_OK;
}

int mps_expert_sort(const void *ids, int32_t ids_64, int64_t tokens, int64_t top, int64_t experts, int32_t *order,
                    int32_t *positions, int32_t *offsets, void *workspace, int64_t workspace_bytes, void *stream) {
  last_error().clear();
  const int rc = check_sizes("expert_sort", tokens, top, experts);
  if (rc != MPS_OK) return rc;
  const int32_t pairs = (int32_t)(tokens * top);
  if (!offsets || (pairs > 0 && (!ids || !order || !positions)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_sort: null pointer");
  const int32_t chunk = sort_chunk(pairs), chunks = pairs > 0 ? (pairs + chunk - 1) / chunk : 1;
  if (chunks > 1 && (!workspace || workspace_bytes < (int64_t)chunks * (experts + 1) * 4))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_sort: %lld bytes of workspace are needed",
                (long long)chunks * (experts + 1) * 4);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int32_t *const counts = chunks > 1 ? static_cast<int32_t *>(workspace) : nullptr;
  if (ids_64)
    launch_sort(static_cast<const int64_t *>(ids), pairs, chunk, chunks, (int32_t)experts, counts, order, positions, offsets, s);
  else
    launch_sort(static_cast<const int32_t *>(ids), pairs, chunk, chunks, (int32_t)experts, counts, order, positions, offsets, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_gather(const void *x, int32_t type, int64_t tokens, int64_t top, int64_t experts, int64_t width,
                      const int32_t *order, const int32_t *offsets, void *rows, void *stream) {
  last_error().clear();
  const int rc = check_sizes("expert_gather", tokens, top, experts);
  if (rc != MPS_OK) return rc;
  if (!is_float_type(type) || width < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_gather: bad type or width");
  const int64_t pairs = tokens * top;
  if (pairs == 0 || width == 0) return MPS_OK;
  if (!x || !order || !offsets || !rows) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_gather: null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define CALL(T, V)                                                                                             \
  hipLaunchKernelGGL((expert_gather_kernel<T, V>), dim3((unsigned)pairs), dim3(kRowThreads), 0, s,            \
                     static_cast<const Elem<T>::raw *>(x), (int32_t)tokens, (int32_t)top, pairs, (int32_t)experts, \
                     width, order, offsets, static_cast<Elem<T>::raw *>(rows))
  MPS_BY_TYPE(type, whole_rows(width, type, x, rows), CALL);
#undef CALL
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_combine(const void *y, int32_t type, const void *weights, int32_t weights_type, int64_t tokens,
                       int64_t top, int64_t width, const int32_t *positions, void *out, void *stream) {
  last_error().clear();
  const int rc = check_sizes("expert_combine", tokens, top, 1);
  if (rc != MPS_OK) return rc;
  if (!is_float_type(type) || (weights && !is_float_type(weights_type)) || width < 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_combine: bad type or width");
  if (tokens == 0 || width == 0) return MPS_OK;
  if (!out || (top > 0 && (!y || !positions))) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_combine: null pointer");
  const int64_t pairs = tokens * top;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define CALL(T, V)                                                                                            \
  hipLaunchKernelGGL((expert_combine_kernel<T, V>), dim3((unsigned)tokens), dim3(kRowThreads), 0, s,         \
                     static_cast<const Elem<T>::raw *>(y), weights, weights_type, (int32_t)top, pairs, width, \
                     positions, static_cast<Elem<T>::raw *>(out))
  MPS_BY_TYPE(type, whole_rows(width, type, y, out), CALL);
#undef CALL
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_combine_grad(const void *y, const void *dout, int32_t type, const void *weights, int32_t weights_type,
                            int64_t tokens, int64_t top, int64_t experts, int64_t width, const int32_t *order,
                            const int32_t *offsets, void *dy, void *dweights, void *stream) {
  last_error().clear();
  const int rc = check_sizes("expert_combine_grad", tokens, top, experts);
  if (rc != MPS_OK) return rc;
  if (!is_float_type(type) || !is_float_type(weights_type) || width < 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_combine_grad: bad type or width");
  const int64_t pairs = tokens * top;
  if (pairs == 0) return MPS_OK;
  if (!weights || !order || !offsets || !dweights || (width > 0 && (!y || !dout || !dy)))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_combine_grad: null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define CALL(T, V)                                                                                                   \
  hipLaunchKernelGGL((expert_combine_grad_kernel<T, V>), dim3((unsigned)pairs), dim3(kRowThreads), 0, s,            \
                     static_cast<const Elem<T>::raw *>(y), static_cast<const Elem<T>::raw *>(dout), weights,         \
                     weights_type, (int32_t)tokens, (int32_t)top, pairs, (int32_t)experts, width, order, offsets,    \
                     static_cast<Elem<T>::raw *>(dy), dweights)
  MPS_BY_TYPE(type, whole_rows(width, type, y, dout, dy), CALL);
#undef CALL
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
