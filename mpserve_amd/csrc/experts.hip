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
// workgroup, 13 in chunks.)
constexpr int32_t kOneWorkgroup = 4096, kMostChunks = 64;
inline int32_t sort_chunk(int64_t pairs) {
  const int64_t chunk = (pairs + kMostChunks - 1) / kMostChunks;
  return pairs <= kOneWorkgroup ? kOneWorkgroup : (int32_t)(chunk < 2048 ? 2048 : (chunk + 1023) / 1024 * 1024);
}
inline int64_t sort_chunks(int64_t pairs) {  // in 64 bits: near 2^31 pairs the sum passes 32
  const int64_t chunk = sort_chunk(pairs);
  return pairs > 0 ? (pairs + chunk - 1) / chunk : 1;
}
inline int64_t sort_bytes(int64_t pairs, int64_t experts) {
  const int64_t chunks = sort_chunks(pairs);
  return chunks > 1 ? chunks * (experts + 1) * 4 : 0;
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

// Rows are worked off in pieces of 16 bytes, at any alignment; the last piece of a row may be a part
// of one. A token's pieces are shared out to a power of two of work-items (`lanes`, at most the
// workgroup), so that narrow rows share a workgroup. A token's row is read once for all its pairs: gathered by
// place instead, rows of x came from beyond the L2 once a pair (8192 tokens x 4096 BF16, 8 of 128 experts:
// 171 us, by token 100).
constexpr int kRowThreads = 256, kPairs = 4;  // pairs whose pieces are in flight together

template <int T>
struct Piece {
  typedef typename Elem<T>::raw raw;
  static constexpr int kVec = 16 / sizeof(raw);
  u32x4 bits = {0, 0, 0, 0};

  __device__ float get(int i) const {
    if constexpr (T == MPS_TYPE_F32)
      return __uint_as_float(bits[i]);
    else
      return Elem<T>::get((uint16_t)(bits[i / 2] >> (16 * (i % 2))));
  }
  __device__ void put(int i, float f) {
    if constexpr (T == MPS_TYPE_F32)
      bits[i] = __float_as_uint(f);
    else
      bits[i / 2] |= (uint32_t)Elem<T>::put(f) << (16 * (i % 2));
  }
  static __device__ Piece load(const raw *row, int64_t col, int64_t width) {
    Piece p;
    if (col + kVec <= width) {
      p.bits = *reinterpret_cast<const u32x4_any *>(row + col);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (col + i < width) {  // bits as they are, those of a NaN too
          if constexpr (T == MPS_TYPE_F32)
            p.bits[i] = __float_as_uint(row[col + i]);
          else
            p.bits[i / 2] |= (uint32_t)row[col + i] << (16 * (i % 2));
        }
    }
    return p;
  }
  __device__ void store(raw *row, int64_t col, int64_t width) const {
    if (col + kVec <= width) {
      *reinterpret_cast<u32x4_any *>(row + col) = bits;
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (col + i < width) {
          if constexpr (T == MPS_TYPE_F32)
            row[col + i] = __uint_as_float(bits[i]);
          else
            row[col + i] = (uint16_t)(bits[i / 2] >> (16 * (i % 2)));
        }
    }
  }
};

struct RowArgs {
  const void *in, *dout, *weights;  // x or y
  void *out, *dweights;
  const int32_t *order, *positions, *offsets;
  int64_t tokens, top, pairs, width;
  int32_t experts, weights_type, lanes;
};

// The places of pairs of no expert, and the rows there: zeros. Workgroups past the tokens' take them in turn.
template <int T, bool kRows, bool kWeights>
__device__ inline void zero_rows(const RowArgs &a, int64_t block, int64_t blocks) {
  typedef Piece<T> P;
  const int64_t first = min(max((int64_t)a.offsets[a.experts], (int64_t)0), a.pairs);
  for (int64_t j = first + block; j < a.pairs; j += blocks) {
    if constexpr (kRows)
      for (int64_t col = threadIdx.x * P::kVec; col < a.width; col += kRowThreads * P::kVec)
        P{}.store(static_cast<typename Elem<T>::raw *>(a.out) + j * a.width, col, a.width);
    if (kWeights && threadIdx.x == 0) {
      const int64_t pair = a.order[j];
      if (pair >= 0 && pair < a.pairs) store_as(a.dweights, a.weights_type, pair, 0.0f);
    }
  }
}
constexpr int kZeroBlocks = 128;

template <int T, bool kWide>
__global__ __launch_bounds__(kRowThreads) void expert_gather_kernel(RowArgs a, int64_t token_blocks) {
  typedef Piece<T> P;
  typedef typename Elem<T>::raw raw;
  const int64_t grid = gridDim.x - kZeroBlocks;
  if (blockIdx.x >= grid) return zero_rows<T, true, false>(a, blockIdx.x - grid, kZeroBlocks);
  const int32_t lanes = kWide ? kRowThreads : a.lanes;  // a token a workgroup: its places are scalars
  for (int64_t block = blockIdx.x; block < token_blocks; block += grid) {
    const int64_t t = kWide ? block : block * (kRowThreads / lanes) + threadIdx.x / lanes;
    if (t >= a.tokens) continue;
    const raw *const row = static_cast<const raw *>(a.in) + t * a.width;
    raw *const out = static_cast<raw *>(a.out);
    for (int64_t col = (threadIdx.x & (lanes - 1)) * P::kVec; col < a.width; col += lanes * P::kVec) {
      const P p = P::load(row, col, a.width);
      for (int64_t i = 0; i < a.top; ++i) {
        const int32_t at = a.positions[t * a.top + i];
        if (at >= 0 && at < a.pairs) p.store(out + at * a.width, col, a.width);
      }
    }
  }
}

// (The pointers stand by themselves so that the compiler may take them to be apart, and loads of the places
// and weights, alike for all lanes, to be scalar.)
template <int T, bool kWide>
__global__ __launch_bounds__(kRowThreads) void expert_combine_kernel(RowArgs a, int64_t token_blocks,
                                                                     const typename Elem<T>::raw *__restrict__ y,
                                                                     const void *__restrict__ weights,
                                                                     const int32_t *__restrict__ positions,
                                                                     typename Elem<T>::raw *__restrict__ out) {
  typedef Piece<T> P;
  const int32_t lanes = kWide ? kRowThreads : a.lanes;  // a token a workgroup: its places are scalars
  for (int64_t block = blockIdx.x; block < token_blocks; block += gridDim.x) {
    const int64_t t = kWide ? block : block * (kRowThreads / lanes) + threadIdx.x / lanes;
    if (t >= a.tokens) continue;
    for (int64_t col = (threadIdx.x & (lanes - 1)) * P::kVec; col < a.width; col += lanes * P::kVec) {
      const bool whole = col + P::kVec <= a.width;
      float sum[P::kVec] = {};
      for (int64_t i0 = 0; i0 < a.top; i0 += kPairs) {
        // Whole pieces without branches, so that their loads are in flight together: an absent pair reads row 0.
        int64_t at[kPairs];
        bool there[kPairs];
        float w[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int64_t in = i0 + i < a.top ? i0 + i : 0;
          const int32_t p = positions[t * a.top + in];
          there[i] = i0 + i < a.top && p >= 0 && p < a.pairs;
          at[i] = there[i] ? p : 0;
          w[i] = 1.0f;
        }
        if (weights) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) w[i] = load_as_float(weights, a.weights_type, t * a.top + (i0 + i < a.top ? i0 + i : 0));
        }
        P p[kPairs];
        if (whole) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) p[i].bits = *reinterpret_cast<const u32x4_any *>(y + at[i] * a.width + col);
        } else {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) p[i] = P::load(y + at[i] * a.width, col, a.width);
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
#pragma unroll
          for (int v = 0; v < P::kVec; ++v) sum[v] = there[i] ? __builtin_fmaf(w[i], p[i].get(v), sum[v]) : sum[v];
      }
      P o;
#pragma unroll
      for (int v = 0; v < P::kVec; ++v) o.put(v, sum[v]);
      o.store(out + t * a.width, col, a.width);
    }
  }
}

// kPairs pairs of a token at a time. A work-item's products are added up in the order of its pieces, and
// the work-items' sums by a tree: a fixed order. kDy and kDw: which gradients are asked for; the weights' alone
// write no rows, those of y alone read none.
template <int T, bool kWide, bool kDy, bool kDw>
__global__ __launch_bounds__(kRowThreads) void expert_combine_grad_kernel(RowArgs a, int64_t token_blocks) {
  typedef Piece<T> P;
  typedef typename Elem<T>::raw raw;
  __shared__ float parts[kPairs][kRowThreads / 64];
  const int64_t grid = gridDim.x - kZeroBlocks;
  if (blockIdx.x >= grid) return zero_rows<T, kDy, kDw>(a, blockIdx.x - grid, kZeroBlocks);
  const int32_t lanes = kWide ? kRowThreads : a.lanes;  // a token a workgroup: its places are scalars
  for (int64_t block = blockIdx.x; block < token_blocks; block += grid) {
    const int64_t t = kWide ? block : block * (kRowThreads / lanes) + threadIdx.x / lanes;
    const bool token = t < a.tokens;
    const raw *const y = static_cast<const raw *>(a.in), *const g = static_cast<const raw *>(a.dout) + (token ? t : 0) * a.width;
    raw *const dy = static_cast<raw *>(a.out);
    for (int64_t i0 = 0; i0 < a.top; i0 += kPairs) {
      float w[kPairs], dot[kPairs] = {};
      int64_t at[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int64_t pair = t * a.top + i0 + i;
        at[i] = token && i0 + i < a.top ? a.positions[pair] : -1;
        if (at[i] >= a.pairs) at[i] = -1;
        w[i] = kDy && at[i] >= 0 ? load_as_float(a.weights, a.weights_type, pair) : 0.0f;
      }
      if (token)
        for (int64_t col = (threadIdx.x & (lanes - 1)) * P::kVec; col < a.width; col += lanes * P::kVec) {
          const P d = P::load(g, col, a.width);
          P p[kPairs];
          if constexpr (kDw) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i)
              if (at[i] >= 0) p[i] = P::load(y + at[i] * a.width, col, a.width);
          }
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            if (at[i] >= 0) {
#pragma clang fp contract(off)  // one multiply-add each, whichever gradients are asked for (FP16 pairs became dot products in one form)
              P o;
#pragma unroll
              for (int v = 0; v < P::kVec; ++v) {
                const float gv = d.get(v);
                if constexpr (kDw) dot[i] = __builtin_fmaf(gv, p[i].get(v), dot[i]);
                if constexpr (kDy) o.put(v, w[i] * gv);
              }
              if constexpr (kDy) o.store(dy + at[i] * a.width, col, a.width);
            }
        }
      if constexpr (!kDw) continue;
      const int in_wave = lanes < 64 ? lanes : 64;
      for (int d = in_wave / 2; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < kPairs; ++i) dot[i] += __shfl_xor(dot[i], d);
      if (lanes > 64) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
          for (int i = 0; i < kPairs; ++i) parts[i][threadIdx.x >> 6] = dot[i];
        __syncthreads();
        const int first = threadIdx.x / lanes * (lanes / 64);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          dot[i] = 0;
          for (int j = 0; j < lanes / 64; ++j) dot[i] += parts[i][first + j];
        }
        __syncthreads();
      }
      if ((threadIdx.x & (lanes - 1)) == 0)
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          if (at[i] >= 0) store_as(a.dweights, a.weights_type, t * a.top + i0 + i, dot[i]);
    }
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

int32_t lanes_of(int64_t width, int32_t type) {
  const int64_t pieces = (width * type_bytes(type) + 15) / 16;
  int32_t lanes = 1;
  while (lanes < kRowThreads && lanes < pieces) lanes *= 2;
  return lanes;
}

#define MPS_BY_TYPE(type, wide, CALL)                                                       \
  do {                                                                                      \
    if ((type) == MPS_TYPE_F32) {                                                           \
      if (wide) { CALL(MPS_TYPE_F32, true); } else { CALL(MPS_TYPE_F32, false); }           \
    } else if ((type) == MPS_TYPE_BF16) {                                                   \
      if (wide) { CALL(MPS_TYPE_BF16, true); } else { CALL(MPS_TYPE_BF16, false); }         \
    } else {                                                                                \
      if (wide) { CALL(MPS_TYPE_F16, true); } else { CALL(MPS_TYPE_F16, false); }           \
    }                                                                                       \
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
  *bytes = sort_bytes(tokens * top, experts);
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
  const int32_t chunk = sort_chunk(pairs), chunks = (int32_t)sort_chunks(pairs);
  const int64_t need = sort_bytes(pairs, experts);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_sort: %lld bytes of workspace are needed", (long long)need);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int32_t *const counts = need > 0 ? static_cast<int32_t *>(workspace) : nullptr;
  if (ids_64)
    launch_sort(static_cast<const int64_t *>(ids), pairs, chunk, chunks, (int32_t)experts, counts, order, positions, offsets, s);
  else
    launch_sort(static_cast<const int32_t *>(ids), pairs, chunk, chunks, (int32_t)experts, counts, order, positions, offsets, s);
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_gather(const void *x, int32_t type, int64_t tokens, int64_t top, int64_t experts, int64_t width,
                      const int32_t *order, const int32_t *positions, const int32_t *offsets, void *rows, void *stream) {
  last_error().clear();
  const int rc = check_sizes("expert_gather", tokens, top, experts);
  if (rc != MPS_OK) return rc;
  if (!is_float_type(type) || width < 0) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_gather: bad type or width");
  const int64_t pairs = tokens * top;
  if (pairs == 0 || width == 0) return MPS_OK;
  if (!x || !order || !positions || !offsets || !rows) return fail(MPS_ERR_INVALID_ARGUMENT, "expert_gather: null pointer");
  RowArgs a = {};
  a.in = x, a.out = rows, a.order = order, a.positions = positions, a.offsets = offsets;
  a.tokens = tokens, a.top = top, a.pairs = pairs, a.width = width, a.experts = (int32_t)experts, a.lanes = lanes_of(width, type);
  const int64_t per = kRowThreads / a.lanes, blocks = (tokens + per - 1) / per;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define CALL(T, W) \
  hipLaunchKernelGGL((expert_gather_kernel<T, W>), dim3(workgroups(blocks) + kZeroBlocks), dim3(kRowThreads), 0, s, a, blocks)
  MPS_BY_TYPE(type, a.lanes == kRowThreads, CALL);
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
  RowArgs a = {};
  a.in = y, a.out = out, a.weights = weights, a.weights_type = weights_type, a.positions = positions;
  a.tokens = tokens, a.top = top, a.pairs = tokens * top, a.width = width, a.lanes = lanes_of(width, type);
  const int64_t per = kRowThreads / a.lanes, blocks = (tokens + per - 1) / per;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define CALL(T, W) hipLaunchKernelGGL((expert_combine_kernel<T, W>), dim3(workgroups(blocks)), dim3(kRowThreads), 0, s, a, blocks, \
                                      static_cast<const Elem<T>::raw *>(y), weights, positions, static_cast<Elem<T>::raw *>(out))
  MPS_BY_TYPE(type, a.lanes == kRowThreads, CALL);
#undef CALL
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

int mps_expert_combine_grad(const void *y, const void *dout, int32_t type, const void *weights, int32_t weights_type,
                            int64_t tokens, int64_t top, int64_t experts, int64_t width, const int32_t *order,
                            const int32_t *positions, const int32_t *offsets, void *dy, void *dweights, void *stream) {
  last_error().clear();
  const int rc = check_sizes("expert_combine_grad", tokens, top, experts);
  if (rc != MPS_OK) return rc;
  if (!is_float_type(type) || !is_float_type(weights_type) || width < 0)
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_combine_grad: bad type or width");
  const int64_t pairs = tokens * top;
  if (pairs == 0 || (width == 0 && !dweights)) return MPS_OK;
  if (!weights || !order || !positions || !offsets || (!dy && !dweights) || (width > 0 && (!dout || (dweights && !y))))
    return fail(MPS_ERR_INVALID_ARGUMENT, "expert_combine_grad: null pointer");
  RowArgs a = {};
  a.in = y, a.dout = dout, a.out = dy, a.weights = weights, a.weights_type = weights_type, a.dweights = dweights;
  a.order = order, a.positions = positions, a.offsets = offsets;
  a.tokens = tokens, a.top = top, a.pairs = pairs, a.width = width, a.experts = (int32_t)experts, a.lanes = lanes_of(width, type);
  const int64_t per = kRowThreads / a.lanes, blocks = (tokens + per - 1) / per;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define LAUNCH(T, W, DY, DW) \
  hipLaunchKernelGGL((expert_combine_grad_kernel<T, W, DY, DW>), dim3(workgroups(blocks) + kZeroBlocks), dim3(kRowThreads), 0, s, a, blocks)
#define CALL(T, W)                                    \
  if (!dy) { LAUNCH(T, W, false, true); }             \
  else if (!dweights) { LAUNCH(T, W, true, false); }  \
  else { LAUNCH(T, W, true, true); }
  MPS_BY_TYPE(type, a.lanes == kRowThreads, CALL);
#undef CALL
#undef LAUNCH
  MPS_HIP_CHECK(hipGetLastError());
  return MPS_OK;
}

}  // extern "C"
