// Products of many rows: tiles of BT rows of x times BN weight rows, with both operands' pieces of
// k staged in LDS.
//
// A step covers 128 bytes of every row of x: 64 BF16 elements or 256 codes. The weights of a step
// are 32 bytes a row beside BF16 x (written out as BF16 in registers, after LDS) and 128 beside
// MXFP4 x, which the matrix cores multiply as it is. Pieces of 16 bytes go from memory to LDS
// without passing through registers; piece p of row r lies at place p ^ (r / 2 % 8) of its row's
// eight, or p ^ (r / 8 % 2) of two, so that sixteen lanes reading one piece of sixteen rows meet
// all 64 banks once (with r % 8, which serves eight lanes, half of all LDS cycles were conflicts). A lane of a
// 32-row fragment reads four neighbouring pieces (one half of the row each for lanes 0-31 and
// 32-63): k is summed in this order for both operands, so that a lane's four blocks have
// neighbouring scale bytes.
#include "mxfp4_product.h"

namespace mps {
namespace {

template <int J>
__device__ inline f32x16 multiply4(i32x4 w, uint32_t ws, i32x4 x, uint32_t xs, f32x16 c) {
  const i32x8 a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, J, ws, J, xs);
}

template <int XT, int BT, int BN, int WT, int WN>
struct Shape {
  static constexpr bool k4 = XT == MPS_TYPE_MXFP4;
  static constexpr int kThreads = WT * WN * 64;
  static constexpr int kXPieces = 8, kWPieces = k4 ? 8 : 2;      // a row and step
  static constexpr int kSteps = k4 ? 2 : 8;                      // steps that 16 scale bytes last
  static constexpr int kScaleRows = k4 ? BT + BN : BN;           // x's rows, then the weight's
  static constexpr int kXLoads = BT * kXPieces / kThreads;       // pieces a work-item and step
  static constexpr int kWLoads = (BN * kWPieces + kThreads - 1) / kThreads;
  static constexpr int kFT = BT / WT / 32, kFN = BN / WN / 32;   // 32 x 32 fragments of a wave
  static_assert(BT * kXPieces % kThreads == 0 && kScaleRows <= kThreads, "");
};

template <int XT, int BT, int BN, int WT, int WN>
__global__ __launch_bounds__(WT *WN * 64) void mxfp4_tile_kernel(ProductArgs a, int32_t tiles_t, int32_t tiles_n) {
  typedef Shape<XT, BT, BN, WT, WN> S;
  constexpr bool k4 = S::k4;
  constexpr int kXBytes = BT * 128, kWBytes = BN * S::kWPieces * 16, kSBytes = S::kScaleRows * 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * (kXBytes + kWBytes + kSBytes)];
  uint8_t *const xs = lds, *const ws = lds + 2 * kXBytes, *const ss = lds + 2 * (kXBytes + kWBytes);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, g = lane >> 5;
  const int wt = wave / WN, wn = wave % WN;

  // Workgroups go to the 8 XCDs in turn. Each XCD takes a stretch of the tiles, in which
  // groups of 8 tiles of rows run through the weight's tiles together, so that its L2 serves both.
  const uint32_t total = (uint32_t)tiles_t * (uint32_t)tiles_n;
  const uint32_t per = (total + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || id >= total) return;
  const uint32_t group = id / (8u * tiles_n), in_group = id - group * 8u * tiles_n;
  const uint32_t group_t = min(8u, (uint32_t)tiles_t - group * 8);
  const int32_t tile_t = group * 8 + in_group % group_t, n0 = (in_group / group_t) * BN;

  Tile tile = {0, tile_t * BT, min(a.rows, tile_t * BT + BT)};
  if (a.offsets) tile = find_tile(a.offsets, a.experts, a.rows, BT, tile_t);
  if (tile.expert < 0) return;
  const bool none = tile.expert >= max(a.experts, 1);  // rows of no expert
  const int32_t blocks = a.row_blocks;
  const int32_t steps = none ? 0 : (blocks + (k4 ? 7 : 1)) / (k4 ? 8 : 2);

  // Where this work-item's pieces come from. Rows past the tile's end or the weight's are read
  // from the last one; what they give is not stored.
  const int64_t x_row_bytes = k4 ? (int64_t)blocks * 16 : a.x_stride * 2;
  const int64_t w_row_bytes = (int64_t)blocks * 16;
  // MXFP4 x and the weights lie row by row, so an offset from the tile's first row, cut at the
  // last, finds every piece; gathered rows need an address each.
  const int xrow = tid / 8, wrow = tid / S::kWPieces;
  const int32_t x_piece = (tid % 8) ^ (xrow >> 1 & 7), w_piece = k4 ? (tid % 8) ^ (wrow >> 1 & 7) : (tid % 2) ^ (wrow >> 3 & 1);
  const int64_t w_first = (int64_t)(none ? 0 : tile.expert) * a.n + n0;
  const uint8_t *const w_base = a.w + w_first * w_row_bytes;
  const uint32_t w_last = (uint32_t)min(BN - 1, a.n - 1 - n0) * (uint32_t)w_row_bytes;
  const uint32_t x_last = (uint32_t)(tile.end - 1 - tile.first) * (uint32_t)x_row_bytes;
  const uint8_t *const x_base = static_cast<const uint8_t *>(a.x) + tile.first * x_row_bytes;
  const uint8_t *x_from[k4 ? 1 : S::kXLoads];
  if constexpr (!k4) {
#pragma unroll
    for (int i = 0; i < S::kXLoads; ++i) {
      int32_t from = min(tile.first + xrow + i * (S::kThreads / 8), tile.end - 1);
      if (a.gather) from = min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1);
      x_from[i] = static_cast<const uint8_t *>(a.x) + from * x_row_bytes + x_piece * 16;
    }
  }
  const uint8_t *s_from = nullptr;
  if (tid < S::kScaleRows) {
    const int row = k4 ? tid - BT : tid;
    if (k4 && row < 0)
      s_from = a.x_scales + (int64_t)min(tile.first + tid, tile.end - 1) * blocks;
    else
      s_from = a.w_scales + (w_first + min(row, a.n - 1 - n0)) * blocks;
  }

  auto fetch = [&](int32_t step, int buffer) {
    if constexpr (k4) {
      const uint32_t at = (uint32_t)min(step * 8 + x_piece, blocks - 1) * 16;
#pragma unroll
      for (int i = 0; i < S::kXLoads; ++i)
        copy16(x_base + (min((uint32_t)(xrow + i * (S::kThreads / 8)) * (uint32_t)x_row_bytes, x_last) + at),
               xs + buffer * kXBytes + (i * S::kThreads + wave * 64) * 16);
    } else {
      const int64_t at = (int64_t)step * 128;
#pragma unroll
      for (int i = 0; i < S::kXLoads; ++i)
        copy16(x_from[i] + at, xs + buffer * kXBytes + (i * S::kThreads + wave * 64) * 16);
    }
    const uint32_t at = (uint32_t)min(step * S::kWPieces + w_piece, blocks - 1) * 16;
#pragma unroll
    for (int i = 0; i < S::kWLoads; ++i)
      if (BN * S::kWPieces % S::kThreads == 0 || i * S::kThreads + wave * 64 < BN * S::kWPieces)
        copy16(w_base + (min((uint32_t)(wrow + i * (S::kThreads / S::kWPieces)) * (uint32_t)w_row_bytes, w_last) + at),
               ws + buffer * kWBytes + (i * S::kThreads + wave * 64) * 16);
  };
  // The scales of a period (16 blocks) are fetched a period ahead.
  auto put_scales = [&](u32x4 v, int buffer) {
    if (s_from) *reinterpret_cast<u32x4 *>(ss + buffer * kSBytes + tid * 16) = v;
  };

  f32x16 acc[S::kFT][S::kFN] = {};
  // Keeps the products of a step inside it: the compiler would read all fragments of a step first.
  auto pin = [&]() {
#pragma unroll
    for (int t = 0; t < S::kFT; ++t)
#pragma unroll
      for (int n = 0; n < S::kFN; ++n) asm volatile("" : "+v"(acc[t][n]));
  };
  const int32_t periods = (blocks + 15) / 16;
  if (steps > 0) {
    if (s_from) put_scales(move_scales(load_scales(s_from, 0, blocks), 0, blocks), 0);
    fetch(0, 0);
  }
  if constexpr (k4) {
    auto compute = [&](const uint8_t *xl, const uint8_t *wl, const uint8_t *sl) {
      uint32_t sx[S::kFT], sw[S::kFN];
#pragma unroll
      for (int t = 0; t < S::kFT; ++t)
        sx[t] = *reinterpret_cast<const uint32_t *>(sl + (wt * S::kFT * 32 + t * 32 + r) * 16 + g * 4);
#pragma unroll
      for (int n = 0; n < S::kFN; ++n)
        sw[n] = *reinterpret_cast<const uint32_t *>(sl + (BT + wn * S::kFN * 32 + n * 32 + r) * 16 + g * 4);
      // The fragments of a quarter are read while the one before is multiplied.
      i32x4 fx[2][S::kFT], fw[2][S::kFN];
      auto read = [&](int j) {
        const int at = ((4 * g + j) ^ (r >> 1 & 7)) * 16;
#pragma unroll
        for (int n = 0; n < S::kFN; ++n)
          fw[j & 1][n] = *reinterpret_cast<const i32x4 *>(wl + (wn * S::kFN * 32 + n * 32 + r) * 128 + at);
#pragma unroll
        for (int t = 0; t < S::kFT; ++t)
          fx[j & 1][t] = *reinterpret_cast<const i32x4 *>(xl + (wt * S::kFT * 32 + t * 32 + r) * 128 + at);
      };
      auto multiply = [&](auto jc) {
        constexpr int j = decltype(jc)::value;
#pragma unroll
        for (int t = 0; t < S::kFT; ++t)
#pragma unroll
          for (int n = 0; n < S::kFN; ++n) acc[t][n] = multiply4<j>(fw[j & 1][n], sw[n], fx[j & 1][t], sx[t], acc[t][n]);
      };
      read(0);
      read(1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(std::integral_constant<int, 0>{});
      __builtin_amdgcn_sched_barrier(0);
      read(2);
      __builtin_amdgcn_sched_barrier(0);
      multiply(std::integral_constant<int, 1>{});
      __builtin_amdgcn_sched_barrier(0);
      read(3);
      __builtin_amdgcn_sched_barrier(0);
      multiply(std::integral_constant<int, 2>{});
      multiply(std::integral_constant<int, 3>{});
      pin();
    };
    // Two steps a period; steps past the last block read zero scales and add nothing.
    int sbuf = 0;
    for (int32_t p = 0; p < (none ? 0 : periods); ++p) {
      u32x4 scales = {0, 0, 0, 0};
      __syncthreads();  // this step's pieces have landed, and nobody reads the other buffers any more
      if (p + 1 < periods && s_from) scales = load_scales(s_from, 16 * (p + 1), blocks);
      fetch(2 * p + 1, 1);
      compute(xs, ws, ss + sbuf * kSBytes);
      __syncthreads();
      put_scales(move_scales(scales, 16 * (p + 1), blocks), sbuf ^ 1);
      fetch(2 * p + 2, 0);
      compute(xs + kXBytes, ws + kWBytes, ss + sbuf * kSBytes + 8);
      sbuf ^= 1;
    }
  } else {
    int32_t step = 0;
    int sbuf = 0;
    for (int32_t p = 0; p < (none ? 0 : periods); ++p) {
      u32x4 scales = {0, 0, 0, 0};
      const int32_t last = min(steps - p * S::kSteps, S::kSteps);
      for (int32_t in = 0; in < last; ++in, ++step) {
        const int buffer = step & 1;
        __syncthreads();
        if (in == 0 && s_from && p + 1 < periods) scales = load_scales(s_from, 16 * (p + 1), blocks);
        if (in == last - 1) put_scales(move_scales(scales, 16 * (p + 1), blocks), sbuf ^ 1);
        if (step + 1 < steps) fetch(step + 1, buffer ^ 1);
        const uint8_t *xl = xs + buffer * kXBytes, *wl = ws + buffer * kWBytes, *sl = ss + sbuf * kSBytes + in * 2;
        typedef typename std::conditional<XT == MPS_TYPE_F16, f16x8, bf16x8>::type x8;
        auto read = [&](int piece, x8(&fx)[S::kFT]) {
#pragma unroll
          for (int t = 0; t < S::kFT; ++t)
            fx[t] = *reinterpret_cast<const x8 *>(xl + (wt * S::kFT * 32 + t * 32 + r) * 128 + (piece ^ (r >> 1 & 7)) * 16);
        };
        if constexpr (XT == MPS_TYPE_F16) {
          // Lanes 0-31 have the first half of a block of k, lanes 32-63 the second.
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            x8 fx[2][S::kFT];
            read(4 * b + 2 * g, fx[0]);
            read(4 * b + 2 * g + 1, fx[1]);
#pragma unroll
            for (int n = 0; n < S::kFN; ++n) {
              const int row = wn * S::kFN * 32 + n * 32 + r;
              const uint64_t codes = *reinterpret_cast<const uint64_t *>(wl + row * 32 + (b ^ (r >> 3 & 1)) * 16 + g * 8);
              const float scale = mx_scale_value(sl[row * 16 + b]);
              const f16x8 w0 = widen_f16((uint32_t)codes), w1 = widen_f16((uint32_t)(codes >> 32));
#pragma unroll
              for (int t = 0; t < S::kFT; ++t) {
                f32x16 part = __builtin_amdgcn_mfma_f32_32x32x16_f16(fx[0][t], w0, f32x16{}, 0, 0, 0);
                part = __builtin_amdgcn_mfma_f32_32x32x16_f16(fx[1][t], w1, part, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][n][i] = __builtin_fmaf(scale, part[i], acc[t][n][i]);
              }
            }
          }
        } else {
          // Lanes 0-31 have the step's first block of k, lanes 32-63 the second.
          u32x4 fw[S::kFN];
          float sw[S::kFN];
#pragma unroll
          for (int n = 0; n < S::kFN; ++n) {
            const int row = wn * S::kFN * 32 + n * 32 + r;
            fw[n] = *reinterpret_cast<const u32x4 *>(wl + row * 32 + (g ^ (r >> 3 & 1)) * 16);
            sw[n] = mx_scale(sl[row * 16 + g]);
          }
          x8 fx[2][S::kFT];
          read(4 * g, fx[0]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < 3) read(4 * g + j + 1, fx[(j + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < S::kFN; ++n) {
              const bf16x8 w = widen(fw[n][j], sw[n]);
#pragma unroll
              for (int t = 0; t < S::kFT; ++t)
                acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, fx[j & 1][t], acc[t][n], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        pin();
      }
      sbuf ^= 1;
    }
  }

  // A lane's 16 sums are places 8 i + 4 g .. + 3 of one side of a fragment, at place r of the other: columns
  // of one row, or with FP16 x rows of one column. The wave turns 32 rows at a time round through its own
  // part of LDS, so that stores go along the rows.
  __syncthreads();
  constexpr int kCols = S::kFN * 32, kPitch = kCols + 4, kLanes = kCols / 4;
  static_assert(WT * WN * 32 * kPitch * 4 <= sizeof(lds), "");
  float *mine = reinterpret_cast<float *>(lds) + wave * 32 * kPitch;
  const bool quads = a.n % 4 == 0 && aligned16(a.out);
  const int32_t col = n0 + wn * kCols + lane % kLanes * 4;
  float bias[4] = {0, 0, 0, 0};
  if (a.bias && !none) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < a.n) bias[j] = load_as_float(a.bias, a.bias_type, (int64_t)tile.expert * a.n + col + j);
  }
#pragma unroll
  for (int t = 0; t < S::kFT; ++t) {
#pragma unroll
    for (int n = 0; n < S::kFN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (XT == MPS_TYPE_F16) {
#pragma unroll
          for (int j = 0; j < 4; ++j) mine[(8 * i + 4 * g + j) * kPitch + n * 32 + r] = acc[t][n][4 * i + j];
        } else {
          *reinterpret_cast<f32x4 *>(mine + r * kPitch + n * 32 + 8 * i + 4 * g) =
              f32x4{acc[t][n][4 * i], acc[t][n][4 * i + 1], acc[t][n][4 * i + 2], acc[t][n][4 * i + 3]};
        }
      }
    __builtin_amdgcn_wave_barrier();
    const int32_t first = tile.first + (wt * S::kFT + t) * 32;
    for (int row = lane / kLanes; row < 32; row += 64 / kLanes) {
      f32x4 v = *reinterpret_cast<const f32x4 *>(mine + row * kPitch + lane % kLanes * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += bias[j];
      if (first + row >= tile.end || col >= a.n) continue;
      store4(a, first + row, col, v, quads);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int XT, int BT, int BN, int WT, int WN>
void launch(const ProductArgs &a, hipStream_t stream) {
  const int64_t tt = product_tiles(a, BT), tn = (a.n + BN - 1) / BN;
  const int64_t grid = (tt * tn + 7) / 8 * 8;
  hipLaunchKernelGGL((mxfp4_tile_kernel<XT, BT, BN, WT, WN>), dim3((unsigned)grid), dim3(WT * WN * 64), 0, stream, a,
                     (int32_t)tt, (int32_t)tn);
}

}  // namespace

void launch_tiles(const ProductArgs &a, int32_t x_type, hipStream_t stream) {
  if (x_type == MPS_TYPE_MXFP4)
    launch<MPS_TYPE_MXFP4, 256, 256, 2, 4>(a, stream);
  else if (x_type == MPS_TYPE_BF16)
    launch<MPS_TYPE_BF16, 256, 256, 2, 4>(a, stream);
  else
    launch<MPS_TYPE_F16, 256, 256, 2, 4>(a, stream);
}

}  // namespace mps
