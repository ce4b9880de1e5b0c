// Products of few rows, which are bound by the weights' bytes: a workgroup takes 16 * FN weight rows
// and 8 * XL rows of x, and its waves take k in turn, 16 blocks (512 elements) at a time.
//
// A wave works alone until the end: it streams its pieces of x and of the weights from memory to
// a ring of S stages in its own part of LDS, without registers and without barriers, waits for
// the oldest stage by the count of loads since, and multiplies it. At the end the waves' sums are
// added up in wave order, so results do not depend on timing.
//
// A stage is 128 bytes of every row of x (64 elements of 16 bits, or 256 codes), in pieces of 16
// bytes, piece p of row r at place p ^ (r / 2 % 8), and the weights of the same k: 32 bytes a row, or
// 128 beside MXFP4 x (their two pieces at p ^ (r / 8 % 2), their eight as x's). In a lane 16 g + r of a 16-row fragment, MXFP4 takes pieces 2 g and 2 g + 1
// of row r, and 16-bit x piece g of one block of k after the other.
//
// FP16 x meets the codes' values in FP16, without their scale, which could leave FP16's range;
// the products of a block are summed by themselves and added with the scale in FP32, exactly as
// if it had been in the weight. (BF16 holds the scaled weight. FP16 as a sum of two BF16 took
// twice the matrix instructions and 32 conversions a fragment: 31.7 us for 37 rows of 5000 x 3001.)
#include "mxfp4_product.h"

namespace mps {
namespace {

template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int XT, int XL, int FN, int W, int S>
struct Rows {
  static constexpr bool k4 = XT == MPS_TYPE_MXFP4;
  static constexpr int kRows = 8 * XL, kFT = XL < 2 ? 1 : XL / 2;  // rows of x; 16-row fragments
  static constexpr int kBN = 16 * FN, kWPieces = k4 ? 8 : 2, kWL = kBN * kWPieces / 64;
  static constexpr int kSteps = k4 ? 2 : 8;  // steps a period of 16 blocks
  static constexpr int kXBytes = kFT * 16 * 128, kWBytes = kWL * 1024, kStage = kXBytes + kWBytes;
  static constexpr int kScaleRows = (k4 ? kRows : 0) + kBN, kSL = (kScaleRows + 63) / 64;
  static constexpr int kWave = S * kStage + kSL * 1024;  // LDS bytes of a wave
  static constexpr int kSums = W * kFT * FN * 1024;
  static constexpr int kLds = W * kWave > kSums ? W * kWave : kSums;
  static_assert(kBN * kWPieces % 64 == 0 && kLds <= 160 * 1024 && (S - 1) * (XL + kWL) < 64, "");
};

template <int XT, int XL, int FN, int W, int S>
__global__ __launch_bounds__(W * 64) void mxfp4_rows_kernel(ProductArgs a) {
  typedef Rows<XT, XL, FN, W, S> R;
  constexpr bool k4 = R::k4;
  constexpr int kFT = R::kFT;
  __shared__ __attribute__((aligned(16))) uint8_t lds[R::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  Tile tile = {0, (int32_t)blockIdx.y * R::kRows, 0};
  tile.end = min(a.rows, tile.first + R::kRows);
  if (a.offsets) tile = find_tile(a.offsets, a.experts, a.rows, R::kRows, blockIdx.y);
  if (tile.expert < 0) return;
  const bool none = tile.expert >= max(a.experts, 1);  // rows of no expert
  const int32_t n0 = blockIdx.x * R::kBN, blocks = a.row_blocks;

  uint8_t *const mine = lds + wave * R::kWave, *const ss = mine + S * R::kStage;
  f32x4 acc[kFT][FN] = {};
  const int32_t periods = none ? 0 : (blocks + 15) / 16;
  if (wave < periods) {
    const int32_t items = ((periods - wave + W - 1) / W) * R::kSteps;
    // Where this lane's pieces come from; rows past the tile's end or the weight's are the last ones.
    const int64_t x_row_bytes = k4 ? (int64_t)blocks * 16 : a.x_stride * 2;
    const int32_t x_piece = (lane % 8) ^ (lane / 16), x_pieces = k4 ? blocks : a.k / 8;
    const uint8_t *x_from[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      int32_t from = min(tile.first + 8 * i + lane / 8, tile.end - 1);
      if (!k4 && a.gather) from = min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1);
      x_from[i] = static_cast<const uint8_t *>(a.x) + from * x_row_bytes;
    }
    const int64_t w_first = (int64_t)tile.expert * a.n + n0;
    const uint8_t *const w_base = a.w + w_first * blocks * 16;
    const uint32_t w_row_bytes = (uint32_t)blocks * 16, w_last = (uint32_t)min(R::kBN - 1, a.n - 1 - n0) * w_row_bytes;
    const int wrow = lane / R::kWPieces;
    const int32_t w_piece = k4 ? (lane % 8) ^ (wrow >> 1) : (lane % 2) ^ (wrow >> 3 & 1);
    const uint8_t *s_from[R::kSL];
#pragma unroll
    for (int i = 0; i < R::kSL; ++i) {
      const int at = i * 64 + lane, row = k4 ? at - R::kRows : at;
      if (k4 && row < 0)
        s_from[i] = a.x_scales + (int64_t)min(tile.first + at, tile.end - 1) * blocks;
      else
        s_from[i] = a.w_scales + (w_first + min(min(row, R::kBN - 1), a.n - 1 - n0)) * blocks;
    }

    auto period_of = [&](int32_t item) { return wave + W * (item / R::kSteps); };
    auto fetch = [&](int32_t item, int slot) {
      const int32_t step = period_of(item) * R::kSteps + item % R::kSteps;
      uint8_t *const to = mine + slot * R::kStage;
      // Eight rows a load: rows of odd loads have the other half of the places' keys.
      const int32_t x_at[2] = {min(step * 8 + x_piece, x_pieces - 1) * 16, min(step * 8 + (x_piece ^ 4), x_pieces - 1) * 16};
#pragma unroll
      for (int i = 0; i < XL; ++i) copy16(x_from[i] + x_at[i & 1], to + i * 1024);
      const uint32_t w_at[2] = {(uint32_t)min(step * R::kWPieces + w_piece, blocks - 1) * 16,
                                (uint32_t)min(step * R::kWPieces + (w_piece ^ 4), blocks - 1) * 16};
#pragma unroll
      for (int i = 0; i < R::kWL; ++i)
        copy16(w_base + (min((uint32_t)(wrow + i * (64 / R::kWPieces)) * w_row_bytes, w_last) + w_at[k4 ? i & 1 : 0]),
               to + R::kXBytes + i * 1024);
    };
    u32x4 scales[R::kSL];
    auto get_scales = [&](int32_t period) {
#pragma unroll
      for (int i = 0; i < R::kSL; ++i) scales[i] = load_scales(s_from[i], 16 * period, blocks);
    };

    get_scales(wave);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < items) fetch(i, i);
    int slot = 0;
    for (int32_t item = 0; item < items; ++item) {
      const int32_t in = item % R::kSteps;
      if (in == 0) {  // the lane's rows' 16 scale bytes, at its place; LDS keeps a wave's order
#pragma unroll
        for (int i = 0; i < R::kSL; ++i) 
          *reinterpret_cast<u32x4 *>(ss + (i * 64 + lane) * 16) = move_scales(scales[i], 16 * period_of(item), blocks);
        if (item + R::kSteps < items) get_scales(period_of(item) + W);
      }
      if (item + S - 1 < items) {
        fetch(item + S - 1, slot == 0 ? S - 1 : slot - 1);
        wait_loads<(S - 1) * (XL + R::kWL)>();
      } else {
        wait_loads<0>();
      }
      const uint8_t *const xl = mine + slot * R::kStage, *const wl = xl + R::kXBytes;
      if constexpr (k4) {
        uint32_t sx[kFT], sw[FN];
#pragma unroll
        for (int t = 0; t < kFT; ++t)
          sx[t] = *reinterpret_cast<const uint16_t *>(ss + (t * 16 + r) % R::kRows * 16 + in * 8 + g * 2);
#pragma unroll
        for (int n = 0; n < FN; ++n)
          sw[n] = *reinterpret_cast<const uint16_t *>(ss + (R::kRows + n * 16 + r) * 16 + in * 8 + g * 2);
        auto half = [&](auto jc) {
          constexpr int j = decltype(jc)::value;
          const int at = ((2 * g + j) ^ (r >> 1)) * 16;
          i32x4 fw[FN];
#pragma unroll
          for (int n = 0; n < FN; ++n) fw[n] = *reinterpret_cast<const i32x4 *>(wl + (n * 16 + r) * 128 + at);
#pragma unroll
          for (int t = 0; t < kFT; ++t) {
            const i32x4 fx = *reinterpret_cast<const i32x4 *>(xl + (t * 16 + r) % R::kRows * 128 + at);
#pragma unroll
            for (int n = 0; n < FN; ++n) {
              const i32x8 wb = {fw[n][0], fw[n][1], fw[n][2], fw[n][3], 0, 0, 0, 0}, xa = {fx[0], fx[1], fx[2], fx[3], 0, 0, 0, 0};
              acc[t][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, wb, acc[t][n], 4, 4, j, sx[t], j, sw[n]);
            }
          }
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
      } else {
        u32x4 fx[kFT][2];
        uint32_t fw[FN][2], bytes[FN];
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          bytes[n] = *reinterpret_cast<const uint16_t *>(ss + (n * 16 + r) * 16 + in * 2);
#pragma unroll
          for (int j = 0; j < 2; ++j) fw[n][j] = *reinterpret_cast<const uint32_t *>(wl + (n * 16 + r) * 32 + (j ^ (r >> 3)) * 16 + g * 4);
        }
#pragma unroll
        for (int t = 0; t < kFT; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            fx[t][j] = *reinterpret_cast<const u32x4 *>(xl + (t * 16 + r) % R::kRows * 128 + ((4 * j + g) ^ (r >> 1)) * 16);
        __builtin_amdgcn_sched_barrier(0);
        // Pieces past the end of x's rows hold other elements: they are taken as zeros.
        const int32_t left = a.k / 8 - (period_of(item) * R::kSteps + in) * 8;
        if (left < 8) {
#pragma unroll
          for (int t = 0; t < kFT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (4 * j + g >= left) fx[t][j] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int n = 0; n < FN; ++n) {
            const uint32_t byte = j ? bytes[n] >> 8 : bytes[n] & 255;
            if constexpr (XT == MPS_TYPE_F16) {
              const f16x8 w = widen_f16(fw[n][j]);
              const float scale = mx_scale_value(byte);
#pragma unroll
              for (int t = 0; t < kFT; ++t) {
                const f32x4 part = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fx[t][j]), w, f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][n][i] = __builtin_fmaf(scale, part[i], acc[t][n][i]);
              }
            } else {
              const bf16x8 w = widen(fw[n][j], mx_scale(byte));
#pragma unroll
              for (int t = 0; t < kFT; ++t)
                acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fx[t][j]), w, acc[t][n], 0, 0, 0);
            }
          }
      }
      slot = slot == S - 1 ? 0 : slot + 1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read: the next loads may take its place
    }
  }

  __syncthreads();
  float *const sums = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int t = 0; t < kFT; ++t)
#pragma unroll
    for (int n = 0; n < FN; ++n) *reinterpret_cast<f32x4 *>(sums + ((wave * kFT + t) * FN + n) * 256 + lane * 4) = acc[t][n];
  __syncthreads();
  // In fragment (t, n) lane 16 g + r has rows 16 t + 4 g .. + 3 of column 16 n + r; the waves share
  // the fragments, a lane now taking four columns of row 16 t + lane / 4.
  const bool quads = a.n % 4 == 0 && aligned16(a.out);
  for (int f = wave; f < kFT * FN; f += W) {
    const int in_row = lane / 4, in_col = lane % 4 * 4;
    const int32_t row = tile.first + f / FN * 16 + in_row, col = n0 + f % FN * 16 + in_col;
    if (f / FN * 16 + in_row >= R::kRows || row >= tile.end || col >= a.n) continue;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float *const from = sums + (w * kFT * FN + f) * 256 + (in_row / 4 * 16 + in_col) * 4 + in_row % 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += from[4 * j];
    }
    if (a.bias && !none) v += load_bias4(a, tile.expert, col);
    store4(a, row, col, v, quads);
  }
}

template <int XT, int XL, int FN, int W, int S>
void launch(const ProductArgs &a, hipStream_t stream) {
  typedef Rows<XT, XL, FN, W, S> R;
  const dim3 grid((unsigned)((a.n + R::kBN - 1) / R::kBN), (unsigned)product_tiles(a, R::kRows));
  hipLaunchKernelGGL((mxfp4_rows_kernel<XT, XL, FN, W, S>), grid, dim3(W * 64), 0, stream, a);
}

// Rows of x a workgroup: enough for one pass over the weights, or (experts, whose rows are spread
// unevenly) twice their share.
template <int XT>
void launch_type(const ProductArgs &a, hipStream_t stream) {
  const int64_t rows = a.offsets ? 2 * (((int64_t)a.rows + a.experts - 1) / a.experts) : a.rows;
  if constexpr (XT == MPS_TYPE_MXFP4) {
    if (rows <= 8)
      launch<XT, 1, 2, 4, 4>(a, stream);
    else if (rows <= 16)
      launch<XT, 2, 2, 4, 3>(a, stream);
    else if (rows <= 32)
      launch<XT, 4, 2, 4, 4>(a, stream);
    else
      launch<XT, 8, 2, 4, 3>(a, stream);
  } else {
    if (rows <= 8)
      launch<XT, 1, 2, 8, 3>(a, stream);
    else if (rows <= 16)
      launch<XT, 2, 2, 8, 3>(a, stream);
    else if (rows <= 32)
      launch<XT, 4, 2, 8, 3>(a, stream);
    else
      launch<XT, 8, 2, 4, 3>(a, stream);
  }
}

}  // namespace

void launch_rows(const ProductArgs &a, int32_t x_type, hipStream_t stream) {
  if (x_type == MPS_TYPE_MXFP4)
    launch_type<MPS_TYPE_MXFP4>(a, stream);
  else if (x_type == MPS_TYPE_BF16)
    launch_type<MPS_TYPE_BF16>(a, stream);
  else
    launch_type<MPS_TYPE_F16>(a, stream);
}

}  // namespace mps
