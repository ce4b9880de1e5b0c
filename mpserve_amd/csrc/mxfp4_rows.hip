// Products of few rows, which are bound by the weights' bytes: a workgroup takes 16 * FN weight rows
// and 8 * XL rows of x, and its waves take k in turn, 16 blocks (512 elements) at a time.
//
// A wave works alone until the end: it streams its pieces of x and of the weights from memory to
// a ring of S stages in its own part of LDS, without registers and without barriers, waits for
// the oldest stage by the count of loads since, and multiplies it. At the end the waves' sums are
// added up in wave order, so results do not depend on timing.
//
// A stage is U cache lines of every row of x (64 U elements of 16 bits, or 256 codes, U = 1) and the
// weights of the same k, 32 U bytes a row, or 128 beside MXFP4 x: the more, the fewer instructions and
// waits a byte (one token through 4096 x 14336: U = 1 9.1 us, U = 4 7.5), the fewer, the more rows
// of x fit. Pieces of 16 bytes lie in rows as in mxfp4_tile.hip: piece p of row r of x at place
// p ^ (r / 2 % 8), of P pieces of a weight row at p ^ (r / (16 / P)).
// In a lane 16 g + r of a 16-row fragment, MXFP4 takes pieces 2 g and 2 g + 1 of row r, and 16-bit x
// piece g of one block of k after the other.
//
// FP16 x meets the codes' values in FP16, without their scale, which could leave FP16's range;
// the products of a block are summed by themselves and added with the scale in FP32, exactly as
// if it had been in the weight. (BF16 holds the scaled weight; for scales near 2^127 a quarter of it. FP16 as a sum of two BF16 took
// twice the matrix instructions and 32 conversions a fragment.)
#include "mxfp4_product.h"

namespace mps {
namespace {

template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int XT, int XL, int FN, int U, int W, int S>
struct Rows {
  static constexpr bool k4 = XT == MPS_TYPE_MXFP4;
  static constexpr int kRows = 8 * XL, kFT = XL < 2 ? 1 : XL / 2;  // rows of x; 16-row fragments
  static constexpr int kBN = 16 * FN, kWPieces = k4 ? 8 : 2 * U, kWL = kBN * kWPieces / 64;
  static constexpr int kSteps = k4 ? 2 : 8 / U;  // stages a period of 16 blocks
  static constexpr int kLoads = XL * U + kWL;    // a stage
  static constexpr int kLine = kRows * 128, kXBytes = U * kLine, kWBytes = kWL * 1024, kStage = kXBytes + kWBytes;
  static constexpr int kScaleRows = (k4 ? kRows : 0) + kBN, kSL = (kScaleRows + 63) / 64;
  static constexpr int kWave = S * kStage + kSL * 1024;  // LDS bytes of a wave
  static constexpr int kSums = W * kFT * FN * 1024;
  static constexpr int kLds = W * kWave > kSums ? W * kWave : kSums;
  static_assert(kBN * kWPieces % 64 == 0 && kLds <= 160 * 1024 && (S - 1) * kLoads < 64 && (!k4 || U == 1), "");
};

template <int XT, int XL, int FN, int U, int W, int S>
__global__ __launch_bounds__(W * 64) void mxfp4_rows_kernel(ProductArgs a) {
  typedef Rows<XT, XL, FN, U, W, S> R;
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
    // A load has 64 / kWPieces weight rows; with 8 pieces a row, odd loads have the other half of the keys.
    const int wrow = lane / R::kWPieces;
    const int32_t w_piece = (lane % R::kWPieces) ^ (wrow % 16 / (16 / R::kWPieces));
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
#pragma unroll
      for (int u = 0; u < U; ++u) {  // eight rows a load, so odd loads have the other half of the keys
        const int32_t x_at[2] = {min((step * U + u) * 8 + x_piece, x_pieces - 1) * 16, min((step * U + u) * 8 + (x_piece ^ 4), x_pieces - 1) * 16};
#pragma unroll
        for (int i = 0; i < XL; ++i) copy16(x_from[i] + x_at[i & 1], to + u * R::kLine + i * 1024);
      }
      const uint32_t w_at[2] = {(uint32_t)min(step * R::kWPieces + w_piece, blocks - 1) * 16,
                                (uint32_t)min(step * R::kWPieces + (w_piece ^ 4), blocks - 1) * 16};
#pragma unroll
      for (int i = 0; i < R::kWL; ++i)
        copy16(w_base + (min((uint32_t)(wrow + i * (64 / R::kWPieces)) * w_row_bytes, w_last) + w_at[R::kWPieces == 8 ? i & 1 : 0]),
               to + R::kXBytes + i * 1024);
    };
    u32x4 scales[R::kSL];
    auto get_scales = [&](int32_t period) {
#pragma unroll
      for (int i = 0; i < R::kSL; ++i) scales[i] = load_scales(s_from[i], 16 * period, blocks);
    };

    uint32_t large = 0;  // BF16: whether this lane has met a large scale
    auto put_scales = [&](int32_t period) {  // the lane's rows' 16 scale bytes, at its place; LDS keeps a wave's order
#pragma unroll
      for (int i = 0; i < R::kSL; ++i) {
        const u32x4 moved = move_scales(scales[i], 16 * period, blocks);
        *reinterpret_cast<u32x4 *>(ss + (i * 64 + lane) * 16) = moved;
        if constexpr (XT == MPS_TYPE_BF16) large |= large_scales(moved);
      }
    };
    auto multiply = [&](int32_t item, int slot, auto quartered) {
      const int32_t in = item % R::kSteps;
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
        u32x4 fx[U][kFT][2];
        uint32_t fw[U][FN][2];
        uint64_t bytes[FN];
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          const uint8_t *const at = ss + (n * 16 + r) * 16 + in * 2 * U;
          bytes[n] = U == 4 ? *reinterpret_cast<const uint64_t *>(at) : U == 2 ? *reinterpret_cast<const uint32_t *>(at) : *reinterpret_cast<const uint16_t *>(at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int n = 0; n < FN; ++n)
              fw[u][n][j] = *reinterpret_cast<const uint32_t *>(wl + (n * 16 + r) * R::kWPieces * 16 + ((2 * u + j) ^ (r / (16 / R::kWPieces))) * 16 + g * 4);
#pragma unroll
            for (int t = 0; t < kFT; ++t)
              fx[u][t][j] = *reinterpret_cast<const u32x4 *>(xl + u * R::kLine + (t * 16 + r) % R::kRows * 128 + ((4 * j + g) ^ (r >> 1)) * 16);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        // Pieces past the end of x's rows hold other elements: they are taken as zeros.
        const int32_t left = a.k / 8 - (period_of(item) * R::kSteps + in) * 8 * U;
        if (left < 8 * U) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < kFT; ++t)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (8 * u + 4 * j + g >= left) fx[u][t][j] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = 0; n < FN; ++n) {
              const uint32_t byte = (uint32_t)(bytes[n] >> (16 * u + 8 * j)) & 255;
              if constexpr (XT == MPS_TYPE_F16) {
                const f16x8 w = widen_f16(fw[u][n][j]);
                const float scale = mx_scale_value(byte);
#pragma unroll
                for (int t = 0; t < kFT; ++t) {
                  const f32x4 part = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fx[u][t][j]), w, f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[t][n][i] = __builtin_fmaf(scale, part[i], acc[t][n][i]);
                }
              } else {
                constexpr bool quarters = decltype(quartered)::value;
                const bf16x8 w = quarters ? widen_quarter(fw[u][n][j], byte) : widen(fw[u][n][j], mx_scale(byte));
#pragma unroll
                for (int i = 0; i < (quarters ? 4 : 1); ++i)
#pragma unroll
                  for (int t = 0; t < kFT; ++t)
                    acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fx[u][t][j]), w, acc[t][n], 0, 0, 0);
              }
            }
      }
    };

    get_scales(wave);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < items) fetch(i, i);
    int slot = 0;
    for (int32_t item = 0; item < items; ++item) {
      if (item % R::kSteps == 0) {
        put_scales(period_of(item));
        if (item + R::kSteps < items) get_scales(period_of(item) + W);
      }
      if (item + S - 1 < items) {
        fetch(item + S - 1, slot == 0 ? S - 1 : slot - 1);
        wait_loads<(S - 1) * R::kLoads>();
      } else {
        wait_loads<0>();
      }
      multiply(item, slot, std::false_type{});
      slot = slot == S - 1 ? 0 : slot + 1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read: the next loads may take its place
    }
    if constexpr (XT == MPS_TYPE_BF16) {
      if (__builtin_expect(__any(large & kLargeScale), 0)) {  // a weight may have overflowed: all again, one at a time
#pragma unroll
        for (int t = 0; t < kFT; ++t)
#pragma unroll
          for (int n = 0; n < FN; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll 1
        for (int32_t item = 0; item < items; ++item) {
          if (item % R::kSteps == 0) {
            get_scales(period_of(item));
            put_scales(period_of(item));
          }
          fetch(item, 0);
          wait_loads<0>();
          multiply(item, 0, std::true_type{});
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
      }
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
    store4(a, row, col, v);
  }
}

template <int XT, int XL, int FN, int U, int W, int S>
void launch(const ProductArgs &a, hipStream_t stream) {
  typedef Rows<XT, XL, FN, U, W, S> R;
  const dim3 grid((unsigned)((a.n + R::kBN - 1) / R::kBN), (unsigned)product_tiles(a, R::kRows));
  hipLaunchKernelGGL((mxfp4_rows_kernel<XT, XL, FN, U, W, S>), grid, dim3(W * 64), 0, stream, a);
}

// The shapes of a workgroup: 8 XL rows of x, 16 FN weight rows, U lines a stage, W waves, S stages. `resident`
// of them fit a CU, and one takes `us` for each period of k (512 elements) that a wave has, as
// measured with CUs full and half full (1 x 4096 x 14336, 16 x 4096 x 4096, 32 x 14336 x 4096, 64 x 8192 x
// 8192, 64 x 4096 x 28672). More rows a workgroup spare reads of the weights, fewer fill more CUs, and more
// waves share a long k: 64 x 8192 x 8192 in BF16 takes 17.0 us with XL 4, FN 4 and 41 with XL 1, FN 2, which
// takes 6.7 to 7.5 for 1 x 4096 x 14336 where the first takes 9.3 to 10.5.
struct Choice {
  int32_t rows, cols, waves, resident;
  float us, start;
};
// Workgroups past the first on a CU cost `start` each beside (1200 to 8000 rows of 60 and 64 experts; 1200 rows spread
// evenly over 64 experts, 4096 x 2048, in BF16: 97 us with XL 4, FN 4, and 82 to 88 in tiles of 128 x 256, which are taken).
constexpr Choice kChoicesBf16[] = {{8, 32, 4, 2, 2.5f, 1.3f}, {8, 32, 8, 1, 2.7f, 1.9f}, {16, 32, 8, 1, 3.2f, 2.5f}, {16, 64, 4, 1, 2.8f, 2.1f},
                                   {32, 32, 6, 1, 3.2f, 1.2f}, {32, 64, 4, 1, 3.8f, 2.7f}, {64, 64, 4, 1, 6.2f, 3.5f}};
// FP16's scaled sums cost more, the more rows (64 x 2048 x 8192 with XL 4, FN 4 7.2 us in BF16, 9.7 in FP16).
constexpr Choice kChoicesF16[] = {{8, 32, 4, 2, 3.1f, 1.3f}, {8, 32, 8, 1, 3.4f, 1.9f}, {16, 32, 8, 1, 3.8f, 2.5f}, {16, 64, 4, 1, 3.6f, 2.1f},
                                  {32, 32, 6, 1, 3.8f, 1.2f}, {32, 64, 4, 1, 5.6f, 2.7f}, {64, 64, 4, 1, 9.6f, 3.5f}};
constexpr Choice kChoices4[] = {{8, 32, 4, 2, 1.9f, 0}, {8, 32, 8, 1, 2.2f, 0}, {16, 32, 4, 2, 1.9f, 0}, {16, 32, 8, 1, 2.3f, 0},
                                {32, 64, 4, 1, 2.5f, 0}, {64, 32, 6, 1, 2.7f, 0}};

template <int N>
Prediction least(const ProductArgs &a, const Choice (&choices)[N], int32_t cus) {
  Prediction best = {-1, 0};
  const int64_t periods = (a.row_blocks + 15) / 16;
  for (int i = 0; i < N; ++i) {
    const Choice &c = choices[i];
    if (product_tiles(a, c.rows) > 65535 || (double)((a.n + c.cols - 1) / c.cols) * c.waves * 64 > kMostWorkItems) continue;
    const double each = expected_tiles(a, c.rows) * (double)((a.n + c.cols - 1) / c.cols) / ((double)cus * c.resident);
    const double rounds = each <= 1 ? 1.0 : __builtin_ceil(each - 0.01);
    const double us = rounds * (double)((periods + c.waves - 1) / c.waves) * c.us + (each > 1 ? each - 1 : 0) * c.start;
    if (best.choice < 0 || us < best.us) best = {i, us};
  }
  return best;
}

template <int XT>
void launch_type(const ProductArgs &a, int choice, hipStream_t stream) {
  if constexpr (XT == MPS_TYPE_MXFP4) {
    switch (choice) {
      case 0: return launch<XT, 1, 2, 1, 4, 3>(a, stream);
      case 1: return launch<XT, 1, 2, 1, 8, 2>(a, stream);
      case 2: return launch<XT, 2, 2, 1, 4, 3>(a, stream);
      case 3: return launch<XT, 2, 2, 1, 8, 2>(a, stream);
      case 4: return launch<XT, 4, 4, 1, 4, 2>(a, stream);
      default: return launch<XT, 8, 2, 1, 6, 2>(a, stream);
    }
  } else {
    switch (choice) {
      case 0: return launch<XT, 1, 2, 4, 4, 2>(a, stream);
      case 1: return launch<XT, 1, 2, 4, 8, 2>(a, stream);
      case 2: return launch<XT, 2, 2, 2, 8, 2>(a, stream);
      case 3: return launch<XT, 2, 4, 4, 4, 2>(a, stream);
      case 4: return launch<XT, 4, 2, 2, 6, 2>(a, stream);
      case 5: return launch<XT, 4, 4, 2, 4, 3>(a, stream);
      default: return launch<XT, 8, 4, 1, 4, 3>(a, stream);
    }
  }
}

}  // namespace

Prediction predict_rows(const ProductArgs &a, int32_t x_type, int32_t cus) {
  if (x_type == MPS_TYPE_MXFP4) return least(a, kChoices4, cus);
  return x_type == MPS_TYPE_BF16 ? least(a, kChoicesBf16, cus) : least(a, kChoicesF16, cus);
}

void launch_rows(const ProductArgs &a, int32_t x_type, int choice, hipStream_t stream) {
  if (x_type == MPS_TYPE_MXFP4)
    launch_type<MPS_TYPE_MXFP4>(a, choice, stream);
  else if (x_type == MPS_TYPE_BF16)
    launch_type<MPS_TYPE_BF16>(a, choice, stream);
  else
    launch_type<MPS_TYPE_F16>(a, choice, stream);
}

}  // namespace mps
