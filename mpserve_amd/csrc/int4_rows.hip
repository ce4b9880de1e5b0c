// Products of few rows, which are bound by the weights' bytes: a workgroup takes 16 FN weight rows and 8 XL rows of
// x, and its waves take k in turn, 16 blocks (512 elements) at a time.
//
// A wave works alone until the end: it streams its pieces of x and of the weights from memory to a ring of S stages in
// its own part of LDS, without registers and without barriers, waits for the oldest stage by the count of loads
// since, and multiplies it. At the end the waves' sums are added up in wave order, so results do not depend on timing.
//
// A stage is U cache lines of every row of x (64 U elements) and the weights of the same k, 32 U bytes a row. Pieces of 16
// bytes lie so that the sixteen lanes that LDS serves in a cycle meet all banks: piece p of row r of x at place p ^ (r / 2 % 8),
// of P pieces of a weight row at p ^ (r / (16 / P)); a single row of x lies as it is, and all lanes read it. In a lane 16 g + r of a 16-row fragment, x takes piece g of one
// block of k after the other.
//
// The matrix cores multiply x by the whole numbers q as they are, and by ones, of which one fragment serves all
// weight rows: sum x (q - z) = sum x q - z sum x, with a group's scale, in FP32. Where that is not finite (x holds an infinity, or its sums pass
// 2^128) a wave makes its sums again from q - z, three times the instructions.
#include "int4_product.h"

namespace mps {
namespace {

template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <bool kFew, int XL, int FN, int U, int W, int S>
struct Rows {
  static constexpr bool kOne = XL == 0;                            // a single row of x, whose lines a load has side by side
  static constexpr int kRows = kOne ? 1 : 8 * XL, kFT = XL < 2 ? 1 : XL / 2;  // rows of x; 16-row fragments
  static constexpr int kBN = 16 * FN, kWPieces = 2 * U, kWL = kBN * kWPieces / 64;
  static constexpr int kSteps = 8 / U;         // stages a period
  static constexpr int kXLoads = kOne ? 1 : XL, kLoads = kOne ? 1 + kWL : XL * U + kWL;  // x's a line; all of a stage
  static constexpr int kLine = kRows * 128, kXBytes = U * kLine, kWBytes = kWL * 1024, kStage = kXBytes + kWBytes;
  static constexpr int kWindow = Window<kFew>::kBytes, kSL = (kBN + 63) / 64;
  static constexpr int kWave = S * kStage + kBN * kWindow;  // LDS bytes of a wave
  static constexpr int kChain = kFew ? (2 * U < 4 ? 2 * U : 4) : 1;  // blocks that certainly share a scale
  static constexpr int kSums = W * kFT * FN * 1024;
  static constexpr int kLds = W * kWave > kSums ? W * kWave : kSums;
  static_assert(kBN * kWPieces % 64 == 0 && U <= 8 && kLds <= 160 * 1024 && (S - 1) * kLoads < 64, "");
};

template <int XT, bool kFew, int XL, int FN, int U, int W, int S>
__global__ __launch_bounds__(W * 64) void int4_rows_kernel(Int4Args a) {
  typedef Rows<kFew, XL, FN, U, W, S> R;
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
    const int32_t x_piece = R::kOne ? lane : (lane % 8) ^ (lane / 16), x_pieces = a.k / 8;
    const uint8_t *x_from[R::kXLoads];
#pragma unroll
    for (int i = 0; i < R::kXLoads; ++i) {
      int32_t from = min(tile.first + 8 * i + (R::kOne ? 0 : lane / 8), tile.end - 1);
      if (a.gather) from = min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1);
      x_from[i] = static_cast<const uint8_t *>(a.x) + from * a.x_stride * 2;
    }
    // Of eight rows those that are not there are not read: what LDS holds of them gives sums that nobody looks at.
    const bool has_row = R::kOne ? lane < 8 * U : lane / 8 < tile.end - tile.first;
    const uint32_t lds_at = lds_address(mine);
    const int64_t w_first = (int64_t)tile.expert * a.n + n0;
    const uint8_t *const w_base = a.w + w_first * blocks * 16;
    const uint32_t w_row_bytes = (uint32_t)blocks * 16, w_last = (uint32_t)min(R::kBN - 1, a.n - 1 - n0) * w_row_bytes;
    // A load has 64 / kWPieces weight rows; with 8 pieces a row, odd loads have the other half of the keys.
    const int wrow = lane / R::kWPieces;
    const int32_t w_piece = (lane % R::kWPieces) ^ (wrow % 16 / (16 / R::kWPieces));

    auto period_of = [&](int32_t item) { return wave + W * (item / R::kSteps); };
    auto fetch = [&](int32_t item, int slot) {
      const int32_t step = period_of(item) * R::kSteps + item % R::kSteps;
      if constexpr (R::kOne) {
        if (has_row) copy16_apart(x_from[0] + min(step * U * 8 + x_piece, x_pieces - 1) * 16, lds_at + slot * R::kStage);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {  // eight rows a load, so odd loads have the other half of the keys
          const int32_t x_at[2] = {min((step * U + u) * 8 + x_piece, x_pieces - 1) * 16, min((step * U + u) * 8 + (x_piece ^ 4), x_pieces - 1) * 16};
          if (XL > 1 || has_row) {
#pragma unroll
            for (int i = 0; i < XL; ++i) copy16_apart(x_from[i] + x_at[i & 1], lds_at + slot * R::kStage + u * R::kLine + i * 1024);
          }
        }
      }
      const uint32_t w_at[2] = {(uint32_t)min(step * R::kWPieces + w_piece, blocks - 1) * 16,
                                (uint32_t)min(step * R::kWPieces + (w_piece ^ 4), blocks - 1) * 16};
#pragma unroll
      for (int i = 0; i < R::kWL; ++i)
        copy16_apart(w_base + (min((uint32_t)(wrow + i * (64 / R::kWPieces)) * w_row_bytes, w_last) + w_at[R::kWPieces == 8 ? i & 1 : 0]),
                     lds_at + slot * R::kStage + R::kXBytes + i * 1024);
    };
    Window<kFew> window[R::kSL];
    const bool turns = a.groups >= Window<kFew>::kEntries;
    auto scales_row = [&](int i) -> int64_t { return w_first + min(min(i * 64 + lane, R::kBN - 1), a.n - 1 - n0); };
    auto get_scales = [&](int32_t period) {
#pragma unroll
      for (int i = 0; i < R::kSL; ++i) load_window(a, scales_row(i), window_start<kFew>(a, period), window[i]);
    };
    auto put_scales = [&]() {  // LDS keeps a wave's order
#pragma unroll
      for (int i = 0; i < R::kSL; ++i)
        if (i * 64 + lane < R::kBN) put_window(a, window[i], ss + (i * 64 + lane) * R::kWindow);
    };
    auto multiply = [&](int32_t item, int slot, auto exactly) {
      constexpr bool kExact = decltype(exactly)::value;
      const int32_t in = item % R::kSteps, period = period_of(item);
      const uint8_t *const xl = mine + slot * R::kStage, *const wl = xl + R::kXBytes;
      u32x4 fx[2 * U][kFT];
      uint32_t fw[2 * U][FN];
#pragma unroll
      for (int b = 0; b < 2 * U; ++b) {
#pragma unroll
        for (int n = 0; n < FN; ++n)
          fw[b][n] = *reinterpret_cast<const uint32_t *>(wl + (n * 16 + r) * R::kWPieces * 16 + (b ^ (r / (16 / R::kWPieces))) * 16 + g * 4);
#pragma unroll
        for (int t = 0; t < kFT; ++t)
          fx[b][t] = *reinterpret_cast<const u32x4 *>(xl + b / 2 * R::kLine + (t * 16 + r) % R::kRows * 128 + ((4 * (b % 2) + g) ^ (R::kOne ? 0 : r >> 1)) * 16);
      }
      const int32_t first = 16 * period + in * 2 * U, start = window_start<kFew>(a, period);
      // Pieces past the end of x's rows hold other elements: they are taken as zeros.
      const int32_t left = a.k / 8 - first * 4;
      if (left < 8 * U) {
#pragma unroll
        for (int b = 0; b < 2 * U; ++b)
#pragma unroll
          for (int t = 0; t < kFT; ++t)
            if (4 * b + g >= left) fx[b][t] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int c = 0; c < 2 * U; c += R::kChain) {
        if (first + c >= blocks) break;  // nothing but zeros of x, and no scale
        const int32_t entry = ((first + c) >> a.shift) - start;
        f32x4 sum[kFT];  // of x
        if constexpr (!kExact) {
#pragma unroll
          for (int t = 0; t < kFT; ++t) {
            sum[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int b = c; b < c + R::kChain; ++b) sum[t] = mfma16<XT>(fx[b][t], int4_ones<XT>(), sum[t]);
          }
        }
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          float scale, zero;
          read_window<kFew>(a, ss + (n * 16 + r) * R::kWindow, entry, scale, zero);
          f32x4 part[kFT] = {};
#pragma unroll
          for (int b = c; b < c + R::kChain; ++b) {
            const u32x4 w = kExact ? int4_values<XT>(fw[b][n], zero) : int4_codes<XT>(fw[b][n]);
#pragma unroll
            for (int t = 0; t < kFT; ++t) part[t] = mfma16<XT>(fx[b][t], w, part[t]);
          }
#pragma unroll
          for (int t = 0; t < kFT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[t][n][i] = __builtin_fmaf(scale, kExact ? part[t][i] : __builtin_fmaf(-zero, sum[t][i], part[t][i]), acc[t][n][i]);
        }
      }
    };

    if (turns) {
      get_scales(wave);
    } else {
#pragma unroll
      for (int i = 0; i < R::kSL; ++i) load_all(a, scales_row(i), window[i]);
    }
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < items) fetch(i, i);
    int slot = 0;
    for (int32_t item = 0; item < items; ++item) {
      if (item % R::kSteps == 0) {
        put_scales();
        if (turns && item + R::kSteps < items) get_scales(period_of(item) + W);
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
    bool finite = true;
#pragma unroll
    for (int t = 0; t < kFT; ++t)
#pragma unroll
      for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) finite &= __builtin_fabsf(acc[t][n][i]) < __builtin_inff() || tile.first + t * 16 + 4 * g + i >= tile.end;
    if (__builtin_expect(__any(!finite), 0)) {
#pragma unroll
      for (int t = 0; t < kFT; ++t)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll 1
      for (int32_t item = 0; item < items; ++item) {
        if (item % R::kSteps == 0) {
          if (turns) get_scales(period_of(item));
          put_scales();
        }
        fetch(item, 0);
        wait_loads<0>();
        multiply(item, 0, std::true_type{});
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
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

// The shapes of a workgroup: 8 XL rows of x or one, 16 FN weight rows, U lines a stage, W waves, S stages. `resident` of them fit
// a CU, and one takes `us` for each period of k that a wave has; workgroups past the first on a CU cost `start` each beside. One token
// through 4096 x 14336, 4096 x 4096 and 14336 x 4096 (k x n) takes, in microseconds: one row and 32 weight rows 8.1, 5.4, 11.4; one and 16
// 9.3, 4.4, 8.5; eight rows and 32 weight rows, four waves 9.2, 6.4, 16.8, eight waves 10.9, 5.6, 12.0; eight and 16 14.0, 4.7, 9.1.
// 64 x 8192 x 8192: 32 rows and 64 weight rows 23.5, with three stages 24.8, with eight waves of half the stages 26.9, 32 and 32 29,
// 16 and 64 30. 32 x 4096 x 14336: 32 and 64 14.6, 16 and 64 19.0, with four waves 20.7; 64 x 4096 x 4096: 12.5, 9.1, 10.8, and 32 and 32 9.7.
struct Choice {
  int32_t rows, cols, waves, resident;
  float us, start;
};
constexpr Choice kChoices[] = {{1, 32, 8, 2, 2.0f, 1.3f},  {1, 16, 8, 3, 1.4f, 1.0f},  {8, 32, 4, 2, 2.5f, 1.3f},  {8, 32, 8, 1, 2.7f, 1.9f},
                               {8, 16, 8, 1, 2.0f, 1.0f},  {16, 32, 8, 1, 3.2f, 2.5f}, {16, 64, 8, 1, 5.5f, 2.1f}, {32, 32, 6, 1, 3.2f, 1.2f},
                               {32, 64, 4, 1, 3.7f, 2.7f}};
// Alike for all, the launch and the first loads, which the tiles' figures have in them; and what groups below 128 take more.
constexpr double kBase = 5.0, kFine = 1.35;

template <int XT, bool kFew, int XL, int FN, int U, int W, int S>
void launch(const Int4Args &a, hipStream_t stream) {
  typedef Rows<kFew, XL, FN, U, W, S> R;
  const dim3 grid((unsigned)((a.n + R::kBN - 1) / R::kBN), (unsigned)product_tiles(a, R::kRows));
  hipLaunchKernelGGL((int4_rows_kernel<XT, kFew, XL, FN, U, W, S>), grid, dim3(W * 64), 0, stream, a);
}

template <int XT, bool kFew>
void launch_type(const Int4Args &a, int choice, hipStream_t stream) {
  switch (choice) {
    case 0: return launch<XT, kFew, 0, 2, 4, 8, 2>(a, stream);
    case 1: return launch<XT, kFew, 0, 1, 4, 8, 2>(a, stream);
    case 2: return launch<XT, kFew, 1, 2, 4, 4, 2>(a, stream);
    case 3: return launch<XT, kFew, 1, 2, 4, 8, 2>(a, stream);
    case 4: return launch<XT, kFew, 1, 1, 4, 8, 2>(a, stream);
    case 5: return launch<XT, kFew, 2, 2, 2, 8, 2>(a, stream);
    case 6: return launch<XT, kFew, 2, 4, 2, 8, 2>(a, stream);
    case 7: return launch<XT, kFew, 4, 2, 2, 6, 2>(a, stream);
    default: return launch<XT, kFew, 4, 4, 2, 4, 2>(a, stream);
  }
}

}  // namespace

Prediction predict_int4_rows(const Int4Args &a, int32_t cus) {
  Prediction best = {-1, 0};
  const int64_t periods = (a.row_blocks + 15) / 16;
  int i = 0;
  for (const Choice &c : kChoices) {
    const int at = i++;
    // One row a workgroup reads its weights for that row alone: for a single row, or experts that have hardly more.
    if (c.rows == 1 && !a.offsets && a.rows > 1) continue;
    if (product_tiles(a, c.rows) > 65535 || (double)((a.n + c.cols - 1) / c.cols) * c.waves * 64 > kMostWorkItems) continue;
    const double each = (c.rows == 1 ? a.rows : expected_tiles(a, c.rows)) * (double)((a.n + c.cols - 1) / c.cols) / ((double)cus * c.resident);
    const double rounds = each <= 1 ? 1.0 : __builtin_ceil(each - 0.01);
    const double us = kBase + (rounds * (double)((periods + c.waves - 1) / c.waves) * c.us + (each > 1 ? each - 1 : 0) * c.start) * (a.shift < 2 ? kFine : 1.0);
    if (best.choice < 0 || us < best.us) best = {at, us};
  }
  return best;
}

void launch_int4_rows(const Int4Args &a, int32_t x_type, int choice, hipStream_t stream) {
  const bool few = a.shift >= 2;
  if (x_type == MPS_TYPE_BF16)
    few ? launch_type<MPS_TYPE_BF16, true>(a, choice, stream) : launch_type<MPS_TYPE_BF16, false>(a, choice, stream);
  else
    few ? launch_type<MPS_TYPE_F16, true>(a, choice, stream) : launch_type<MPS_TYPE_F16, false>(a, choice, stream);
}

}  // namespace mps
