// Products of many rows: tiles of 32 FT rows of x times 32 WN weight rows, a wave 32 of these and all of x's, with both operands'
// pieces of k staged in LDS.
//
// A step covers 64 elements of k: 128 bytes of every row of x, a cache line, and 32 of codes, which are widened in registers,
// after LDS. Pieces of 16 bytes go from memory to a ring of S stages in LDS without passing through registers; piece p of row r of x
// lies at place p ^ (r / 2 % 8), of codes at p ^ (r / 8 % 2), so that the sixteen lanes that LDS serves in a cycle
// meet all banks. A step's fragments are read while the one before is multiplied, quarter by quarter, so that a
// stage is free again, and the next one has to be there, at one place: the step's barrier.
//
// The matrix cores multiply x by the whole numbers q as they are. Products of columns that share a scale are summed by
// themselves and added with the scale in FP32. What the zeros take away, sum over groups of s z sum x, is another
// product, of the groups' sums of x and of s z, with which the sums begin: the sums of x (int4_sums_kernel) as three BF16
// numbers, s z as two, which hold it exactly; of the six products the least is left out (2^-25 of the sums). Where a tile's
// sums are not finite (x holds an infinity, or its sums pass 2^128) it makes them again from q - z.
#include "int4_product.h"

namespace mps {
namespace {

enum Chain { kBlock, kStep, kPair };  // columns that certainly share a scale: 32, 64, 128

template <Chain C, int FT, int WN, int S>
struct Shape {
  static constexpr int kBT = 32 * FT, kBN = 32 * WN, kThreads = 64 * WN;
  static constexpr int kXLoads = kBT * 8 / kThreads, kLoads = kXLoads + 1;  // loads a work-item and step
  static constexpr int kXBytes = kBT * 128, kStage = kXBytes + kBN * 32;
  static constexpr int kEntries = C == kBlock ? 16 : 8;  // scales of a row and period of 16 blocks
  static constexpr int kSBytes = kBN * kEntries * 2;
  static constexpr int kPitch = 36;  // floats of a row of sums, turned round
  static constexpr int kStaged = S * kStage + 2 * kSBytes, kTurned = WN * 32 * kPitch * 4;
  static constexpr int kLds = kStaged > kTurned ? kStaged : kTurned;
  static_assert(kBT * 8 % kThreads == 0 && kLds <= 160 * 1024 && kBN <= kThreads, "");
};

template <int XT>
__device__ inline f32x16 mfma32(u32x4 x, u32x4 w, f32x16 c) {
  if constexpr (XT == MPS_TYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
}

template <int XT, Chain C, int FT, int WN, int S>
__global__ __launch_bounds__(64 * WN) __attribute__((amdgpu_waves_per_eu(2, FT > 2 ? 2 : 4))) void int4_tile_kernel(Int4Args a, int32_t tiles_t, int32_t tiles_n) {
  typedef Shape<C, FT, WN, S> H;
  __shared__ __attribute__((aligned(16))) uint8_t lds[H::kLds];
  uint8_t *const ss = lds + S * H::kStage;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, g = lane >> 5;

  if (a.offsets) tiles_t = count_tiles(a.offsets, a.experts, a.rows, H::kBT);  // the host knows a bound only
  // Workgroups go to the 8 XCDs in turn. Each XCD takes a stretch of the tiles, in which
  // groups of 8 tiles of rows run through the weight's tiles together, so that its L2 serves both.
  const uint32_t total = (uint32_t)tiles_t * (uint32_t)tiles_n;
  const uint32_t per = (total + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || id >= total) return;
  const uint32_t group = id / (8u * tiles_n), in_group = id - group * 8u * tiles_n;
  const uint32_t group_t = min(8u, (uint32_t)tiles_t - group * 8);
  const int32_t tile_t = group * 8 + in_group % group_t, n0 = (in_group / group_t) * H::kBN;

  Tile tile = {0, tile_t * H::kBT, min(a.rows, tile_t * H::kBT + H::kBT)};
  if (a.offsets) tile = find_tile(a.offsets, a.experts, a.rows, H::kBT, tile_t);
  if (tile.expert < 0) return;
  const bool none = tile.expert >= max(a.experts, 1);  // rows of no expert
  const int32_t blocks = none ? 0 : a.row_blocks, steps = (blocks + 1) / 2;

  // Where this lane's pieces come from. Rows past the tile's end or the weight's are the last ones (what they
  // give is not stored), pieces past a row's end its last one.
  auto row_of = [&](int32_t i) -> int32_t {
    const int32_t from = min(tile.first + i, tile.end - 1);
    return a.gather ? min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1) : from;
  };
  const int xrow = tid / 8, wrow = tid / 2;
  const int32_t x_piece = (tid % 8) ^ (xrow >> 1 & 7), w_piece = (tid % 2) ^ (wrow >> 3 & 1), x_pieces = blocks * 4;
  const uint8_t *x_from[H::kXLoads];
#pragma unroll
  for (int i = 0; i < H::kXLoads; ++i) x_from[i] = static_cast<const uint8_t *>(a.x) + row_of(xrow + i * (H::kThreads / 8)) * a.x_stride * 2;
  const int64_t w_first = (int64_t)(none ? 0 : tile.expert) * a.n + n0;
  const int32_t last_col = a.n - 1 - n0;
  const uint8_t *const w_from = a.w + (w_first + min(wrow, last_col)) * a.row_blocks * 16;
  auto fetch = [&](int32_t step, uint32_t slot) {
    uint8_t *const to = lds + slot * H::kStage;
    const uint32_t x_at = (uint32_t)min(step * 8 + x_piece, x_pieces - 1) * 16;
#pragma unroll
    for (int i = 0; i < H::kXLoads; ++i) copy16(x_from[i] + x_at, to + wave * 1024 + i * H::kThreads * 16);
    copy16(w_from + (uint32_t)min(step * 2 + w_piece, blocks - 1) * 16, to + H::kXBytes + wave * 1024);
  };

  // Scales come a period ahead, through registers: a row's kEntries from its first group in the period on, near the
  // row's end from earlier on, alike for all rows.
  auto scales_start = [&](int32_t period) -> int32_t { return max(0, min((16 * period) >> a.shift, a.groups - H::kEntries)); };
  // A row that has fewer in all has them in both buffers from the start.
  uint32_t scales[H::kEntries / 2] = {};
  const bool turns = a.groups >= H::kEntries, has_scales = tid < H::kBN;
  const uint16_t *const s_row = static_cast<const uint16_t *>(a.scales) + (w_first + min(tid, min(H::kBN - 1, last_col))) * a.groups;
  auto get_scales = [&](int32_t period) {
    if (has_scales) __builtin_memcpy(scales, s_row + scales_start(period), sizeof(scales));
  };
  auto put_scales = [&](int32_t period) {
    u32x4 *const to = reinterpret_cast<u32x4 *>(ss + (period & 1) * H::kSBytes + tid * H::kEntries * 2);
    if (has_scales) {
#pragma unroll
      for (int i = 0; i < H::kEntries / 8; ++i) to[i] = u32x4{scales[4 * i], scales[4 * i + 1], scales[4 * i + 2], scales[4 * i + 3]};
    }
  };
  auto scale_of = [&](int32_t block) -> float {
    const int32_t period = block / 16, entry = (block >> a.shift) - scales_start(period);
    return scale_value(*reinterpret_cast<const uint16_t *>(ss + (period & 1) * H::kSBytes + (wave * 32 + r) * H::kEntries * 2 + entry * 2), a.scale_type);
  };

  // Lanes 0-31 and 32-63 take a half each of a step's 64 elements: of either block where blocks have scales of their
  // own, else a block. Quarter q is eight elements of each half.
  f32x16 acc[FT] = {}, part[FT] = {};
  u32x4 fx[4][FT];
  uint32_t fw[4], fw_next[4];
  const int x_lane = r * 128, w_lane = (wave * 32 + r) * 32;
  auto x_place = [&](int q) -> int { return ((C == kBlock ? 4 * (q >> 1) + 2 * g + (q & 1) : 4 * g + q) ^ (r >> 1 & 7)) * 16 + x_lane; };
  auto read_x = [&](int q, uint32_t slot) {
    const uint8_t *const from = lds + slot * H::kStage + x_place(q);
#pragma unroll
    for (int t = 0; t < FT; ++t) fx[q][t] = *reinterpret_cast<const u32x4 *>(from + t * 4096);
  };
  auto read_w = [&](uint32_t (&to)[4], uint32_t slot) {
    const uint8_t *const from = lds + slot * H::kStage + H::kXBytes + w_lane;
    if constexpr (C == kBlock) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t v = *reinterpret_cast<const uint64_t *>(from + (h ^ (r >> 3 & 1)) * 16 + g * 8);
        to[2 * h] = (uint32_t)v, to[2 * h + 1] = (uint32_t)(v >> 32);
      }
    } else {
      const u32x4 v = *reinterpret_cast<const u32x4 *>(from + (g ^ (r >> 3 & 1)) * 16);
#pragma unroll
      for (int q = 0; q < 4; ++q) to[q] = v[q];
    }
  };
  // A last step of one block: the other's pieces are taken as zeros. So are those of a step past the last.
  auto cut = [&](int32_t step) {
    if (2 * step + 1 < blocks) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool past = (C == kBlock ? q >= 2 : g == 1) || (C == kPair && 2 * step >= blocks);
#pragma unroll
      for (int t = 0; t < FT; ++t)
        if (past) fx[q][t] = u32x4{0, 0, 0, 0};
    }
  };

  float pending = 0;  // the scale of the products that `part` holds
  if (steps > 0) {
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (i < steps) fetch(i, i);
    if (turns) {
      get_scales(0);
    } else {
      uint16_t few[H::kEntries];
#pragma unroll
      for (int i = 0; i < H::kEntries; ++i) few[i] = s_row[min(i, a.groups - 1)];
#pragma unroll
      for (int i = 0; i < H::kEntries / 2; ++i) scales[i] = few[2 * i] | (uint32_t)few[2 * i + 1] << 16;
    }
    // What the zeros take away: 16 groups at a time.
    const int64_t col = w_first + min(wave * 32 + r, last_col);
    const uint8_t *sums[FT];
#pragma unroll
    for (int t = 0; t < FT; ++t) sums[t] = static_cast<const uint8_t *>(a.sums) + (int64_t)row_of(t * 32 + r) * a.sums_row + g * 16;
    for (int32_t c = 0; c < a.groups; c += 16) {
      uint32_t sb[8], zb[8];  // loads without branches, so that they are in flight together
#pragma unroll
      for (int i = 0; i < 8; ++i) sb[i] = static_cast<const uint16_t *>(a.scales)[col * a.groups + min(c + 8 * g + i, a.groups - 1)], zb[i] = 8;
      if (a.zeros) {
#pragma unroll
        for (int i = 0; i < 8; ++i) zb[i] = a.zeros[col * a.groups + min(c + 8 * g + i, a.groups - 1)] & 31;
      }
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          f[j] = c + 8 * g + 2 * i + j < a.groups ? -scale_value(sb[2 * i + j], a.scale_type) * (float)zb[2 * i + j] : 0.0f;
        hi[i] = pack2(f[0], f[1], MPS_TYPE_BF16);
        lo[i] = pack2(f[0] - __uint_as_float(hi[i] << 16), f[1] - __uint_as_float(hi[i] & 0xffff0000u), MPS_TYPE_BF16);
      }
#pragma unroll
      for (int t = 0; t < FT; ++t) {
        const uint8_t *const from = sums[t] + c / 16 * 96;
        const u32x4 x0 = *reinterpret_cast<const u32x4 *>(from), x1 = *reinterpret_cast<const u32x4 *>(from + 32), x2 = *reinterpret_cast<const u32x4 *>(from + 64);
        acc[t] = mfma32<MPS_TYPE_BF16>(x2, hi, acc[t]);
        acc[t] = mfma32<MPS_TYPE_BF16>(x1, lo, acc[t]);
        acc[t] = mfma32<MPS_TYPE_BF16>(x1, hi, acc[t]);
        acc[t] = mfma32<MPS_TYPE_BF16>(x0, lo, acc[t]);
        acc[t] = mfma32<MPS_TYPE_BF16>(x0, hi, acc[t]);
      }
    }
    put_scales(0);
    if (!turns) put_scales(1);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int q = 0; q < 4; ++q) read_x(q, 0);
    read_w(fw, 0);
  }
  uint32_t slot = 0;  // of this step
  auto body = [&](int32_t step, auto odd) {
    const uint32_t next = slot + 1 == S ? 0 : slot + 1;
    if (step + S <= steps)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * H::kLoads) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + S < steps) fetch(step + S, slot);
    if (turns && step % 8 == 0 && step + 8 < steps) get_scales(step / 8 + 1);
    if (turns && step % 8 == 6 && step + 2 < steps) put_scales(step / 8 + 1);
    cut(step);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u32x4 w = int4_codes<XT>(fw[q]);
      // Where another scale begins, what has been summed with the last one is added, and the sums begin again.
      if (C == kBlock ? q % 2 == 0 : q == 0 && !decltype(odd)::value) {
        const float scale = scale_of(C == kBlock ? min(2 * step + (q >> 1), blocks - 1) : 2 * step);
#pragma unroll
        for (int t = 0; t < FT; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] = __builtin_fmaf(pending, part[t][i], acc[t][i]);
          asm volatile("" : "+v"(acc[t]));  // the sums stay where they are
          __builtin_amdgcn_sched_barrier(0);
          part[t] = mfma32<XT>(fx[q][t], w, f32x16{});
          asm volatile("" : "+v"(part[t]));
        }
        pending = scale;
      } else {
#pragma unroll
        for (int t = 0; t < FT; ++t) {
          part[t] = mfma32<XT>(fx[q][t], w, part[t]);
          asm volatile("" : "+v"(part[t]));
        }
      }
      read_x(q, next);  // past the last step: of a stage that nobody writes
      if (q == 1) read_w(fw_next, next);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) fw[q] = fw_next[q];
    slot = next;
  };
#pragma unroll 1
  for (int32_t step = 0; step < steps; step += C == kPair ? 2 : 1) {
    body(step, std::false_type{});
    if constexpr (C == kPair) body(step + 1, std::true_type{});  // where there is none, of zeros
  }
  bool finite = true;
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      acc[t][i] = __builtin_fmaf(pending, part[t][i], acc[t][i]);
      finite &= __builtin_fabsf(acc[t][i]) < __builtin_inff();
    }
  if (__builtin_expect(__syncthreads_or(!finite), 0)) {  // all again, a step at a time, with scales and zeros from memory
#pragma unroll
    for (int t = 0; t < FT; ++t) acc[t] = f32x16{};
    const int64_t col = w_first + min(wave * 32 + r, last_col);
#pragma unroll 1
    for (int32_t step = 0; step < steps; ++step) {
      __syncthreads();
      fetch(step, 0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int q = 0; q < 4; ++q) read_x(q, 0);
      read_w(fw, 0);
      cut(step);
#pragma unroll
      for (int h = 0; h < (C == kBlock ? 2 : 1); ++h) {
        if (2 * step + h >= blocks) break;
        const int32_t at = (2 * step + h) >> a.shift;
        const float s = int4_scale(a, col, at), zero = int4_zero(a, col, at);
#pragma unroll
        for (int t = 0; t < FT; ++t) part[t] = f32x16{};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (C == kBlock && q / 2 != h) continue;
          const u32x4 w = int4_values<XT>(fw[q], zero);
#pragma unroll
          for (int t = 0; t < FT; ++t) part[t] = mfma32<XT>(fx[q][t], w, part[t]);
        }
#pragma unroll
        for (int t = 0; t < FT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] = __builtin_fmaf(s, part[t][i], acc[t][i]);
      }
    }
    __syncthreads();
  }

  // A lane's 16 sums are rows 8 i + 4 g .. + 3 of column r. The wave turns 32 rows at a time round through its own part
  // of LDS, so that a store has neighbouring columns.
  constexpr int kPitch = H::kPitch;
  float *const mine = reinterpret_cast<float *>(lds) + wave * 32 * kPitch;
  const int32_t col = n0 + wave * 32 + lane % 4 * 8;
  f32x4 bias[2] = {};
  if (a.bias && !none) bias[0] = load_bias4(a, tile.expert, col), bias[1] = load_bias4(a, tile.expert, col + 4);
#pragma unroll
  for (int t = 0; t < FT; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mine[(8 * i + 4 * g + j) * kPitch + r] = acc[t][4 * i + j];
    __builtin_amdgcn_wave_barrier();
    f32x4 v[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[i][h] = *reinterpret_cast<const f32x4 *>(mine + (i * 16 + lane / 4) * kPitch + lane % 4 * 8 + 4 * h) + bias[h];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t row = tile.first + t * 32 + i * 16 + lane / 4;
      if (row < tile.end && col < a.n) store8(a, row, col, v[i][0], v[i][1]);
    }
  }
}

template <int XT, Chain C, int FT, int WN, int S>
void launch(const Int4Args &a, hipStream_t stream) {
  typedef Shape<C, FT, WN, S> H;
  const int64_t tt = product_tiles(a, H::kBT), tn = (a.n + H::kBN - 1) / H::kBN;
  const int64_t grid = (tt * tn + 7) / 8 * 8;
  hipLaunchKernelGGL((int4_tile_kernel<XT, C, FT, WN, S>), dim3((unsigned)grid), dim3(WN * 64), 0, stream, a, (int32_t)tt, (int32_t)tn);
}

struct Choice {
  int32_t bt, bn;
  float start, one, many;
};
constexpr Choice kChoices[] = {{128, 256, 4.6f, 51.0f, 53.0f}, {128, 128, 2.6f, 35.0f, 30.0f}, {64, 128, 1.8f, 26.0f, 18.5f}};

template <int XT, Chain C>
void launch_chain(const Int4Args &a, int choice, hipStream_t stream) {
  switch (choice) {
    case 0: return launch<XT, C, 4, 8, 3>(a, stream);
    case 1: return launch<XT, C, 4, 4, 3>(a, stream);
    default: return launch<XT, C, 2, 4, 3>(a, stream);
  }
}
template <int XT>
void launch_type(const Int4Args &a, int choice, hipStream_t stream) {
  if (a.shift == 0)
    launch_chain<XT, kBlock>(a, choice, stream);
  else if (a.shift == 1)
    launch_chain<XT, kStep>(a, choice, stream);
  else
    launch_chain<XT, kPair>(a, choice, stream);
}

}  // namespace

Prediction predict_int4_tiles(const Int4Args &a, int32_t x_type, int32_t cus) {
  Prediction best = {-1, 0};
  int i = 0;
  for (const Choice &c : kChoices) {
    const int at = i++;
    if (((double)product_tiles(a, c.bt) * (double)((a.n + c.bn - 1) / c.bn) + 8) * 512 > kMostWorkItems) continue;
    const double tiles = expected_tiles(a, c.bt) * (double)((a.n + c.bn - 1) / c.bn) / cus, k = a.row_blocks / 128.0;
    const double each = __builtin_ceil(tiles - 0.01);
    const double us = each <= 1 ? c.start + c.one * k : each * (c.start + c.many * k);
    if (best.choice < 0 || us < best.us) best = {at, us};
  }
  return best;
}

void launch_int4_tiles(const Int4Args &a, int32_t x_type, int choice, hipStream_t stream) {
  if (x_type == MPS_TYPE_BF16)
    launch_type<MPS_TYPE_BF16>(a, choice, stream);
  else
    launch_type<MPS_TYPE_F16>(a, choice, stream);
}

}  // namespace mps
