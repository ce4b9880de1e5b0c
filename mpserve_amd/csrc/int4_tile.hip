// Products of many rows: tiles of 32 FT WT rows of x times 32 FN WN weight rows, a wave FT x FN fragments of 32 x 32, with
// both operands' pieces of k staged in LDS.
//
// A step covers 64 elements of k: 128 bytes of every row of x, a cache line, and 32 of codes, which are widened in registers,
// after LDS. A stage is two steps. Pieces of 16 bytes go from memory to a ring of three stages in LDS without passing through
// registers; piece p of row r of x lies at place p ^ (r / 2 % 8), of codes at p ^ (r / 8 % 2), so that the sixteen lanes that
// LDS serves in a cycle meet all banks. A step's fragments are read two quarters of it ahead, among the products.
// A stage's one barrier stands before its second step, for two things: the next stage has come, and nobody needs the one
// before any more, whose fragments all have used, so that no wave waits there for reads of its own. (BF16, groups of 128, 4096 x 4096 x
// 14336: loads and reads in a row behind the barrier 560 us, among the products 505.)
//
// The matrix cores multiply x by the whole numbers q as they are. Products of columns that share a scale are summed by
// themselves and added with the scale in FP32. What the zeros take away, sum over spans of s z sum x (a span is a group, at
// most 128 columns), is another product, of the spans' sums of x and of s z: the sums of x (int4_sums_kernel) as three BF16
// numbers, s z as two, which hold it exactly; of the six products the least is left out (2^-25 of the sums). It is taken away four spans at a
// time, beside these spans' own products: no sum on the way is larger than the result and four spans' part. (All of it in front of the first
// product takes 2 % fewer matrix instructions, and 2.5 % less time there, but where x has a mean every addition then rounds at the size of
// the whole: x of mean and sigma 1, 28672 columns, groups of 128, results in FP32 off by 4.6e-6 of their size, so by 3.8e-7.) Where a tile's
// sums are not finite (x holds an infinity, or its sums pass 2^128) it makes them again from q - z.
#include "int4_product.h"

namespace mps {
namespace {

// What a piece past the end of a row of x is read from.
__device__ __attribute__((aligned(16))) const uint32_t kNothing[4] = {0, 0, 0, 0};

enum Chain { kBlock, kStep, kPair };  // columns that certainly share a scale: 32, 64, 128

constexpr int kStages = 3;

template <Chain C, int FT, int FN, int WT, int WN>
struct Shape {
  static constexpr int kBT = 32 * FT * WT, kBN = 32 * FN * WN, kWaves = WT * WN, kThreads = 64 * kWaves;
  static constexpr int kXLoads = kBT * 8 / kThreads, kWLoads = (kBN * 2 + kThreads - 1) / kThreads;  // a work-item and step
  static constexpr int kLoads = 2 * (kXLoads + kWLoads);                                             // and stage
  static constexpr int kWLanes = kBN * 2 / kWaves < 64 ? kBN * 2 / kWaves : 64;                      // that load codes
  static constexpr int kXBytes = kBT * 128, kStep = kXBytes + kBN * 32, kStage = 2 * kStep;
  static constexpr int kEntries = 8, kPeriod = C == kBlock ? 2 : 4;  // scales of a row in a period; stages a period
  static constexpr int kSBytes = kBN * kEntries * 2;
  // Spans: their columns as a power of two of blocks; stages of four of them; bytes of all rows' four sums of x, and places for these.
  static constexpr int kSpan = C == kBlock ? 0 : C == Chain::kStep ? 1 : 2, kFour = 1 << kSpan, kFourBytes = kBT * 32, kFours = C == kBlock ? 2 : 1;
  static constexpr int kAhead = 2;  // quarters of a step by which x is read ahead
  static constexpr int kPitch = 32 * FN + 4;  // floats of a row of sums, turned round
  static constexpr int kStaged = kStages * kStage + 2 * kSBytes + kFours * kFourBytes, kTurned = kWaves * 32 * kPitch * 4;
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

template <int XT, Chain C, int FT, int FN, int WT, int WN>
__global__ __launch_bounds__(64 * WT * WN) __attribute__((amdgpu_waves_per_eu(2, 2))) void int4_tile_kernel(Int4Args a, int32_t tiles_t, int32_t tiles_n) {
  typedef Shape<C, FT, FN, WT, WN> H;
  __shared__ __attribute__((aligned(16))) uint8_t lds[H::kLds];
  uint8_t *const ss = lds + kStages * H::kStage, *const xs = ss + 2 * H::kSBytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, g = lane >> 5;
  const int wt = wave / WN, wn = wave % WN;

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
  tile = {__builtin_amdgcn_readfirstlane(tile.expert), __builtin_amdgcn_readfirstlane(tile.first), __builtin_amdgcn_readfirstlane(tile.end)};
  if (tile.expert < 0) return;
  const bool none = tile.expert >= max(a.experts, 1);  // rows of no expert
  const int32_t blocks = none ? 0 : a.row_blocks, pairs = (blocks + 3) / 4;  // of steps

  // Where this lane's pieces come from. Rows past the tile's end or the weight's are the last ones (what they
  // give is not stored), pieces past a row's end its last one.
  auto row_of = [&](int32_t i) -> int32_t {
    const int32_t from = min(tile.first + i, tile.end - 1);
    return a.gather ? min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1) : from;
  };
  const int w_first_piece = wave * H::kWLanes + lane;  // of the first load's
  const int xrow = tid / 8, wrow = w_first_piece / 2;
  const uint32_t x_piece = ((tid % 8) ^ (xrow >> 1 & 7)) * 16, w_piece = ((w_first_piece % 2) ^ (wrow >> 3 & 1)) * 16;
  const uint32_t x_end = blocks * 64, w_last = blocks * 16 - 16;
  const uint8_t *x_from[H::kXLoads];
#pragma unroll
  for (int i = 0; i < H::kXLoads; ++i)
    x_from[i] = static_cast<const uint8_t *>(a.x) + row_of(xrow + i * (H::kThreads / 8)) * a.x_stride * 2 + x_piece;
  const int64_t w_first = (int64_t)(none ? 0 : tile.expert) * a.n + n0;
  const int32_t last_col = a.n - 1 - n0;
  const uint8_t *const w_base = scalar(a.w + w_first * a.row_blocks * 16);
  uint32_t w_from[H::kWLoads];  // from there on: below 256 rows of 2^23 bytes
#pragma unroll
  for (int i = 0; i < H::kWLoads; ++i) w_from[i] = (uint32_t)min(wrow + i * (H::kThreads / 2), last_col) * (uint32_t)(a.row_blocks * 16) + w_piece;
  // Load l of a stage, to `to` in LDS. The stages at a row's end may be parts of one or none at all: x's pieces past
  // its end are zeros, the codes' what they are.
  const uint32_t lds_at = lds_address(lds) + wave * 1024, w_lds_at = lds_address(lds) + H::kXBytes + wave * H::kWLanes * 16;
  auto fetch = [&](int32_t pair, uint32_t to, int l, auto whole) __attribute__((always_inline)) {
    const int h = l / (H::kLoads / 2), i = l % (H::kLoads / 2);
    asm volatile("" : "+s"(pair));  // lest every load of an unrolled period gets an address of its own to count up
    if (i < H::kXLoads) {
      const uint32_t at = pair * 256 + h * 128;
      const uint8_t *from = x_from[i] + at;
      if (!decltype(whole)::value) from = at + x_piece < x_end ? from : reinterpret_cast<const uint8_t *>(kNothing);
      copy16_apart(from, lds_at + to + h * H::kStep + i * H::kThreads * 16);
    } else if (H::kWLanes == 64 || lane < H::kWLanes) {
      const uint32_t at = pair * 64 + h * 32, lds_to = w_lds_at + to + h * H::kStep + (i - H::kXLoads) * H::kThreads * 16;
      if (decltype(whole)::value)
        copy16_apart(w_base + at, w_from[i - H::kXLoads], lds_to);
      else
        copy16_apart(w_base, w_from[i - H::kXLoads] - w_piece + min(at + w_piece, w_last), lds_to);
    }
  };
  auto fetch_all = [&](int32_t pair, uint32_t to) __attribute__((always_inline)) {
#pragma unroll
    for (int l = 0; l < H::kLoads; ++l) fetch(pair, to, l, std::false_type{});
  };

  // Scales come a period ahead, through registers: a row's kEntries from its first group in the period on, near the
  // row's end from earlier on, alike for all rows.
  auto scales_start = [&](int32_t period) -> int32_t { return max(0, min((4 * H::kPeriod * period) >> a.shift, a.groups - H::kEntries)); };
  // A row that has fewer in all has them in both buffers from the start.
  uint32_t scales[H::kEntries / 2] = {};
  const bool turns = a.groups >= H::kEntries, has_scales = tid < H::kBN;
  const uint8_t *const s_first = scalar(static_cast<const uint8_t *>(a.scales) + w_first * a.groups * 2);
  auto get_scales = [&](int32_t period) {
    if (has_scales) {
      uint32_t row = min(tid, last_col);
      asm volatile("" : "+v"(row));
      __builtin_memcpy(scales, s_first + (row * (uint32_t)a.groups + (uint32_t)scales_start(period)) * 2, sizeof(scales));
    }
  };
  auto put_scales = [&](int32_t period) {
    u32x4 *const to = reinterpret_cast<u32x4 *>(ss + (period & 1) * H::kSBytes + tid * H::kEntries * 2);
    if (has_scales) *to = u32x4{scales[0], scales[1], scales[2], scales[3]};
  };
  auto scale_of = [&](int n, int32_t block) -> float {
    const int32_t period = block / (4 * H::kPeriod), entry = (block >> a.shift) - scales_start(period);
    return scale_value(*reinterpret_cast<const uint16_t *>(ss + (period & 1) * H::kSBytes + ((wn * FN + n) * 32 + r) * H::kEntries * 2 + entry * 2),
                       a.scale_type);
  };

  // Lanes 0-31 and 32-63 take a half each of a step's 64 elements: of either block where blocks have scales of their
  // own, else a block. Quarter q is eight elements of each half.
  f32x16 acc[FT][FN] = {}, part[FT][FN] = {};
  u32x4 fx[H::kAhead][FT];
  uint32_t fw[2][FN][4];  // of even and odd steps
  u32x4 w0[FN], w1[FN];   // widened: of the even and the odd quarter
  const int x_lane = (wt * FT * 32 + r) * 128, w_lane = (wn * FN * 32 + r) * 32;
  auto x_place = [&](int q) -> int { return ((C == kBlock ? 4 * (q >> 1) + 2 * g + (q & 1) : 4 * g + q) ^ (r >> 1 & 7)) * 16 + x_lane; };
  auto read_x = [&](int q, int t, uint32_t at) { fx[q % H::kAhead][t] = *reinterpret_cast<const u32x4 *>(lds + at + x_place(q) + t * 4096); };
  auto read_w = [&](uint32_t (&to)[FN][4], uint32_t at) {
    const uint8_t *const from = lds + at + H::kXBytes + w_lane;
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      if constexpr (C == kBlock) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t v = *reinterpret_cast<const uint64_t *>(from + n * 1024 + (h ^ (r >> 3 & 1)) * 16 + g * 8);
          to[n][2 * h] = (uint32_t)v, to[n][2 * h + 1] = (uint32_t)(v >> 32);
        }
      } else {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(from + n * 1024 + (g ^ (r >> 3 & 1)) * 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) to[n][q] = v[q];
      }
    }
  };
  float pending[FN] = {};  // the scales of the products that `part` holds
  int64_t cols[FN];
#pragma unroll
  for (int n = 0; n < FN; ++n) cols[n] = w_first + min((wn * FN + n) * 32 + r, last_col);
  // What the zeros take away, four sums of x at a time, which come to LDS ahead; the zeros a period ahead to registers, a column's
  // kEntries as its scales. Addresses are made each time: registers are what the largest tiles lack.
  const int32_t sum_row = pairs > 0 && tid < 2 * H::kBT ? row_of(tid / 2) : 0;
  const uint8_t *const z_first = scalar(a.zeros + w_first * a.groups);
  uint32_t zeros[FN][2];
  auto get_sums = [&](int32_t four) {
    if (wave < H::kBT / 32) {
      int32_t row = sum_row;
      asm volatile("" : "+v"(row));
      copy16_apart(static_cast<const uint8_t *>(a.sums) + row * a.sums_row + (four * 32 + lane % 2 * 16), lds_address(xs) + four % H::kFours * H::kFourBytes + wave * 1024);
    }
  };
  auto get_zeros = [&](int32_t period) {
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      uint32_t col = min((wn * FN + n) * 32 + r, last_col);
      asm volatile("" : "+v"(col));
      __builtin_memcpy(zeros[n], z_first + col * (uint32_t)a.groups + (uint32_t)scales_start(period), 8);
    }
  };
  auto read_sums = [&](int32_t four, int t) -> u32x4 {
    return *reinterpret_cast<const u32x4 *>(xs + four % H::kFours * H::kFourBytes + ((wt * FT + t) * 32 + r) * 32 + g * 16);
  };
  // This lane's two spans of the four: their scales, and minus s z, its first eight bits and above them what these leave.
  auto four_entry = [&](int32_t four, int j) -> int32_t {
    return (min((4 * four + 2 * g + j) << H::kSpan, blocks - 1) >> a.shift) - scales_start(four * H::kFour / H::kPeriod);
  };
  auto read_scale = [&](int32_t four, int n, int j) -> uint32_t {
    return *reinterpret_cast<const uint16_t *>(ss + (four * H::kFour / H::kPeriod & 1) * H::kSBytes + ((wn * FN + n) * 32 + r) * H::kEntries * 2 + four_entry(four, j) * 2);
  };
  auto scaled_zero = [&](int32_t four, int n, int j, uint32_t scale) -> uint32_t {
    const uint32_t zero = __builtin_amdgcn_perm(zeros[n][1], zeros[n][0], 0x0c0c0c00u | (uint32_t)four_entry(four, j)) & 31;
    const float f = -scale_value(scale, a.scale_type) * (float)zero;
    return pack2(f, f - Elem<MPS_TYPE_BF16>::get(Elem<MPS_TYPE_BF16>::put(f)), MPS_TYPE_BF16);
  };
  if (pairs > 0) {
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch_all(i, i * H::kStage);
    if (turns) {
      get_scales(0);
    } else {
      uint16_t few[H::kEntries];
#pragma unroll
      for (int i = 0; i < H::kEntries; ++i)
        few[i] = reinterpret_cast<const uint16_t *>(s_first)[(uint32_t)min(min(tid, H::kBN - 1), last_col) * (uint32_t)a.groups + (uint32_t)min(i, a.groups - 1)];
#pragma unroll
      for (int i = 0; i < H::kEntries / 2; ++i) scales[i] = few[2 * i] | (uint32_t)few[2 * i + 1] << 16;
    }
    get_sums(0);
    if (!a.zeros) {
#pragma unroll
      for (int n = 0; n < FN; ++n) zeros[n][0] = zeros[n][1] = 0x08080808u;
    } else if (turns) {
      get_zeros(0);
    } else {
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = z_first[(uint32_t)min((wn * FN + n) * 32 + r, last_col) * (uint32_t)a.groups + (uint32_t)min(i, a.groups - 1)];
#pragma unroll
        for (int i = 0; i < 2; ++i) zeros[n][i] = e[4 * i] | e[4 * i + 1] << 8 | e[4 * i + 2] << 16 | e[4 * i + 3] << 24;
      }
    }
    put_scales(0);
    if (!turns) put_scales(1);
    if (H::kPeriod == 2 && turns && H::kPeriod < pairs) get_scales(1);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int q = 0; q < H::kAhead; ++q)
#pragma unroll
      for (int t = 0; t < FT; ++t) read_x(q, t, 0);
    read_w(fw[0], 0);
#pragma unroll
    for (int n = 0; n < FN; ++n) w0[n] = int4_codes<XT>(fw[0][n][0]);
  }
  // Where this stage, the next and the one after it lie.
  uint32_t here = 0, then = H::kStage, after = 2 * H::kStage;
  // A step. The fragments' products come in an order in which, where another scale begins, the 16 multiply-adds a lane that
  // add what has been summed with the last one stand beside two products each. Between two products there is room for
  // a read of the next step's fragments, a load of the stage after the next, or the widening of a quarter's codes.
  // `known`: the stage's place in its period, or -1, which makes it be asked for.
  auto body = [&](int32_t pair, auto odd, auto whole, auto known) __attribute__((always_inline)) {
    constexpr int kOdd = decltype(odd)::value, kM = FT * FN, kKnown = decltype(known)::value;
    constexpr int kMade = FT == 1 ? 1 : 2;  // products behind which s z is made, from scales read behind the first
    const int32_t place = kKnown >= 0 ? kKnown : pair % H::kPeriod;
    if constexpr (kOdd == 1) {
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      if (place == H::kPeriod - 2 && turns && pair + 2 < pairs) {
        const int32_t period = pair / H::kPeriod + 1;  // the next one
        put_scales(period);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
#pragma unroll
      for (int n = 0; n < FN; ++n) asm volatile("" : "+v"(zeros[n][0]), "+v"(zeros[n][1]));  // here the wait for them costs nothing
    }
    // The first stage of four spans takes away what their zeros do, among the odd step's products.
    const bool takes = kOdd && place % H::kFour == 0;
    const int32_t four = pair / H::kFour;
    u32x4 sums[FT];
    uint32_t sz[FN][2];
    const uint32_t next = kOdd ? then : here + H::kStep;
    int load = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool fresh = C == kBlock || (h == 0 && (C == kStep || kOdd == 0));
      float scale[FN];
      if (fresh) {
#pragma unroll
        for (int n = 0; n < FN; ++n) scale[n] = scale_of(n, min(4 * pair + 2 * kOdd + (C == kBlock ? h : 0), blocks - 1));
      }
#pragma unroll
      for (int s = 0; s < 2 * kM; ++s) {
        // Fresh: 0, 1, 0', 2, 1', 3, 2' ..; else 0, 1, 2 .. 0', 1', 2' ..
        const int second = fresh ? (s == 2 * kM - 1 || (s > 0 && s % 2 == 0)) : s >= kM;
        const int i = fresh ? (s == 0 ? 0 : s == 2 * kM - 1 ? kM - 1 : second ? s / 2 - 1 : (s + 1) / 2) : s % kM;
        const int t = i % FT, n = i / FT, q = 2 * h + second;
        if (fresh && !second) {
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[t][n][j] = __builtin_fmaf(pending[n], part[t][n][j], acc[t][n][j]);
          asm volatile("" : "+v"(acc[t][n]));  // the sums stay where they are
          __builtin_amdgcn_sched_barrier(0);
          part[t][n] = mfma32<XT>(fx[q % H::kAhead][t], w0[n], f32x16{});
        } else {
          part[t][n] = mfma32<XT>(fx[q % H::kAhead][t], second ? w1[n] : w0[n], part[t][n]);
        }
        asm volatile("" : "+v"(part[t][n]));
        if (n == FN - 1) read_x((q + H::kAhead) % 4, t, q + H::kAhead < 4 ? here + kOdd * H::kStep : next);
        if (s == 0) {
#pragma unroll
          for (int m = 0; m < FN; ++m) w1[m] = int4_codes<XT>(fw[kOdd][m][2 * h + 1]);
        }
        if (h == 0 && s == 1) read_w(fw[kOdd ^ 1], next);
        if (!second && i == kM - 1) {  // the last of the even quarter
#pragma unroll
          for (int m = 0; m < FN; ++m) w0[m] = int4_codes<XT>(h == 0 ? fw[kOdd][m][2] : fw[kOdd ^ 1][m][0]);
        }
        if (kOdd == 1) {
          const int slot = 2 * kM * h + s;
          if (load < H::kLoads) fetch(pair + 2, after, load++, whole);
          if (takes) {
            if (slot == 0 || slot == kMade) {
#pragma unroll
              for (int m = 0; m < FN; ++m)
#pragma unroll
                for (int j = 0; j < 2; ++j) sz[m][j] = slot == 0 ? read_scale(four, m, j) : scaled_zero(four, m, j, sz[m][j]);
            }
#pragma unroll
            for (int u = 0; u < FT; ++u) {
              // all sums at once, or where registers lack one after the other
              if (slot == (FT <= 2 ? 0 : 3 * u + 1)) sums[u] = read_sums(four, u);
              if (slot == (FT <= 2 ? 2 * kM + u : 3 * u + 3)) {
#pragma unroll
                for (int m = 0; m < FN; ++m) {
                  const uint32_t s0 = sz[m][0], s1 = sz[m][1];
                  acc[u][m] = mfma32<MPS_TYPE_BF16>(sums[u], u32x4{s0 & 0xffff0000u, 0, s1 & 0xffff0000u, 0}, acc[u][m]);
                  acc[u][m] = mfma32<MPS_TYPE_BF16>(sums[u], u32x4{s0 << 16 | (s0 & 0xffffu), s0, s1 << 16 | (s1 & 0xffffu), s1}, acc[u][m]);
                  asm volatile("" : "+v"(acc[u][m]));
                }
              }
            }
          }
          if (slot == kMade + 1 && (kKnown >= 0 || pair + 1 < pairs)) {
            if ((place + 1) % H::kFour == 0) get_sums(four + 1);
            if (place + 1 == H::kPeriod && turns && a.zeros) get_zeros((pair + 1) / H::kPeriod);
          }
          // A stage before put_scales; a period of two stages has that in its first, so these are the one's after the next.
          if (slot == (FT == 1 ? 3 : 4) && place == 1 && turns) {
            const int32_t period = pair / H::kPeriod + (H::kPeriod == 4 ? 1 : 2);
            if (period * H::kPeriod < pairs) get_scales(period);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (fresh) {
#pragma unroll
        for (int n = 0; n < FN; ++n) pending[n] = scale[n];
      }
    }
    if constexpr (kOdd == 1) {
      static_assert(H::kLoads <= 4 * kM, "");
      const uint32_t last = here;
      here = then, then = after, after = last;
    }
  };
  int32_t pair = 0;
  auto stage = [&](int32_t pair, auto known) __attribute__((always_inline)) {
    body(pair, std::integral_constant<int, 0>{}, std::true_type{}, known);
    body(pair, std::integral_constant<int, 1>{}, std::true_type{}, known);
  };
#pragma unroll 1
  for (; 4 * (pair + H::kPeriod) + 8 <= blocks; pair += H::kPeriod) {  // the stages after their next are whole ones
    stage(pair, std::integral_constant<int, 0>{});
    stage(pair + 1, std::integral_constant<int, 1>{});
    if constexpr (H::kPeriod == 4) {
      stage(pair + 2, std::integral_constant<int, 2>{});
      stage(pair + 3, std::integral_constant<int, 3>{});
    }
  }
#pragma unroll 1
  for (; pair < pairs; ++pair) {
    body(pair, std::integral_constant<int, 0>{}, std::false_type{}, std::integral_constant<int, -1>{});
    body(pair, std::integral_constant<int, 1>{}, std::false_type{}, std::integral_constant<int, -1>{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads past the last stage
  bool finite = true;
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        acc[t][n][i] = __builtin_fmaf(pending[n], part[t][n][i], acc[t][n][i]);
        finite &= __builtin_fabsf(acc[t][n][i]) < __builtin_inff();
      }
  uint32_t *const flags = reinterpret_cast<uint32_t *>(ss);
  uint32_t again = 0;
  __syncthreads();
  flags[wave] = __any(!finite);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < H::kWaves; ++w) again |= flags[w];
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(again), 0)) {  // all again, a step at a time, with scales and zeros from memory
#pragma unroll
    for (int t = 0; t < FT; ++t)
#pragma unroll
      for (int n = 0; n < FN; ++n) acc[t][n] = f32x16{};
#pragma unroll 1
    for (int32_t step = 0; 2 * step < blocks; ++step) {
      const uint32_t at_step = step % 2 * H::kStep;
      __syncthreads();
      fetch_all(step / 2, 0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      read_w(fw[0], at_step);
#pragma unroll
      for (int h = 0; h < (C == kBlock ? 2 : 1); ++h) {
        if (2 * step + h >= blocks) break;
        const int32_t at = (2 * step + h) >> a.shift;
#pragma unroll
        for (int n = 0; n < FN; ++n)
#pragma unroll
          for (int t = 0; t < FT; ++t) part[t][n] = f32x16{};
#pragma unroll
        for (int q = C == kBlock ? 2 * h : 0; q < (C == kBlock ? 2 * h + 2 : 4); ++q) {
#pragma unroll
          for (int t = 0; t < FT; ++t) read_x(q, t, at_step);
#pragma unroll
          for (int n = 0; n < FN; ++n) {
            const u32x4 w = int4_values<XT>(fw[0][n][q], int4_zero(a, cols[n], at));
#pragma unroll
            for (int t = 0; t < FT; ++t) part[t][n] = mfma32<XT>(fx[q % H::kAhead][t], w, part[t][n]);
          }
        }
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          const float scale = int4_scale(a, cols[n], at);
#pragma unroll
          for (int t = 0; t < FT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][n][i] = __builtin_fmaf(scale, part[t][n][i], acc[t][n][i]);
        }
      }
    }
    __syncthreads();
  }

  // A lane's 16 sums are rows 8 i + 4 g .. + 3 of column r. The wave turns 32 rows at a time round through its own part
  // of LDS, so that a store has neighbouring columns.
  constexpr int kPitch = H::kPitch, kLanes = 4 * FN, kPasses = 32 * kLanes / 64;
  float *const mine = reinterpret_cast<float *>(lds) + wave * 32 * kPitch;
  const int32_t col = n0 + wn * FN * 32 + lane % kLanes * 8;
  f32x4 bias[2] = {};
  if (a.bias && !none) bias[0] = load_bias4(a, tile.expert, col), bias[1] = load_bias4(a, tile.expert, col + 4);
#pragma unroll
  for (int t = 0; t < FT; ++t) {
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mine[(8 * i + 4 * g + j) * kPitch + n * 32 + r] = acc[t][n][4 * i + j];
    __builtin_amdgcn_wave_barrier();
    f32x4 v[kPasses][2];
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[i][h] = *reinterpret_cast<const f32x4 *>(mine + (i * (64 / kLanes) + lane / kLanes) * kPitch + lane % kLanes * 8 + 4 * h) + bias[h];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int32_t row = tile.first + (wt * FT + t) * 32 + i * (64 / kLanes) + lane / kLanes;
      if (row < tile.end && col < a.n) store8(a, row, col, v[i][0], v[i][1]);
    }
  }
}

template <int XT, Chain C, int FT, int FN, int WT, int WN>
void launch(const Int4Args &a, hipStream_t stream) {
  typedef Shape<C, FT, FN, WT, WN> H;
  const int64_t tt = product_tiles(a, H::kBT), tn = (a.n + H::kBN - 1) / H::kBN;
  const int64_t grid = (tt * tn + 7) / 8 * 8;
  hipLaunchKernelGGL((int4_tile_kernel<XT, C, FT, FN, WT, WN>), dim3((unsigned)grid), dim3(H::kThreads), 0, stream, a, (int32_t)tt, (int32_t)tn);
}

// The tiles, in microseconds: `start` is what a tile takes at any k, `few` and `full` what k = 4096 adds to a tile that has a
// CU to itself, on a card with few of them and a full one, and `many` to each of several. Groups of 64 and of 32 cost more, and the first is not
// for groups of 32. The four in turn take, of groups of 128 (rows x k x n): 96 x 4096 x 14336 60, 43, 35, 35; 256 x 4096 x 4096 53, 34, 27, 23;
// 256 x 4096 x 14336 61, 47, 48, 63; 1024 x 4096 x 14336 143, 180, 163, 207; 4096 x 4096 x 14336 505, 610, 594, 769; of 64, 4096 x 4096 x 14336 594,
// 681, 685, 885; of 32, 256 x 4096 x 14336 -, 65, 67, 90; 1024 x 8192 x 28672 (FP16) -, 828, 842, 1122.
struct Choice {
  int32_t bt, bn;
  float start, few, full, many, step, block;
};
constexpr Choice kChoices[] = {{128, 256, 9.0f, 42.0f, 58.0f, 63.0f, 1.15f, 0.0f}, {64, 256, 7.0f, 25.0f, 41.0f, 34.4f, 1.15f, 1.55f},
                               {64, 128, 6.0f, 18.0f, 30.0f, 15.8f, 1.15f, 1.7f}, {32, 128, 5.0f, 16.0f, 18.5f, 8.5f, 1.15f, 1.5f}};

template <int XT, Chain C>
void launch_chain(const Int4Args &a, int choice, hipStream_t stream) {
  switch (choice) {
    case 0:
      if constexpr (C != kBlock) launch<XT, C, 4, 1, 1, 8>(a, stream);  // whose sums' two places LDS has no room for
      return;
    case 1: return launch<XT, C, 2, 1, 1, 8>(a, stream);
    case 2: return launch<XT, C, 2, 1, 1, 4>(a, stream);
    default: return launch<XT, C, 1, 1, 1, 4>(a, stream);
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

Prediction predict_int4_tiles(const Int4Args &a, int32_t cus) {
  Prediction best = {-1, 0};
  int i = 0;
  for (const Choice &c : kChoices) {
    const int at = i++;
    if (at == 0 && a.shift == 0) continue;
    if (((double)product_tiles(a, c.bt) * (double)((a.n + c.bn - 1) / c.bn) + 8) * 512 > kMostWorkItems) continue;
    const double tiles = expected_tiles(a, c.bt) * (double)((a.n + c.bn - 1) / c.bn) / cus;
    const double k = a.row_blocks / 128.0 * (a.shift == 0 ? c.block : a.shift == 1 ? c.step : 1.0f);
    // The count of experts' tiles is a guess: the mean over a tenth less and more, lest another round of a few tiles comes
    // unawares. Experts' weights are no other tile's, and come later.
    const double start = c.start + (a.offsets ? 3.5 : 0), spread = a.offsets ? 0.1 : 0;
    double us = 0;
    for (int j = -1; j <= 1; ++j) {
      const double n = tiles * (1 + spread * j), each = __builtin_ceil(n - 0.01);
      us += (each <= 1 ? start + (c.few + (c.full - c.few) * n) * k : each * (start + c.many * k)) / 3;
    }
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
