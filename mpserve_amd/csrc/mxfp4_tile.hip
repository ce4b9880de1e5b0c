// Products of many rows: tiles of BT rows of x times BN weight rows, with both operands' pieces of
// k staged in LDS.
//
// A step covers 128 bytes of every row of x, a cache line: 64 elements of 16 bits or 256 codes. The
// weights of a step are 32 bytes a row beside 16-bit x (widened in registers, after LDS) and 128
// beside MXFP4 x, which the matrix cores multiply as it is. Pieces of 16 bytes go from memory to LDS
// without passing through registers; piece p of row r lies at place p ^ (r / 2 % 8) of its row's
// eight, or p ^ (r / 8 % 2) of two: the sixteen lanes that LDS serves in a cycle (0-3, 12-15, 20-27
// and 4-11, 16-19, 28-31, and so on) then meet all 64 banks once. With r % 8 half of LDS's cycles
// were conflicts. (Stages of 64 bytes a row, four of them, halve the lines' use: 1177 us for 8192 x
// 8192 x 28672 where these took 1030 then.)
//
// A step is multiplied in quarters, each from fragments read during the one before. Once the last
// quarter's fragments are read nobody needs the buffer any more: the barrier stands there, the
// loads of the step after next are issued among that quarter's products, and the next step's first
// fragments are read there too, so that the matrix cores do not wait for a new buffer. (All loads before
// the quarter: BF16 4096 x 4096 x 14336 411 us where these take 403, MXFP4 alike. Two barriers a
// step, one for each half of x's rows, give loads half a step more to arrive and took 3 % longer.)
//
// What bounds it: the matrix cores, at clocks that the load brings down. BF16 4096 x 4096 x 14336 takes 391 to
// 417 us, 1.15 to 1.23 PFLOP/s, with the matrix cores busy for 64 % of the cycles; the library's product with a BF16
// weight [n, k] takes 326 to 368 on the same cards, with one [k, n] 395 where this took 391. MXFP4 8192 x 8192 x
// 28672 takes 970 to 1010 us, 3.8 to 4.0 PFLOP/s, busy for 56 %; at 955, no loads to LDS and no barriers would have
// made it 770, no stores 870.
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
  static constexpr int kWaves = WT * WN, kThreads = kWaves * 64;
  static constexpr int kWPieces = k4 ? 8 : 2;                    // a weight row and step; x has 8
  static constexpr int kXLoads = BT * 8 / kThreads;              // loads a wave and step, 64 pieces each
  static constexpr int kWLoads = (BN * kWPieces + kThreads - 1) / kThreads;
  static constexpr int kWLanes = BN * kWPieces / kWaves < 64 ? BN * kWPieces / kWaves : 64;  // that load
  static constexpr int kSteps = k4 ? 2 : 8;                      // steps a period of 16 blocks
  static constexpr int kScaleRows = k4 ? BT + BN : BN;           // x's rows, then the weight's
  static constexpr int kSLoads = (kScaleRows + kThreads - 1) / kThreads;
  static constexpr int kFT = BT / WT / 32, kFN = BN / WN / 32;   // 32 x 32 fragments of a wave
  static constexpr int kXBytes = BT * 128, kWBytes = BN * kWPieces * 16, kSBytes = kScaleRows * 16;
  static constexpr int kPitch = kFN * 32 + 4;                    // floats of a row of sums, turned round
  static constexpr int kStaged = 2 * (kXBytes + kWBytes + kSBytes), kTurned = kWaves * 32 * kPitch * 4;
  static constexpr int kFlags = kStaged > kTurned ? kStaged : kTurned;  // a word a wave
  static constexpr int kLds = kFlags + (XT == MPS_TYPE_BF16 ? kWaves * 4 : 0);
  static_assert(BT * 8 % kThreads == 0 && kThreads % 128 == 0 && kLds <= 160 * 1024, "");
};

template <int XT, int BT, int BN, int WT, int WN>
__global__ __launch_bounds__(WT *WN * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void mxfp4_tile_kernel(ProductArgs a, int32_t tiles_t, int32_t tiles_n) {
  typedef Shape<XT, BT, BN, WT, WN> S;
  constexpr bool k4 = S::k4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kLds];
  uint8_t *const xs = lds, *const ws = lds + 2 * S::kXBytes, *const ss = ws + 2 * S::kWBytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, g = lane >> 5;
  const int wt = wave / WN, wn = wave % WN;

  if (a.offsets) tiles_t = count_tiles(a.offsets, a.experts, a.rows, BT);  // the host knows a bound only
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
  const int32_t blocks = a.row_blocks, periods = none ? 0 : (blocks + 15) / 16;

  // Where this lane's pieces come from. Rows past the tile's end or the weight's are read from
  // the last one (what they give is not stored), pieces past a row's end from its last one; their
  // scales are zeros. MXFP4 x and the weights lie row by row, so an offset from the tile's
  // first row, cut at the last, finds every piece; gathered rows need an address each.
  const int64_t x_row_bytes = k4 ? (int64_t)blocks * 16 : a.x_stride * 2;
  const uint32_t w_row_bytes = (uint32_t)blocks * 16;
  const int w_first_piece = wave * S::kWLanes + lane;  // of the first load's
  const int xrow = tid / 8, wrow = w_first_piece / S::kWPieces;
  const int32_t x_piece = (tid % 8) ^ (xrow >> 1 & 7);
  const int32_t w_piece = k4 ? (w_first_piece % 8) ^ (wrow >> 1 & 7) : (w_first_piece % 2) ^ (wrow >> 3 & 1);
  const int64_t w_first = (int64_t)(none ? 0 : tile.expert) * a.n + n0;
  const uint8_t *const w_base = a.w + w_first * w_row_bytes;
  const uint32_t w_last = (uint32_t)min(BN - 1, a.n - 1 - n0) * w_row_bytes;
  const uint32_t x_last = (uint32_t)(tile.end - 1 - tile.first) * (uint32_t)x_row_bytes;
  const uint8_t *const x_base = static_cast<const uint8_t *>(a.x) + tile.first * x_row_bytes;
  const uint8_t *x_from[k4 ? 1 : S::kXLoads];
  if constexpr (!k4) {
#pragma unroll
    for (int i = 0; i < S::kXLoads; ++i) {
      int32_t from = min(tile.first + xrow + i * (S::kThreads / 8), tile.end - 1);
      if (a.gather) from = min((uint32_t)a.order[from] / (uint32_t)a.top, (uint32_t)a.x_rows - 1);
      x_from[i] = static_cast<const uint8_t *>(a.x) + from * x_row_bytes;
    }
  }
  const uint8_t *s_from[S::kSLoads];
  const bool has_scales = S::kScaleRows % S::kThreads == 0 || tid < S::kScaleRows;
#pragma unroll
  for (int i = 0; i < S::kSLoads; ++i) {
    const int at = tid + i * S::kThreads, row = k4 ? at - BT : at;
    if (k4 && row < 0)
      s_from[i] = a.x_scales + (int64_t)min(tile.first + at, tile.end - 1) * blocks;
    else
      s_from[i] = a.w_scales + (w_first + min(min(row, BN - 1), a.n - 1 - n0)) * blocks;
  }
  const int32_t x_pieces = k4 ? blocks : blocks * 4;
  // Loads `from` to `to` of a step, x's before the weights'.
  constexpr int kLoads = S::kXLoads + S::kWLoads;
  auto fetch = [&](int32_t step, int buffer, int from, int to) {
    uint8_t *const xt = xs + buffer * S::kXBytes + wave * 1024, *const wt = ws + buffer * S::kWBytes + wave * S::kWLanes * 16;
    const uint32_t x_at = (uint32_t)min(step * 8 + x_piece, x_pieces - 1) * 16;
    const uint32_t w_at = (uint32_t)min(step * S::kWPieces + w_piece, blocks - 1) * 16;
#pragma unroll
    for (int l = from; l < to; ++l) {
      const int i = l < S::kXLoads ? l : l - S::kXLoads;
      if (l >= S::kXLoads) {
        if (S::kWLanes == 64 || lane < S::kWLanes)
          copy16(w_base + (min((uint32_t)(wrow + i * (S::kThreads / S::kWPieces)) * w_row_bytes, w_last) + w_at), wt + i * S::kThreads * 16);
      } else if constexpr (k4) {
        copy16(x_base + (min((uint32_t)(xrow + i * (S::kThreads / 8)) * (uint32_t)x_row_bytes, x_last) + x_at), xt + i * S::kThreads * 16);
      } else {
        copy16(x_from[i] + x_at, xt + i * S::kThreads * 16);
      }
    }
  };
  // Scales come 16 blocks at a time, a period ahead, through registers.
  u32x4 scales[S::kSLoads] = {};
  auto get_scales = [&](int32_t period) {
    if (has_scales) {
#pragma unroll
      for (int i = 0; i < S::kSLoads; ++i) scales[i] = load_scales(s_from[i], 16 * period, blocks);
    }
  };
  auto put_scales = [&](int32_t period, int buffer) {
    if (has_scales) {
#pragma unroll
      for (int i = 0; i < S::kSLoads; ++i)
        *reinterpret_cast<u32x4 *>(ss + buffer * S::kSBytes + (tid + i * S::kThreads) * 16) = move_scales(scales[i], 16 * period, blocks);
    }
    if constexpr (XT == MPS_TYPE_BF16) {
#pragma unroll
      for (int i = 0; i < S::kSLoads; ++i) asm volatile("" : "+v"(scales[i]));  // are there, for all waves: waited for here, not below
    }
  };
  // BF16: a wave that meets a large scale says so in LDS, by the next barrier.
  uint32_t *const flags = reinterpret_cast<uint32_t *>(lds + S::kFlags);
  auto note_scales = [&]() {
    if constexpr (XT == MPS_TYPE_BF16) {
      uint32_t large = 0;
#pragma unroll
      for (int i = 0; i < S::kSLoads; ++i) large |= large_scales(scales[i]);
      if (__builtin_expect(__any(large & kLargeScale), 0)) flags[wave] = 1;
    }
  };

  // Fragments of x by quarter. MXFP4: lanes 0-31 take the step's first four blocks of k, 32-63 the
  // others, one a quarter, so that their scales are a word of neighbouring bytes. 16 bits: half a
  // step is a block, of which lanes 0-31 take the first pieces of codes and 32-63 the others, and a quarter
  // half of these.
  constexpr int kBuffers = XT == MPS_TYPE_F16 ? 4 : 2;
  u32x4 fx[kBuffers][S::kFT];
  u32x4 fw4[2][k4 ? S::kFN : 1];               // MXFP4: by quarter
  uint64_t fw[2][S::kFN];                      // 16 bits: by half
  uint32_t sx[2][k4 ? S::kFT : 1], sw[2][S::kFN];  // scales: MXFP4 by step, 16 bits by half
  f32x16 acc[S::kFT][S::kFN] = {};
  const uint8_t *const xl = xs + (wt * S::kFT * 32 + r) * 128, *const wl = ws + (wn * S::kFN * 32 + r) * S::kWPieces * 16;
  const uint8_t *const sl = ss + r * 16;
  // Quarter q of the step in `buffer`, the in-th of its period.
  auto read = [&](auto tc, int q, int buffer, int in, int sbuf) {
    constexpr int kFT = decltype(tc)::value;
    const int at = ((k4 ? 4 * g + q : 4 * (q >> 1) + 2 * g + (q & 1)) ^ (r >> 1 & 7)) * 16;
    if constexpr (k4) {
#pragma unroll
      for (int n = 0; n < S::kFN; ++n) fw4[q & 1][n] = *reinterpret_cast<const u32x4 *>(wl + buffer * S::kWBytes + n * 32 * 128 + at);
      if (q == 0) {
#pragma unroll
        for (int t = 0; t < kFT; ++t)
          sx[in & 1][t] = *reinterpret_cast<const uint32_t *>(sl + sbuf * S::kSBytes + (wt * S::kFT + t) * 32 * 16 + in * 8 + g * 4);
#pragma unroll
        for (int n = 0; n < S::kFN; ++n)
          sw[in & 1][n] = *reinterpret_cast<const uint32_t *>(sl + sbuf * S::kSBytes + (BT + (wn * S::kFN + n) * 32) * 16 + in * 8 + g * 4);
      }
    } else if (q % 2 == 0) {
#pragma unroll
      for (int n = 0; n < S::kFN; ++n) {
        fw[q >> 1][n] = *reinterpret_cast<const uint64_t *>(wl + buffer * S::kWBytes + n * 32 * 32 + ((q >> 1) ^ (r >> 3 & 1)) * 16 + g * 8);
        sw[q >> 1][n] = sl[sbuf * S::kSBytes + (wn * S::kFN + n) * 32 * 16 + in * 2 + (q >> 1)];
      }
    }
#pragma unroll
    for (int t = 0; t < kFT; ++t)
      fx[q % kBuffers][t] = *reinterpret_cast<const u32x4 *>(xl + buffer * S::kXBytes + t * 32 * 128 + at);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](auto tc, auto qc, int in, int from, int to) {
    constexpr int q = decltype(qc)::value, kFT = decltype(tc)::value;
#pragma unroll
    for (int n = from; n < to; ++n) {
      if constexpr (k4) {
#pragma unroll
        for (int t = 0; t < kFT; ++t)
          acc[t][n] = multiply4<q>(__builtin_bit_cast(i32x4, fw4[q & 1][n]), sw[in & 1][n], __builtin_bit_cast(i32x4, fx[q % kBuffers][t]),
                                   sx[in & 1][t], acc[t][n]);
      } else if constexpr (XT == MPS_TYPE_BF16) {
        const bf16x8 w = widen((uint32_t)(fw[q >> 1][n] >> (32 * (q & 1))), mx_scale(sw[q >> 1][n]));
#pragma unroll
        for (int t = 0; t < kFT; ++t)
          acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, __builtin_bit_cast(bf16x8, fx[q % kBuffers][t]), acc[t][n], 0, 0, 0);
      } else if constexpr (q % 2 == 1) {
        // FP16: both quarters of a block, summed without the scale, which FP16 weights could not hold.
        const f16x8 w0 = widen_f16((uint32_t)fw[q >> 1][n]), w1 = widen_f16((uint32_t)(fw[q >> 1][n] >> 32));
        const float scale = mx_scale_value(sw[q >> 1][n]);
#pragma unroll
        for (int t = 0; t < kFT; ++t) {
          f32x16 part = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fx[q - 1][t]), w0, f32x16{}, 0, 0, 0);
          part = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fx[q][t]), w1, part, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][n][i] = __builtin_fmaf(scale, part[i], acc[t][n][i]);
        }
      }
    }
    // The products stay where they are.
#pragma unroll
    for (int t = 0; t < kFT; ++t)
#pragma unroll
      for (int n = from; n < to; ++n) asm volatile("" : "+v"(acc[t][n]));
    __builtin_amdgcn_sched_barrier(0);
  };

  auto run = [&](auto tc) {
    if (periods > 0) {
      fetch(0, 0, 0, kLoads);
      get_scales(0);
      if constexpr (XT == MPS_TYPE_BF16) flags[wave] = 0;
      put_scales(0, 0);
      note_scales();
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      fetch(1, 1, 0, kLoads);
      read(tc, 0, 0, 0, 0);
      if constexpr (XT == MPS_TYPE_F16) read(tc, 1, 0, 0, 0);
    }
    // 16 bits: steps past the last are left out, and so is a last block's other half; MXFP4 multiplies them
    // by zero scales.
    const int32_t halves = k4 ? 0 : blocks;
    for (int32_t p = 0; p < periods; ++p) {
      const int sbuf = p & 1;
      if (p + 1 < periods) get_scales(p + 1);
      const int32_t left = blocks - 16 * p;
#pragma unroll
      for (int32_t pair = 0; pair < S::kSteps / 2; ++pair) {  // of steps
        if (pair * (2 * 16 / S::kSteps) >= left) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int32_t in = 2 * pair + i, step = p * S::kSteps + in;
          const bool has[2] = {k4 || 2 * step < halves, k4 || 2 * step + 1 < halves};
          const int32_t next = in + 1 == S::kSteps ? 0 : in + 1;
          const int next_sbuf = next == 0 ? sbuf ^ 1 : sbuf;
          // The next fragments are read between the products of the weights' first fragment and the
          // others': read before them all, they would be waited for together with these.
          auto quarter = [&](auto qc) {
            constexpr int q = decltype(qc)::value;
            if (has[q >> 1]) multiply(tc, qc, in, 0, 1);
            if constexpr (q == 3) {
              read(tc, 0, i ^ 1, next, next_sbuf);
              if constexpr (XT == MPS_TYPE_F16) read(tc, 1, i ^ 1, next, next_sbuf);
            } else if constexpr (XT == MPS_TYPE_F16) {
              read(tc, 2, i, in, sbuf);
              read(tc, 3, i, in, sbuf);
            } else {
              read(tc, q + 1, i, in, sbuf);
            }
            if constexpr (q == 3) {
              fetch(step + 2, i, 0, kLoads / 2);
              __builtin_amdgcn_sched_barrier(0);
            }
            if (has[q >> 1]) multiply(tc, qc, in, 1, S::kFN);
            if constexpr (q == 3) fetch(step + 2, i, kLoads / 2, kLoads);
          };
          if constexpr (XT != MPS_TYPE_F16) quarter(std::integral_constant<int, 0>{});
          quarter(std::integral_constant<int, 1>{});
          if constexpr (XT != MPS_TYPE_F16) quarter(std::integral_constant<int, 2>{});
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
          if (in == S::kSteps - 2) put_scales(p + 1, sbuf ^ 1);
          quarter(std::integral_constant<int, 3>{});
          if (in == S::kSteps - 2) note_scales();
        }
      }
    }
  };
  // A tile with rows in its first half only, as half of the experts' last ones are, skips the others' products
  // (64 experts, four each of 8192 tokens, 4096 -> 2048: 597 us without, 587 so; 128 experts, eight each of
  // 3000 tokens, 1024 -> 4096 in FP16: 447 and 425).
  if constexpr (WT == 1 && S::kFT > 1) {
    if (tile.end - tile.first <= BT / 2)
      run(std::integral_constant<int, S::kFT / 2>{});
    else
      run(std::integral_constant<int, S::kFT>{});
  } else {
    run(std::integral_constant<int, S::kFT>{});
  }

  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads of steps past the last
  if constexpr (XT == MPS_TYPE_BF16) {
    uint32_t any = 0;
    if (periods > 0)
      for (int w = 0; w < S::kWaves; ++w) any |= flags[w];
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(any) != 0, 0)) {  // alike in all waves: a product could have overflowed
#pragma unroll
      for (int t = 0; t < S::kFT; ++t)
#pragma unroll
        for (int n = 0; n < S::kFN; ++n) acc[t][n] = f32x16{};
#pragma unroll 1
      for (int32_t step = 0; 2 * step < blocks; ++step) {  // all again, one at a time, with scales from memory
        __syncthreads();
        fetch(step, 0, 0, kLoads);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int32_t block = 2 * step + (q >> 1);
          if (block >= blocks) break;
          read(std::integral_constant<int, S::kFT>{}, q, 0, 0, 0);
          if (q % 2 == 0) {
#pragma unroll
            for (int n = 0; n < S::kFN; ++n)
              sw[q >> 1][n] = a.w_scales[(w_first + min((wn * S::kFN + n) * 32 + r, a.n - 1 - n0)) * blocks + block];
          }
#pragma unroll
          for (int n = 0; n < S::kFN; ++n) {
            const bf16x8 w = widen_quarter((uint32_t)(fw[q >> 1][n] >> (32 * (q & 1))), sw[q >> 1][n]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int t = 0; t < S::kFT; ++t)
                acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, __builtin_bit_cast(bf16x8, fx[q % kBuffers][t]), acc[t][n], 0, 0, 0);
          }
        }
      }
    }
  }
  if constexpr (XT != MPS_TYPE_BF16) {
    // A lane's 16 sums are places 8 i + 4 g .. + 3 of one side of a fragment, at place r of the other: columns
    // of one row, or with FP16 x rows of one column. The wave turns 32 rows at a time round through
    // its own part of LDS, so that a store has whole lines (MXFP4 8192 x 512 x 8192: 56 us as below, 43 so;
    // BF16, whose shorter tiles end at different times, 460 as below for k = 4096 and 466 so).
    __syncthreads();
    constexpr int kCols = S::kFN * 32, kPitch = S::kPitch, kLanes = kCols / 8, kPasses = 32 * kLanes / 64;
    float *mine = reinterpret_cast<float *>(lds) + wave * 32 * kPitch;
    const int32_t col = n0 + wn * kCols + lane % kLanes * 8;
    f32x4 bias[2] = {};
    if (a.bias && !none) bias[0] = load_bias4(a, tile.expert, col), bias[1] = load_bias4(a, tile.expert, col + 4);
#pragma unroll
    for (int t = 0; t < S::kFT; ++t) {
#pragma unroll
      for (int n = 0; n < S::kFN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (k4) {
            *reinterpret_cast<f32x4 *>(mine + r * kPitch + n * 32 + 8 * i + 4 * g) =
                f32x4{acc[t][n][4 * i], acc[t][n][4 * i + 1], acc[t][n][4 * i + 2], acc[t][n][4 * i + 3]};
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[(8 * i + 4 * g + j) * kPitch + n * 32 + r] = acc[t][n][4 * i + j];
          }
        }
      __builtin_amdgcn_wave_barrier();
      f32x4 v[kPasses][2];
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[i][h] = *reinterpret_cast<const f32x4 *>(mine + (i * (64 / kLanes) + lane / kLanes) * kPitch + lane % kLanes * 8 + 4 * h) + bias[h];
      __builtin_amdgcn_wave_barrier();
      const int32_t row = tile.first + (wt * S::kFT + t) * 32 + lane / kLanes;
      auto store = [&](auto typed) {  // whole 16-byte pieces of a known type
        uint16_t *to = static_cast<uint16_t *>(a.out) + (int64_t)row * a.n + col;
#pragma unroll
        for (int i = 0; i < kPasses; ++i, to += (int64_t)(64 / kLanes) * a.n) {
          const f32x4 lo = v[i][0], hi = v[i][1];
          constexpr int32_t type = decltype(typed)::value;
          const u32x4 piece = {pack2(lo[0], lo[1], type), pack2(lo[2], lo[3], type), pack2(hi[0], hi[1], type), pack2(hi[2], hi[3], type)};
          if (row + i * (64 / kLanes) < tile.end) *reinterpret_cast<u32x4_any *>(to) = piece;
        }
      };
      if (a.out_type == MPS_TYPE_BF16 && n0 + BN <= a.n) {
        store(std::integral_constant<int32_t, MPS_TYPE_BF16>{});
      } else if (a.out_type == MPS_TYPE_F16 && n0 + BN <= a.n) {
        store(std::integral_constant<int32_t, MPS_TYPE_F16>{});
      } else {
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
          if (row + i * (64 / kLanes) < tile.end) store8(a, row + i * (64 / kLanes), col, v[i][0], v[i][1]);
      }
    }
  } else {
    // A lane's 16 sums are columns 8 i + 4 g .. + 3 of row r of a fragment. For 16-bit outputs lanes r and
    // r + 32 trade, so that each has eight neighbouring columns.
    const bool wide = a.out_type != MPS_TYPE_F32;
#pragma unroll
    for (int n = 0; n < S::kFN; ++n) {
      const int32_t col = n0 + (wn * S::kFN + n) * 32;
      if (a.bias && !none) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 bias = load_bias4(a, tile.expert, col + 8 * i + 4 * g);
#pragma unroll
          for (int t = 0; t < S::kFT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][n][4 * i + j] += bias[j];
        }
      }
#pragma unroll
      for (int t = 0; t < S::kFT; ++t) {
        const int32_t row = tile.first + (wt * S::kFT + t) * 32 + r;
        if (wide) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = pack2(acc[t][n][8 * i + 2 * j], acc[t][n][8 * i + 2 * j + 1], a.out_type);
            const auto lo = __builtin_amdgcn_permlane32_swap(p[0], p[2], false, false);
            const auto hi = __builtin_amdgcn_permlane32_swap(p[1], p[3], false, false);
            const int32_t at = col + 16 * i + 8 * g;
            const u32x4 v = {lo[0], hi[0], lo[1], hi[1]};
            uint16_t *const to = static_cast<uint16_t *>(a.out) + (int64_t)row * a.n + at;
            if (row < tile.end && at + 8 <= a.n) {
              *reinterpret_cast<u32x4_any *>(to) = v;
            } else if (row < tile.end) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (at + j < a.n) to[j] = (uint16_t)(v[j / 2] >> (16 * (j % 2)));
            }
          }
        } else if (row < tile.end) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t at = col + 8 * i + 4 * g;
            if (at < a.n)
              store4(a, row, at, f32x4{acc[t][n][4 * i], acc[t][n][4 * i + 1], acc[t][n][4 * i + 2], acc[t][n][4 * i + 3]});
          }
        }
      }
    }
  }
}

template <int XT, int BT, int BN, int WT, int WN>
void launch(const ProductArgs &a, hipStream_t stream) {
  const int64_t tt = product_tiles(a, BT), tn = (a.n + BN - 1) / BN;
  const int64_t grid = (tt * tn + 7) / 8 * 8;
  hipLaunchKernelGGL((mxfp4_tile_kernel<XT, BT, BN, WT, WN>), dim3((unsigned)grid), dim3(WT * WN * 64), 0, stream, a,
                     (int32_t)tt, (int32_t)tn);
}

// The tiles, in microseconds. `start` is what a tile takes at any k, for its first loads and its stores
// (8192 x 32 x 8192); `one` and `many` are what k = 4096 adds to a tile that has a CU to itself (128 x 8192 x
// 8192 and 1024 x 4096 x 4096) and to each of several (4096 x 4096 x 14336). So BF16 4096 x 4096 x 14336 takes
// 128 x 256 tiles, 395 us where 128 x 128 take 450, and for 512 x 2048 x 1024 the least of the tiles are 64 x 64, 13 us
// where 128 x 256 take 31 and the kernel of few rows, which is taken, 7. (BF16 in tiles of 256 x 256, one workgroup of eight waves a CU: 417 us; MXFP4 in 128 x
// 256, 16 % slower than 256 x 256.) `half` is the share that one of several tiles spares if its rows are in
// its first half only (2400 rows spread evenly over 64 experts, 4096 x 2048, in BF16: 86 to 95 us in 128 x 256, 108 in
// 64 x 128; a router that likes some experts more, which the host cannot know, makes it 147 to 160 and 132).
struct Choice {
  int32_t bt, bn;
  float start, one, many, half;
};
constexpr Choice kChoices4[] = {{256, 256, 10.5f, 18.0f, 27.0f, 0}, {128, 128, 3.0f, 11.0f, 8.5f, 0}, {64, 64, 1.5f, 8.9f, 4.2f, 0}};
constexpr Choice kChoicesBf16[] = {
    {128, 256, 4.6f, 51.0f, 53.0f, 0.35f}, {128, 128, 2.6f, 35.0f, 30.0f, 0}, {64, 128, 1.8f, 26.0f, 18.5f, 0}, {64, 64, 1.45f, 24.5f, 13.4f, 0}};
constexpr Choice kChoicesF16[] = {{128, 128, 2.7f, 49.0f, 37.5f, 0.35f}, {64, 128, 1.8f, 33.0f, 21.1f, 0}, {64, 64, 1.4f, 27.5f, 14.2f, 0}};

template <int N>
Prediction least(const ProductArgs &a, const Choice (&choices)[N], int32_t cus) {
  Prediction best = {-1, 0};
  for (int i = 0; i < N; ++i) {
    const Choice &c = choices[i];
    if (((double)product_tiles(a, c.bt) * (double)((a.n + c.bn - 1) / c.bn) + 8) * 512 > kMostWorkItems) continue;
    const double tiles = expected_tiles(a, c.bt) * (double)((a.n + c.bn - 1) / c.bn) / cus, k = a.row_blocks / 128.0;
    // The count of experts' tiles is a guess, unless most have one: the mean over a tenth less and more, lest a
    // second round of a few tiles comes unawares (1872 rows of 60 experts, k = 5016, n = 896, had 264 for 256
    // CUs). Experts' weights are no other tile's, and come later (`start` by 3.5 us: 64 x 64 and 64 x 128
    // take 151 and 96 us for 1200 rows spread evenly over 64 experts, 4096 x 2048, where 119 and 81 would follow).
    const bool sure = a.rows >= 4.0 * a.experts && a.rows <= 0.6 * c.bt * a.experts;
    const double start = c.start + (a.offsets ? 3.5 : 0), spread = a.offsets && !sure ? 0.1 : 0;
    const double whole = 1 - c.half * expected_halves(a, c.bt);
    double us = 0;
    for (int j = -1; j <= 1; ++j) {
      const double each = __builtin_ceil(tiles * (1 + spread * j) - 0.01);
      us += (each <= 1 ? start + c.one * k : each * (start + c.many * k) * whole) / 3;
    }
    if (best.choice < 0 || us < best.us) best = {i, us};
  }
  return best;
}

}  // namespace

Prediction predict_tiles(const ProductArgs &a, int32_t x_type, int32_t cus) {
  if (x_type == MPS_TYPE_MXFP4) return least(a, kChoices4, cus);
  return x_type == MPS_TYPE_BF16 ? least(a, kChoicesBf16, cus) : least(a, kChoicesF16, cus);
}

void launch_tiles(const ProductArgs &a, int32_t x_type, int choice, hipStream_t stream) {
  if (x_type == MPS_TYPE_MXFP4) {
    switch (choice) {
      case 0: return launch<MPS_TYPE_MXFP4, 256, 256, 2, 4>(a, stream);
      case 1: return launch<MPS_TYPE_MXFP4, 128, 128, 2, 2>(a, stream);
      default: return launch<MPS_TYPE_MXFP4, 64, 64, 2, 2>(a, stream);
    }
  }
  if (x_type == MPS_TYPE_BF16) {
    switch (choice) {
      case 0: return launch<MPS_TYPE_BF16, 128, 256, 1, 4>(a, stream);
      case 1: return launch<MPS_TYPE_BF16, 128, 128, 2, 2>(a, stream);
      case 2: return launch<MPS_TYPE_BF16, 64, 128, 1, 4>(a, stream);
      default: return launch<MPS_TYPE_BF16, 64, 64, 2, 2>(a, stream);
    }
  }
  switch (choice) {
    case 0: return launch<MPS_TYPE_F16, 128, 128, 1, 4>(a, stream);
    case 1: return launch<MPS_TYPE_F16, 64, 128, 1, 4>(a, stream);
    default: return launch<MPS_TYPE_F16, 64, 64, 2, 2>(a, stream);
  }
}

}  // namespace mps
