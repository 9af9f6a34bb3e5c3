// Low-rank adapters of many requests beside a shared projection: with l the adapter of row t,
//
//   v[t] = a_l x[t]   (a_l: rank x hidden_in)        out[t] = base[t] + scale_l * b_l v[t]   (b_l: hidden_out x rank)
//
// Bound by base and out for many rows, by the adapters' weights for rows of many adapters, and by the latencies of two launches for few.
// 8192 rows of prompts, bf16, 4096 -> 14336: rank 64 42 + 143 us (556 MB in all; the second kernel moves 470 MB of base and out at 3.3 TB/s, and
// reads as much of b_l again from the L2s, 64 rows at a time: with one adapter 127 us; vector instructions are in 16 % of its cycles, and a block's
// loads stand behind the stores of the one before it), rank 16, 4096 wide 21 + 34 us (134 MB: 4.0 TB/s, as a
// copy), rank 8 19 + 35.  64 rows of 16 adapters, rank 16, 4096 wide 4.9 + 5.1 us, one row 4.0 + 5.0.  The second kernel spills
// 4 to 18 words of ranks 17 to 64 (four waves to a SIMD leave 128 registers): none of them is read in the loop over whole blocks.
// Rows are taken in windows of 64 in their own order, and the rows of a window that share an adapter together: the
// rows of a prompt are neighbours, and the rows of a decode step are one window, so nothing has to be sorted.  A wave knows
// its window's rows from one load and a ballot for each adapter.
//
// v is kept in fp32, summed over pieces of the depth by its readers, and split there into two numbers of the
// element type (high, and what its rounding left), each multiplied by b_l: v is exact to twice the bits of the type, in float16 to 2^-38 of its
// row's largest.
#include "operators.hpp"

#include <math.h>

#include <algorithm>

#include "few_rows.hpp"
#include "gmm_kernel.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kWindow = 64;

// The adapters of a window in the order of their first rows, with the rows of each as a mask.  The first kernel writes it for the second.
struct WindowPlan {
  int32_t count;
  int32_t pieces;          // of the depth, into which v of these rows is cut
  uint64_t none;           // rows without an adapter
  uint64_t rows[kWindow];
  int32_t adapter[kWindow];
};

struct AdapterParams {
  AdapterArgs a;
  float* v;            // [pieces][rows][v_pitch]
  WindowPlan* plans;   // [windows]
  int32_t v_pitch;
  int32_t pieces;      // of the depth hidden_in, at most
  int32_t shares;      // workgroups of a window
};

// The same from the rows' adapters, in the lanes of a wave.
struct Window {
  int32_t adapter;    // of this lane's row, -1 without one
  uint64_t left;      // rows not yet taken
  uint64_t none;

  __device__ __forceinline__ Window(const AdapterArgs& a, int64_t first) {
    const int lane = threadIdx.x & 63, rows = (int)(a.rows - first < kWindow ? a.rows - first : kWindow);
    adapter = lane < rows ? a.adapters[first + lane] : -1;
    if ((uint32_t)adapter >= (uint32_t)a.num) adapter = -1;
    left = __ballot(adapter >= 0);
    none = __ballot(lane < rows && adapter < 0);
  }
  // The next adapter and its rows; left must not be 0.
  __device__ __forceinline__ uint64_t next(int& which) {
    which = __builtin_amdgcn_readlane(adapter, __ffsll((unsigned long long)left) - 1);
    const uint64_t mine = __ballot(adapter == which);
    left &= ~mine;
    return mine;
  }
};

// Lane i gets the number of the i-th row of `mine` in its window (lanes past the last: any).
__device__ __forceinline__ int list_rows(uint64_t mine) {
  const int lane = threadIdx.x & 63, count = __popcll(mine);
  const int before = __popcll(mine & ((uint64_t(1) << lane) - 1));
  const bool in = (mine >> lane) & 1;
  // (the rows of the mask go to the first lanes, the others behind them: every lane is written once)
  return __builtin_amdgcn_ds_permute(4 * (in ? before : count + lane - before), lane);
}

// v of one piece of the depth.  TILES: of 16 rows of a_l; more than 64 of them are taken 64 at a time.
// MT: of 16 rows, taken at a time (1 and 2, us: 64 rows of one adapter, rank 64, 15.0, 12.4; decode, a row or two to an adapter, 8.3, 8.4; one row 3.9, 4.1;
// 8192 rows of prompts 59, 41).
template <int DT, int TILES, bool ODD>
__global__ __launch_bounds__(kFewThreads, 2) void adapter_shrink_kernel(AdapterParams p) {
  constexpr int MT = 2;
  using S = Stream<DT, true, TILES, MT, ODD>;
  __shared__ f32x4 lds[kFewWaves * 256];
  const AdapterArgs& a = p.a;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int64_t window = blockIdx.x / p.shares, first = window * kWindow;
  const int share = (int)(blockIdx.x - window * p.shares);
  Window w(a, first);
  // What is in the window, the i-th adapter and its rows in lane i: the workgroups that its adapters leave cut the depth.
  int count = 0, its_adapter = 0;
  uint64_t its_rows = 0;
  for (; w.left != 0; ++count) {
    int which;
    const uint64_t mine = w.next(which);
    if (lane == count) its_adapter = which, its_rows = mine;
  }
  const int pieces = min(max(p.shares / max(count, 1), 1), p.pieces), splits = p.shares / pieces;
  if (share == 0 && threadIdx.x < kWindow) {
    WindowPlan& plan = p.plans[window];
    plan.adapter[lane] = its_adapter, plan.rows[lane] = its_rows;
    if (lane == 0) plan.count = count, plan.pieces = pieces, plan.none = w.none;
  }
  const int piece = share % pieces, split = share / pieces;
  if (split >= splits) return;
  const int steps = (a.hidden_in + S::DEPTH - 1) / S::DEPTH;
  const int begin = (int)((int64_t)steps * piece / pieces), end = (int)((int64_t)steps * (piece + 1) / pieces);
  float* v = p.v + (uint64_t)piece * a.rows * p.v_pitch;
  S s;
  s.depth = a.hidden_in;
  s.width = 8;
  s.x = static_cast<const uint16_t*>(a.x) + (uint64_t)first * a.hidden_in;
  const Exchange<true> exchange{lds};
  for (int turn = split; turn < count; turn += splits) {
    const int which = __builtin_amdgcn_readlane(its_adapter, turn);
    const uint64_t mine = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(its_rows >> 32), turn) << 32 |
                          (uint32_t)__builtin_amdgcn_readlane((int)its_rows, turn);
    const int list = list_rows(mine), rows = __popcll(mine);
    const uint16_t* weights = static_cast<const uint16_t*>(a.a) + (uint64_t)which * a.rank * a.hidden_in;
    for (int r0 = 0; r0 < a.rank; r0 += 16 * TILES) {
      s.first = s.second = weights + (uint64_t)r0 * a.hidden_in;
#pragma unroll
      for (int i = 0; i < TILES; ++i)   // (rows past the last: the last one's, not stored)
        s.at[i] = (uint32_t)(min(16 * i + c, a.rank - 1 - r0)) * (uint32_t)a.hidden_in * 2 + q * 32;
      s.set_weights();
      for (int row0 = 0; row0 < rows; row0 += 16 * MT) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
          s.set_row(m, (uint32_t)__shfl(list, min(row0 + 16 * m + c, rows - 1)) * (uint32_t)a.hidden_in * 2);
        s.prepare(uniform((int)(threadIdx.x >> 6)), begin, end);
        s.run(end);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (row0 + 16 * m >= rows) break;
          __syncthreads();
          exchange.put(s, m, 0);
          __syncthreads();
#pragma unroll
          for (int turn_of = 0; turn_of < 1024 / kFewThreads; ++turn_of) {
            const int item = turn_of * kFewThreads + threadIdx.x, token = item / (16 * TILES), n = item % (16 * TILES);
            const int row = row0 + 16 * m + token, from = __shfl(list, row & 63);
            if (token < 16 && row < rows && r0 + n < a.rank)
              v[(uint64_t)(first + from) * p.v_pitch + r0 + n] = exchange.column_of_tiles(n, token);
          }
        }
      }
    }
  }
}

// out for a strip of columns: 64 at a time for each wave, of which a lane has twice 8 neighbouring ones of one row of the 16 of a tile.
// KS: the rank in steps of 32, rounded up to a power of two; 0: at most 16, where one step has both halves of v, each against the
// same of b_l.  v is split in LDS, as many rows of it at a time as take 20 KiB at most.
constexpr int kExpandWaves = 4;
constexpr int kExpandThreads = kExpandWaves * 64;
constexpr int kBlock = kExpandWaves * 64;   // columns that a workgroup takes at a time

template <int DT, int KS>
__global__ __launch_bounds__(kExpandThreads, KS <= 2 ? 4 : 2) void adapter_expand_kernel(AdapterParams p) {
  constexpr int STEPS = KS == 0 ? 1 : KS, RANKS = KS == 0 ? 16 : 32 * KS;
  constexpr int M = KS <= 2 ? 4 : 8 / KS, GROUP = 16 * M;                  // tiles of rows, rows
  constexpr int PITCH = RANKS + 8;                                         // (so that the 16 rows of a fragment start in different banks)
  constexpr int TPR = kExpandThreads / GROUP, EACH = RANKS / TPR / 4;      // threads of a row, and times four of its ranks for each
  constexpr int IN_FLIGHT = 4;                                             // pieces of v
  __shared__ __attribute__((aligned(16))) uint16_t split_v[2][GROUP][PITCH];   // high, low
  __shared__ float unit[GROUP];
  const AdapterArgs& a = p.a;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int64_t window = blockIdx.x / p.shares, first = window * kWindow;
  const int share = (int)(blockIdx.x - window * p.shares), columns = a.hidden_out, blocks = (columns + kBlock - 1) / kBlock;
  const WindowPlan& plan = p.plans[window];
  const uint16_t* base = static_cast<const uint16_t*>(a.base);
  uint16_t* out = static_cast<uint16_t*>(a.out);
  if (plan.none != 0 && out != base) {   // rows without an adapter: every workgroup has a part of their columns
    const int begin = (int)((int64_t)blocks * share / p.shares) * kBlock;
    const int end = min((int)((int64_t)blocks * (share + 1) / p.shares) * kBlock, columns);
    int r = 0;
    for (uint64_t none = plan.none; none != 0; none &= none - 1, ++r) {
      if (r % kExpandWaves != wave) continue;
      const uint64_t at = (uint64_t)(first + __ffsll((unsigned long long)none) - 1) * columns;
      for (int n = begin + lane * 8; n < end; n += 512) {
        if (n + 8 <= end) {
          store8(out + at + n, base != nullptr ? load8(base + at + n) : u32x4{0u, 0u, 0u, 0u});
        } else {
          for (int e = n; e < end; ++e) out[at + e] = base != nullptr ? base[at + e] : uint16_t(0);
        }
      }
    }
  }
  const int count = plan.count, pieces = plan.pieces;
  if (count == 0) return;
  // the window's workgroups: one to a strip of columns of an adapter, or, of more adapters, all columns of every shares-th one
  const int strips = min(max(p.shares / count, 1), blocks), strip = share / count;
  if (count <= p.shares && strip >= strips) return;
  const int strip_begin = count <= p.shares ? (int)((int64_t)blocks * strip / strips) * kBlock : 0;
  const int strip_end = count <= p.shares ? min((int)((int64_t)blocks * (strip + 1) / strips) * kBlock, columns) : columns;
  for (int turn = count <= p.shares ? share % count : share; turn < count; turn += p.shares) {
    const int which = plan.adapter[turn];
    const uint64_t mine = plan.rows[turn];
    const int list = list_rows(mine), rows = __popcll(mine);
    const uint16_t* weights = static_cast<const uint16_t*>(a.b) + (uint64_t)which * columns * a.rank;
    const float scale = a.scales != nullptr ? a.scales[which] : 1.0f;
    for (int row0 = 0; row0 < rows; row0 += GROUP) {
      int thread = threadIdx.x;
      asm("" : "+v"(thread));   // (what follows from it is worked out here, where it is used: kept from ahead of the loops, some would be spilled)
      const int tid = thread, lane = tid & 63, c = lane & 15, q = lane >> 4;
      {
        const int row = tid / TPR, part = tid % TPR;
        const float* v = p.v + (uint64_t)(first + __shfl(list, min(row0 + row, rows - 1))) * p.v_pitch;
        f32x4 x[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) x[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int piece = 0; piece < pieces; piece += IN_FLIGHT) {
          f32x4 one[IN_FLIGHT][EACH];
#pragma unroll
          for (int f = 0; f < IN_FLIGHT; ++f)
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
              const int r = (j * TPR + part) * 4;
              one[f][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
              if (piece + f < pieces && r < a.rank && row0 + row < rows)
                one[f][j] = *reinterpret_cast<const f32x4*>(v + (uint64_t)(piece + f) * a.rows * p.v_pitch + r);
            }
#pragma unroll
          for (int f = 0; f < IN_FLIGHT; ++f)
#pragma unroll
            for (int j = 0; j < EACH; ++j) x[j] += one[f][j];
        }
#pragma unroll
        for (int j = 0; j < EACH; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((j * TPR + part) * 4 + e >= a.rank) x[j][e] = 0.0f;   // (what lies behind a row of v is not written)
        float scaling = 1.0f;
        int up = 0;
        if constexpr (DT == kF16) {
          // v may be larger than the type holds, or have elements too small for its bits: its row is scaled by a power of two, exactly, so that
          // the largest comes to 2^14 .. 2^15
          float most = 0.0f;
#pragma unroll
          for (int j = 0; j < EACH; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[j][e]));
#pragma unroll
          for (int other = 1; other < TPR; other *= 2) most = fmaxf(most, __shfl_xor(most, other));
          // (beside an infinity, whose place no finite sum can show in, all else may vanish)
          up = max((int)(__builtin_bit_cast(uint32_t, most) >> 23 & 0xff) - 127 - 14, -126);
          scaling = __builtin_bit_cast(float, (uint32_t)(127 - up) << 23);   // 2^-up
        }
        __syncthreads();
        if (DT == kF16 && part == 0) unit[row] = __builtin_bit_cast(float, (uint32_t)(127 + up) << 23);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          u32x2 high, low;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t h[2], l[2];
#pragma unroll
            for (int o = 0; o < 2; ++o) split<DT>(x[j][2 * e + o] * scaling, h[o], l[o]);
            high[e] = h[0] | h[1] << 16;
            low[e] = l[0] | l[1] << 16;
          }
          const int r = (j * TPR + part) * 4;
          *reinterpret_cast<u32x2*>(&split_v[0][row][r]) = high;
          *reinterpret_cast<u32x2*>(&split_v[1][row][r]) = low;
        }
        __syncthreads();
      }
      auto product = [&](const u32x4 (&b)[STEPS][4], int m, f32x4 (&acc)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
#pragma unroll
          for (int half = 0; half < (KS == 0 ? 1 : 2); ++half) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(KS == 0 ? &split_v[q >> 1][16 * m + c][(q & 1) * 8]
                                                                     : &split_v[half][16 * m + c][k * 32 + q * 8]);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = mfma_16x16x32<DT>(__builtin_bit_cast(bf16x8, b[k][i]), __builtin_bit_cast(bf16x8, x), acc[i]);
          }
      };
      auto joined = [&](u32x4 base, const f32x4& y0, const f32x4& y1, int m) {
        const float s = DT == kF16 ? scale * unit[16 * m + c] : scale;
        u32x4 bits;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4& y = e < 2 ? y0 : y1;
          const float lo = widen_bits<DT>((uint16_t)base[e]) + s * y[e % 2 * 2];
          const float hi = widen_bits<DT>((uint16_t)(base[e] >> 16)) + s * y[e % 2 * 2 + 1];
          bits[e] = round_bits<DT>(lo) | (uint32_t)round_bits<DT>(hi) << 16;
        }
        return bits;
      };
      // the row of tile i of b_l that is this lane's, of the 64 of a block
      auto row_of_b = [&](int i) { return i / 2 * 32 + (c >> 2) * 8 + i % 2 * 4 + (c & 3); };
      int column0 = strip_begin + wave * 64;
      const int whole_end = a.rank == RANKS ? min(strip_end, columns - 63) : 0;
      if (column0 < whole_end) {
        // Whole blocks: all that a block needs is asked for at once, under no condition of a lane's (as the loop below does it, rank 64: 174 us
        // instead of 144; asked for while the block before is under way, between its stores: 162).
        u32x4 have[M][2], b[STEPS][4];
        uint32_t of_row[M];
        const uint16_t* base_window = base + first * columns;
        uint16_t* out_window = out + first * columns;
#pragma unroll
        for (int m = 0; m < M; ++m)
          of_row[m] = ((uint32_t)__shfl(list, min(row0 + 16 * m + c, rows - 1)) * (uint32_t)columns + q * 8) * 2;
        const uint32_t of_b = (uint32_t)(row_of_b(0) * RANKS + (KS == 0 ? (q & 1) * 8 : q * 8)) * 2;
        auto ask_base = [&](int m, int at) {
#pragma unroll
          for (int h = 0; h < 2; ++h) have[m][h] = load8_at(base_window + at, of_row[m], 64 * h);
        };
        auto ask_b = [&](int at) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < STEPS; ++k) b[k][i] = load8_at(weights + (uint64_t)(at + i / 2 * 32) * RANKS, of_b, i % 2 * 8 * RANKS + 64 * k);
        };
#pragma unroll
        for (int m = 0; m < M; ++m) have[m][0] = have[m][1] = u32x4{0u, 0u, 0u, 0u};
        for (; column0 < whole_end; column0 += kBlock) {
          ask_b(column0);
          if (base != nullptr) {
#pragma unroll
            for (int m = 0; m < M; ++m)
              if (row0 + 16 * m < rows) ask_base(m, column0);   // (places past the last row: the last one's, not stored)
          }
#pragma unroll
          for (int m = 0; m < M; ++m) {
            if (row0 + 16 * m >= rows) break;
            f32x4 acc[4];
            product(b, m, acc);
            const u32x4 lo = joined(have[m][0], acc[0], acc[1], m), hi = joined(have[m][1], acc[2], acc[3], m);
            if (row0 + 16 * m + c < rows) {
              store8_at(out_window + column0, of_row[m], lo);
              store8_at(out_window + column0, of_row[m], hi, 64);
            }
          }
        }
      }
      for (; column0 < strip_end; column0 += kBlock) {
        int rank = a.rank, columns = a.hidden_out;
        asm("" : "+s"(rank), "+s"(columns));   // (nothing of this loop is worked out, and kept in registers, ahead of the one above)
        u32x4 b[STEPS][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint16_t* from = weights + (uint64_t)min(column0 + row_of_b(i), columns - 1) * rank;
#pragma unroll
          for (int k = 0; k < STEPS; ++k) b[k][i] = load8_within(from, KS == 0 ? (q & 1) * 8 : k * 32 + q * 8, rank);
        }
        u32x4 have[M][2];
        uint64_t to[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
          to[m] = (uint64_t)(first + __shfl(list, min(row0 + 16 * m + c, rows - 1))) * columns;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            have[m][h] = u32x4{0u, 0u, 0u, 0u};
            if (base != nullptr && row0 + 16 * m < rows) have[m][h] = load8_within(base + to[m], column0 + q * 8 + 32 * h, columns);
          }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          if (row0 + 16 * m >= rows) break;
          f32x4 acc[4];
          product(b, m, acc);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32x4 bits = joined(have[m][h], acc[2 * h], acc[2 * h + 1], m);
            const int own = column0 + q * 8 + 32 * h;
            uint16_t* at = out + to[m] + own;
            if (row0 + 16 * m + c >= rows) continue;
            if (own + 8 <= columns) {
              store8(at, bits);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (own + e < columns) at[e] = (uint16_t)(bits[e / 2] >> (16 * (e % 2)));
            }
          }
        }
      }
    }
  }
}

struct AdapterPlan {
  int64_t windows, v_pitch, pieces, v_shares, shares;
  uint64_t plans_bytes;
};

// Workgroups that keep the device busy: of the first kernel, where more cut the depth finer than pays (256, 512, 1024, 2048 of them, us: 8192 rows of
// prompts, rank 64, 50, 41, 39, 60; 8192 rows, rank 16, 26, 21, 20, 27; 2048 rows of 64 adapters at random 45, 40, 50, 51), and of the second (512, 1024,
// 2048, us: 8192 rows of prompts, one adapter, rank 64 149, 143, 153; rank 16 37, 34, 35; decode 10.8, 11.1, 15.4; 2048 rows in 30 prompts 40, 33, 31).
constexpr int64_t kBusyShrink = 512, kBusy = 1024;

AdapterPlan adapter_plan(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  AdapterPlan f;
  auto between = [](int64_t v, int64_t hi) { return std::max<int64_t>(1, std::min(v, hi)); };
  const int64_t most = std::min({num, rows, int64_t(kWindow)});   // adapters of a window
  f.windows = (rows + kWindow - 1) / kWindow;
  f.v_pitch = (rank + 3) / 4 * 4;
  // pieces of the depth: at least one step of every wave.  v and out in at most 1, 2, 4, 8, 16 pieces, us: one row (4096 -> 4096) 8.2 + 3.9,
  // 5.7 + 4.1, 4.7 + 4.4, 4.1 + 4.6, 3.7 + 5.3; 333 rows (2047 -> 1023) 38 + 13, 21 + 13, 13 + 13, 10.9 + 12.6, 10.8 + 12.9; 64 rows of one
  // adapter, rank 64 47 + 8, 26 + 8, 17 + 9, 13 + 10, 9 + 13; 8192 rows of prompts (4096 -> 14336) 92 + 140, 52 + 141, 41 + 145, 41 + 144, 41 + 145
  f.pieces = between(hidden_in / (64 * kFewWaves), 8);
  f.v_shares = between(kBusyShrink / f.windows, most * f.pieces);
  f.pieces = std::min(f.pieces, f.v_shares);
  f.shares = between(kBusy / f.windows, most * ((hidden_out + kBlock - 1) / kBlock));
  f.plans_bytes = (uint64_t)f.windows * sizeof(WindowPlan);
  static_assert(sizeof(WindowPlan) % 16 == 0, "");
  return f;
}

template <int DT, int TILES>
void launch_shrink(const AdapterParams& p, const AdapterPlan& f, hipStream_t stream) {
  const dim3 grid((uint32_t)(f.windows * f.v_shares));
  if (on_any_element(p.a.a, p.a.x, p.a.hidden_in)) {
    hipLaunchKernelGGL((adapter_shrink_kernel<DT, TILES, true>), grid, dim3(kFewThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL((adapter_shrink_kernel<DT, TILES, false>), grid, dim3(kFewThreads), 0, stream, p);
  }
}

template <int DT>
hipError_t launch_adapters(const AdapterArgs& a, hipStream_t stream) {
  const AdapterPlan f = adapter_plan(a.rows, a.num, a.rank, a.hidden_in, a.hidden_out);
  AdapterParams p;
  p.a = a;
  p.plans = static_cast<WindowPlan*>(a.scratch);
  p.v = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + f.plans_bytes);
  p.v_pitch = (int32_t)f.v_pitch;
  p.pieces = (int32_t)f.pieces;
  p.shares = (int32_t)f.v_shares;
  if (a.rank <= 16) {
    launch_shrink<DT, 1>(p, f, stream);
  } else if (a.rank <= 32) {
    launch_shrink<DT, 2>(p, f, stream);
  } else {
    launch_shrink<DT, 4>(p, f, stream);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  p.shares = (int32_t)f.shares;
  const dim3 grid((uint32_t)(f.windows * f.shares));
  if (a.rank <= 16) {
    hipLaunchKernelGGL((adapter_expand_kernel<DT, 0>), grid, dim3(kExpandThreads), 0, stream, p);
  } else if (a.rank <= 32) {
    hipLaunchKernelGGL((adapter_expand_kernel<DT, 1>), grid, dim3(kExpandThreads), 0, stream, p);
  } else if (a.rank <= 64) {
    hipLaunchKernelGGL((adapter_expand_kernel<DT, 2>), grid, dim3(kExpandThreads), 0, stream, p);
  } else if (a.rank <= 128) {
    hipLaunchKernelGGL((adapter_expand_kernel<DT, 4>), grid, dim3(kExpandThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL((adapter_expand_kernel<DT, 8>), grid, dim3(kExpandThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

bool adapters_fit(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  const AdapterPlan f = adapter_plan(rows, num, rank, hidden_in, hidden_out);
  const int64_t threads = int64_t(1) << 32;   // of a launch, which are counted in 32 bits
  return f.windows * f.v_shares * kFewThreads < threads && f.windows * f.shares * kExpandThreads < threads;
}

uint64_t adapters_scratch_bytes(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  const AdapterPlan f = adapter_plan(rows, num, rank, hidden_in, hidden_out);
  return f.plans_bytes + (uint64_t)(f.pieces * rows * f.v_pitch) * sizeof(float);
}

hipError_t adapters(const AdapterArgs& a, hipStream_t stream) {
  return a.dt == kBF16 ? launch_adapters<kBF16>(a, stream) : launch_adapters<kF16>(a, stream);
}

}  // namespace gg
