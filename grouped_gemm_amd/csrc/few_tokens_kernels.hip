// A gated expert layer for the few tokens of a decode step, in two kernels:
//
//   h[s] = silu(x[t] @ gate_e) * (x[t] @ up_e)     for each slot s = (t, j), e = experts[t, j]
//   out[t] = sum over j of weights[t, j] * (h[s] @ down_e)
//
// Bound by reading the weights of the experts that are named, once: 3 * hidden * ffn elements each.  So everything is
// laid out for that one stream.  A workgroup has a strip of an expert's weights (32 or 64 columns of gate and of
// up, 64 or 128 of down) over the whole depth, or a piece of it; its waves take the depth in turns, each with its own loads from
// HBM straight into registers, where they are the matrix instructions' first operand: 16 weight columns x 32
// deep against 16 tokens, so that one load of a weight serves all tokens of its expert.  No LDS and no barrier in
// the loop; the waves' sums are added up through LDS at its end.  Depths, widths and addresses are any.
//
// Where the depth is contiguous (trans_b), a lane loads 16 elements along it, in two halves: the order of the
// depth inside an instruction is free as long as both operands have the same.  Where the width is, a lane loads 8 rows
// of 8 columns and transposes them in registers, 32 byte permutations for 64 weights.
//
// The second kernel's sums over the depth's pieces and over a token's experts are joined by the last workgroup to arrive at a
// strip of columns, in the order of the slots and pieces: the same bits on every call.
//
// Measured: 64 tokens, top 8 of 128 experts, 7168 -> 2048, weights contiguous along the depth (11.1 GB) 1184 us of gate and up (6.2 TB/s) and
// 698 of down (5.3 TB/s); one token, two experts, 4096 -> 14336 (705 MB) 85 + 47 us (5.5, 5.0 TB/s), of which about 10 us each are the
// start, the first loads and the joins.  Where 16 rows are taken at a time, three waves to a SIMD have registers: 12 to a compute unit in workgroups of 4
// (with 16, in workgroups of 8, gate and up along the depth run at 5.4 TB/s), 8 where gate and up of a contiguous width are one workgroup of 8.
// Where 32 or 64 are, two have: 8.
#include "operators.hpp"

#include <math.h>

#include <algorithm>

#include "few_rows.hpp"
#include "gmm_kernel.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kFewWords = (int)(kFewMaxExperts / 32);
static_assert(kFewWords <= 64, "");

struct FewParams {
  FewTokensArgs a;
  int32_t slots;         // tokens * top_k
  int32_t tiles;         // strips of this kernel
  int32_t pieces;        // of the depth of down
  int32_t shares;        // of this kernel's: workgroups that an expert's rows are shared among
  int32_t counters;      // arrivals to clear for the second kernel
  int32_t ffn_pitch;     // elements from one row of h to the next
  int32_t* arrivals;     // [strips of down]
  uint16_t* h;           // [slots][2][ffn_pitch] h rounded to the element type, and what the rounding left: two rows for
                         // the second product, which is then exact to twice the bits of the type
  int32_t* units;        // float16: [slots][blocks] h of each block of columns is kept as a multiple of 2^unit
  int32_t blocks;
  int32_t hidden_pitch;  // elements from one row of parts to the next
  uint32_t parts_bytes;
  float* parts;          // [pieces][slots][hidden_pitch]
};

// Which experts are named, and the slots of one of them: in any order (a token's results do not depend on its place), or, where workgroups
// share them and have to agree, in their own.  Up to 64 slots every wave finds the expert by itself, from one load and a ballot for each;
// more go through LDS.
struct FewLds {
  uint32_t named[kFewWords];
  int32_t rows;
  int32_t of_wave[2 * kFewWaves];
  int32_t slot[kFewMaxSlots];
};

// h may be larger than float16 holds, or too small for its bits.  Every block of 32 or 64 columns (a strip's) is kept as multiples of a power of two
// that brings its largest to 2^14 .. 2^15; the second kernel brings the blocks to the largest of a row's units, as it multiplies, and its sums
// back.  So h is exact to 2^-22 of itself and to 2^-37 of its row's largest, whatever its size.  Without and with it, us: one token, two of 8 experts,
// 4096 -> 14336 135, 136; 5 tokens, top 6 of 64, 2048 -> 1408 80, 80; 64, top 8 of 128, 4096 -> 2048 1180, 1182; where many rows meet few weights
// the multiplications show, 64, top 8 of 8, 2048 -> 2048, 138, 161, along the depth 110, 128.
constexpr int kNoUnit = -1024;   // of a block of zeros: below all others
__device__ __forceinline__ int unit_of(float most) {
  if (!(most > 0.0f)) return kNoUnit;
  return (most < INFINITY ? ilogbf(most) + 1 : 129) - 15;   // (beside an infinity, whose place no finite sum can show in, all else may vanish)
}

__device__ __forceinline__ int first_lane(uint64_t mask) { return __ffsll((unsigned long long)mask) - 1; }
__device__ __forceinline__ bool few_slots(const FewParams& p) { return p.slots <= 64; }

// All threads.  Returns the number of experts that are named; `mine` is for find_expert and gather_slots.
__device__ __forceinline__ int find_named(const FewParams& p, FewLds& lds, int& mine) {
  const int lane = threadIdx.x & 63;
  int named = 0;
  mine = -1;
  if (few_slots(p)) {
    if (lane < p.slots) mine = p.a.chosen[lane];
    if ((uint32_t)mine >= (uint32_t)p.a.experts) mine = -1;
    for (uint64_t left = __ballot(mine >= 0); left != 0; ++named) left &= ~__ballot(mine == __builtin_amdgcn_readlane(mine, first_lane(left)));
  } else {
    if (threadIdx.x < kFewWords) lds.named[threadIdx.x] = 0;
    if (threadIdx.x == 0) lds.rows = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.slots; i += (int)blockDim.x) {
      const uint32_t e = (uint32_t)p.a.chosen[i];
      if (e < (uint32_t)p.a.experts) atomicOr(&lds.named[e / 32], 1u << (e % 32));
    }
    __syncthreads();
    named = uniform(__shfl(wave_prefix(lane < kFewWords ? __popc(lds.named[lane]) : 0), 63));
  }
  return named;
}

// The which-th of them.
__device__ __forceinline__ int find_expert(const FewParams& p, const FewLds& lds, int mine, int which) {
  const int lane = threadIdx.x & 63;
  if (few_slots(p)) {
    uint64_t left = __ballot(mine >= 0);
    for (int i = 0; i < which; ++i) left &= ~__ballot(mine == __builtin_amdgcn_readlane(mine, first_lane(left)));
    return __builtin_amdgcn_readlane(mine, first_lane(left));
  }
  uint32_t word = lane < kFewWords ? lds.named[lane] : 0u;
  const int upto = wave_prefix(__popc(word)), before = upto - __popc(word);
  const uint64_t here = __ballot(which >= before && which < upto);
  for (int i = before; i < which && word != 0; ++i) word &= word - 1;
  return __builtin_amdgcn_readlane(lane * 32 + __ffs(word) - 1, first_lane(here));
}

// All threads.  Writes the expert's slots to LDS and returns their number.
__device__ __forceinline__ int gather_slots(const FewParams& p, FewLds& lds, int mine, int expert) {
  const int lane = threadIdx.x & 63;
  if (few_slots(p)) {
    if (threadIdx.x < 64) {
      const uint64_t same = __ballot(mine == expert);
      if (mine == expert) lds.slot[__popcll(same & ((uint64_t(1) << lane) - 1))] = lane;
      if (lane == 0) lds.rows = __popcll(same);
    }
  } else if (p.shares == 1) {
    for (int i = threadIdx.x; i < p.slots; i += (int)blockDim.x)
      if (p.a.chosen[i] == expert) lds.slot[atomicAdd(&lds.rows, 1)] = i;
  } else {
    // every wave its share of the slots: how many are the expert's, then where they go (3 % of the largest launches, whose rows nobody shares)
    const int waves = (int)blockDim.x / 64, wave = threadIdx.x / 64, share = ((p.slots + waves - 1) / waves + 63) / 64 * 64;
    const int begin = min(wave * share, p.slots), end = min(begin + share, p.slots);
    int count = 0;
    for (int i = begin + lane; i - lane < end; i += 64) count += __popcll(__ballot(i < end && p.a.chosen[i] == expert));
    if (lane == 0) lds.of_wave[wave] = count;
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < waves; ++w) {
      at += w < wave ? lds.of_wave[w] : 0;
      all += lds.of_wave[w];
    }
    for (int i = begin + lane; i - lane < end; i += 64) {
      const bool its = i < end && p.a.chosen[i] == expert;
      const uint64_t same = __ballot(its);
      if (its) lds.slot[at + __popcll(same & ((uint64_t(1) << lane) - 1))] = i;
      at += __popcll(same);
    }
    if (threadIdx.x == 0) lds.rows = all;
  }
  __syncthreads();
  return uniform(lds.rows);
}

// Where the width is contiguous, gate and up have waves of their own, so that an instruction reads 256 neighbouring bytes of
// a row.  Against 128 bytes of each of the two by the same wave: one token, two experts, 4096 -> 14336 (470 MB) 85 us, 88; eight experts (1.88 GB)
// 338 us = 5.6 TB/s, 344.
constexpr int gate_up_threads(bool nt) { return nt ? kFewThreads : 2 * kFewThreads; }

template <int DT, bool NT, int MT, bool ODD>
__global__ __launch_bounds__(gate_up_threads(NT), MT == 1 ? 3 : 2) void few_gate_up_kernel(FewParams p) {
  using S = Stream<DT, NT, 4, MT, ODD>;
  constexpr int COLUMNS = NT ? 32 : 128, OF_ROUND = NT ? 32 : 64;   // of h; of a round: a block with a unit of its own
  constexpr int THREADS = gate_up_threads(NT);
  __shared__ FewLds few_lds;
  __shared__ f32x4 lds[THREADS * 4];
  const FewTokensArgs& a = p.a;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4, wave = uniform((int)(threadIdx.x >> 6));
  if (blockIdx.x == 0)   // the second kernel's counters
    for (int i = threadIdx.x; i < p.counters; i += THREADS) p.arrivals[i] = 0;
  int mine;
  const int named = find_named(p, few_lds, mine);
  const int of_expert = p.tiles * p.shares;
  if (blockIdx.x >= named * of_expert) return;
  const int task = (int)task_of_block(blockIdx.x, named * of_expert), which = task / of_expert, left = task - which * of_expert;
  const int tile = left / p.shares, column0 = tile * COLUMNS, row_first = (left - tile * p.shares) * 16 * MT, row_step = p.shares * 16 * MT;
  const int expert = find_expert(p, few_lds, mine, which);
  const int ffn = a.ffn, hidden = a.hidden;
  const uint16_t* w = static_cast<const uint16_t*>(a.w13) + (uint64_t)expert * 2 * ffn * hidden;
  S s;
  s.x = static_cast<const uint16_t*>(a.x);
  s.depth = hidden;
  s.width = 8;
  if constexpr (NT) {
    s.first = w + (uint64_t)column0 * hidden;
    s.second = s.first + (uint64_t)ffn * hidden;
#pragma unroll
    for (int i = 0; i < 4; ++i)   // (rows past the last: the last one's, not stored)
      s.at[i] = (uint32_t)(min(16 * (i & 1) + c, ffn - 1 - column0)) * (uint32_t)hidden * 2 + q * 32;
  } else {
    // (a lane's 8 columns past the last column move back to it)
    const int column = ffn < 8 ? 0 : min(column0 + c * 8, ffn - 8);
    s.width = min(ffn, 8);
    s.first = w + wave / kFewWaves * ffn;
    s.pitch = (uint32_t)ffn * 4;
    s.at[0] = q * 8 * s.pitch + (uint32_t)column * 2;
  }
  s.set_weights();
  const Exchange<NT> exchange{lds};
  const int end = (hidden + S::DEPTH - 1) / S::DEPTH;
  s.prepare(wave % kFewWaves, 0, end);
  const int rows = gather_slots(p, few_lds, mine, expert);
  for (int row0 = row_first; row0 < rows; row0 += row_step) {
    if (row0 > row_first) s.prepare(wave % kFewWaves, 0, end);
#pragma unroll
    for (int m = 0; m < MT; ++m)   // (places past the last row: the last one's, not stored)
      s.set_row(m, (uint32_t)(few_lds.slot[min(row0 + 16 * m + c, rows - 1)] / a.top_k) * (uint32_t)hidden * 2);
    s.run(end);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (row0 + 16 * m >= rows) break;
#pragma unroll
      for (int round = 0; round < Exchange<NT>::ROUNDS; ++round) {
        __syncthreads();
        exchange.put(s, m, round);
        __syncthreads();
        for (int item = threadIdx.x; item < 16 * OF_ROUND; item += THREADS) {
          const int token = item / OF_ROUND, n = item % OF_ROUND;
          const int row = row0 + 16 * m + token;
          if (row >= rows) break;
          float gate, up;
          int column;
          bool own;
          if constexpr (NT) {
            gate = exchange.column_of_tiles(n, token);
            up = exchange.column_of_tiles(32 + n, token);
            column = column0 + n;
            own = column < ffn;
          } else {
            const int start = column0 + round * 64 + (n >> 3) * 8;
            gate = exchange.column_of_block(0, n >> 3, n & 7, token);
            up = exchange.column_of_block(kFewWaves, n >> 3, n & 7, token);
            column = (ffn < 8 ? 0 : min(start, ffn - 8)) + (n & 7);
            own = column >= start && column < ffn;   // (of 8 columns that moved back: their own only)
          }
          float h = own ? gate / (1.0f + expf(-gate)) * up : 0.0f;
          if constexpr (DT == kF16) {   // (the lanes of a row's block are all here)
            const int unit = unit_of(group_reduce<OF_ROUND>(fabsf(h), [](float p, float q) { return fmaxf(p, q); }));
            const int block = column0 / OF_ROUND + round;
            if (n == 0 && block < p.blocks) p.units[(uint64_t)few_lds.slot[row] * p.blocks + block] = unit;
            h = ldexpf(h, -unit);
          }
          if (!own) continue;
          uint16_t* to = p.h + (uint64_t)few_lds.slot[row] * 2 * p.ffn_pitch + column;
          uint32_t high, low;
          split<DT>(h, high, low);
          to[0] = (uint16_t)high, to[p.ffn_pitch] = (uint16_t)low;
        }
      }
    }
  }
}

template <int DT, bool NT, int MT, bool ODD>
__global__ __launch_bounds__(kFewThreads, MT == 1 ? 3 : 2) void few_down_kernel(FewParams p) {
  constexpr bool SCALED = DT == kF16;
  using S = Stream<DT, NT, 4, MT, ODD, SCALED>;
  constexpr int COLUMNS = NT ? 64 : 128;
  __shared__ int32_t row_units[SCALED ? 8 * MT : 1];   // of the slots whose rows are taken
  __shared__ FewLds few_lds;
  __shared__ f32x4 lds[kFewWaves * 256];
  __shared__ int32_t arrived;
  const FewTokensArgs& a = p.a;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  int mine;
  const int named = find_named(p, few_lds, mine), hidden = a.hidden, ffn = a.ffn;
  // strips one after the other, so that their sums are joined on the way (without any expert: zeros are stored)
  const int arrivals = named * p.pieces * p.shares, tasks = max(arrivals, 1) * p.tiles;
  if (blockIdx.x >= tasks) return;
  const int task = (int)task_of_block(blockIdx.x, tasks);
  const int tile = task / max(arrivals, 1), left = task - tile * arrivals, column0 = tile * COLUMNS;
  if (named > 0) {
    const int which = left / (p.pieces * p.shares), in_expert = left - which * p.pieces * p.shares, piece = in_expert / p.shares;
    const int row_first = (in_expert - piece * p.shares) * 16 * MT, row_step = p.shares * 16 * MT;
    const int expert = find_expert(p, few_lds, mine, which);
    const uint16_t* w = static_cast<const uint16_t*>(a.w2) + (uint64_t)expert * ffn * hidden;
    S s;
    s.x = p.h;
    s.depth = ffn;
    s.width = 8;
    if constexpr (NT) {
      s.first = s.second = w + (uint64_t)column0 * ffn;
#pragma unroll
      for (int i = 0; i < 4; ++i) s.at[i] = (uint32_t)(min(16 * i + c, hidden - 1 - column0)) * (uint32_t)ffn * 2 + q * 32;
    } else {
      const int column = hidden < 8 ? 0 : min(column0 + c * 8, hidden - 8);
      s.width = min(hidden, 8);
      s.first = w;
      s.pitch = (uint32_t)hidden * 2;
      s.at[0] = q * 8 * s.pitch + (uint32_t)column * 2;
    }
    s.set_weights();
    const int steps = (ffn + S::DEPTH - 1) / S::DEPTH, begin = (int)((int64_t)steps * piece / p.pieces);
    const int end = (int)((int64_t)steps * (piece + 1) / p.pieces);
    const Exchange<NT> exchange{lds};
    float* parts = p.parts + (uint64_t)piece * p.slots * p.hidden_pitch;
    s.prepare(uniform((int)(threadIdx.x >> 6)), begin, end);
    const int rows = 2 * gather_slots(p, few_lds, mine, expert);   // of h, two for each slot
    for (int row0 = row_first; row0 < rows; row0 += row_step) {
      if (row0 > row_first) s.prepare(uniform((int)(threadIdx.x >> 6)), begin, end);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int row = min(row0 + 16 * m + c, rows - 1);
        s.set_row(m, ((uint32_t)few_lds.slot[row / 2] * 2 + (row & 1)) * (uint32_t)p.ffn_pitch * 2);
        if constexpr (SCALED) s.unit_row[m] = (uint32_t)few_lds.slot[row / 2] * (uint32_t)p.blocks * 4;
      }
      if constexpr (SCALED) {
        s.units = p.units;
        s.run(end, [&] {   // the largest unit of each row's blocks that lie in this piece of the depth
          constexpr int OF_SLOT = kFewThreads / (8 * MT), IN_FLIGHT = 4;   // threads
          const int part = (int)threadIdx.x % OF_SLOT, pair = (int)threadIdx.x / OF_SLOT;
          const int last = (min(end * S::DEPTH, ffn) - 1) / S::BLOCK;
          const int32_t* units = p.units + (uint64_t)few_lds.slot[min(row0 / 2 + pair, rows / 2 - 1)] * p.blocks;
          int most = kNoUnit;
          for (int b = begin * S::DEPTH / S::BLOCK + part; b <= last; b += IN_FLIGHT * OF_SLOT)
#pragma unroll
            for (int f = 0; f < IN_FLIGHT; ++f) most = max(most, units[min(b + f * OF_SLOT, last)]);
#pragma unroll
          for (int other = 1; other < OF_SLOT; other *= 2) most = max(most, __shfl_xor(most, other));
          __syncthreads();   // (what was there is read no more)
          if (part == 0) row_units[pair] = most;
          __syncthreads();
#pragma unroll
          for (int m = 0; m < MT; ++m) s.row_unit[m] = row_units[8 * m + c / 2];
        });
      } else {
        s.run(end);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (row0 + 16 * m >= rows) break;
#pragma unroll
        for (int round = 0; round < Exchange<NT>::ROUNDS; ++round) {
          __syncthreads();
          exchange.put(s, m, round);
          __syncthreads();
          for (int item = threadIdx.x; item < 512; item += kFewThreads) {
            const int pair = item >> 6, n = item & 63;   // of 8 slots, of 64 columns
            const int row = row0 + 16 * m + 2 * pair;
            if (row >= rows) break;
            float y, lower;   // of the two halves of h
            int column;
            bool own;
            if constexpr (NT) {
              y = exchange.column_of_tiles(n, 2 * pair), lower = exchange.column_of_tiles(n, 2 * pair + 1);
              column = column0 + n;
              own = column < hidden;
            } else {
              const int start = column0 + round * 64 + (n >> 3) * 8;
              y = exchange.column_of_block(0, n >> 3, n & 7, 2 * pair), lower = exchange.column_of_block(0, n >> 3, n & 7, 2 * pair + 1);
              column = (hidden < 8 ? 0 : min(start, hidden - 8)) + (n & 7);
              own = column >= start && column < hidden;
            }
            if (!own) continue;
            const int slot = few_lds.slot[row / 2];
            if (fabsf(y) < INFINITY) y += lower;   // (against an infinite weight the lower half, zero or of any sign, would make NaN)
            float part = y * a.weights[slot];
            if constexpr (SCALED) part = ldexpf(part, row_units[8 * m + pair]);
            // (device scope: written to and read from where all XCDs see it, without a fence that empties whole L2s)
            __hip_atomic_store(&parts[(uint64_t)slot * p.hidden_pitch + column], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
      }
    }
    if (arrivals > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every wave's part has arrived before the arrival is counted
      __syncthreads();
      if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(&p.arrivals[tile], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (uniform(arrived) != arrivals - 1) return;
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
  }
  // The strip's sums, in the order of a token's experts and of the pieces, four columns to a thread and IN_FLIGHT terms at a
  // time (one by one each would wait for memory).
  constexpr int IN_FLIGHT = 8;
  uint16_t* out = static_cast<uint16_t*>(a.out);
  const __amdgpu_buffer_rsrc_t parts = make_rsrc(p.parts, p.parts_bytes);
  for (int i = threadIdx.x; i < a.tokens * (COLUMNS / 4); i += kFewThreads) {
    const int token = i / (COLUMNS / 4), column = column0 + i % (COLUMNS / 4) * 4;
    if (column >= hidden) continue;
    const int32_t* chosen = a.chosen + token * a.top_k;
    const int terms = a.top_k * p.pieces;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    int j = 0, piece = 0;
    for (int at = 0; at < terms; at += IN_FLIGHT) {
      f32x4 term[IN_FLIGHT];
#pragma unroll
      for (int f = 0; f < IN_FLIGHT; ++f) {
        term[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (at + f < terms && (uint32_t)chosen[j] < (uint32_t)a.experts)
          term[f] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                  parts, (uint32_t)((piece * p.slots + token * a.top_k + j) * p.hidden_pitch + column) * 4, 0, kDeviceScope));
        if (++piece == p.pieces) piece = 0, j = min(j + 1, a.top_k - 1);
      }
#pragma unroll
      for (int f = 0; f < IN_FLIGHT; ++f) sum += term[f];
    }
    uint16_t* to = out + (uint64_t)token * hidden + column;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (column + e < hidden) to[e] = round_bits<DT>(sum[e]);
  }
}

struct FewPlan {
  int64_t slots, named, up_tiles, down_tiles, pieces, ffn_pitch, blocks, hidden_pitch;
  int up_rows, down_rows;   // of 16, that a workgroup takes at a time
  int64_t up_shares, down_shares;   // workgroups that an expert's rows are shared among
  uint64_t arrivals_bytes, h_bytes, units_bytes, parts_bytes;
};

constexpr int64_t kFewUnits = 256;   // compute units

FewPlan few_plan(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool nt) {
  FewPlan f;
  f.slots = tokens * top_k;
  f.named = std::max<int64_t>(1, std::min(f.slots, experts));   // at most
  f.up_tiles = (ffn + (nt ? 31 : 127)) / (nt ? 32 : 128);
  f.down_tiles = (hidden + (nt ? 63 : 127)) / (nt ? 64 : 128);
  f.ffn_pitch = (ffn + 7) / 8 * 8;
  // the depth of down in pieces where its strips alone are fewer than compute units, each of at least eight steps to a wave.  One
  // token, 4096 -> 14336, in 1, 2, 4, 8 pieces: 64 strips 58, 34, 25, 26 us, 128 strips 65, 43, 44, 53, 512 strips 160, 185, 188, 193; 130 to 250
  // strips of 4096 in 1 and 2: 130 20.7, 25.1, 150 21.0, 26.0, 200 24.5, 27.2, 250 29.1, 30.4
  const int64_t steps = (ffn + (nt ? 63 : 31)) / (nt ? 64 : 32), fit = kFewUnits / (f.named * f.down_tiles), deep = steps / (8 * kFewWaves);
  f.pieces = std::max<int64_t>(1, std::min({fit, deep, int64_t(16)}));
  // Rows taken at a time, by how many an expert has on average (of down two for each slot; those that do not fit read the weights again): more of them
  // leave fewer waves to a compute unit, and 4 spill registers: inside the loop bf16 with the width contiguous and fp16 on any element (36 and 28 words in
  // two steps), others around it or none.  us with 1, 2 and 4 times 16, averages 3, 4, 8, 16 (bf16): gate | up 77 78 81, 279 281 281, 340 348 368, 528 361 373;
  // down 48 54 54, 180 153 161, 281 176 178, 469 316 212.
  f.up_rows = f.slots <= 8 * experts ? 1 : 2;
  f.down_rows = f.slots < 4 * experts ? 1 : (f.slots <= 12 * experts ? 2 : 4);
  // Where the strips leave compute units, an expert's rows are shared among as many workgroups as there are turns on average.  us without and
  // with: 64 tokens, all of 4 experts, 1024 -> 2048 36 + 71, 21 + 47; all of 8, 512 -> 1024 28 + 71, 18 + 47; 4 of 5, 700 -> 300 14 + 27, 10 + 21.
  auto shares = [&](int64_t rows, int64_t strips) {
    const int64_t turns = (f.slots + experts * rows - 1) / (experts * rows);
    return std::max<int64_t>(1, std::min(turns, kFewUnits / strips));
  };
  f.up_shares = shares(16 * f.up_rows, f.named * f.up_tiles);
  f.down_shares = shares(8 * f.down_rows, f.named * f.down_tiles * f.pieces);
  f.arrivals_bytes = (uint64_t)(f.down_tiles * 4 + 255) / 256 * 256;
  f.h_bytes = ((uint64_t)f.slots * f.ffn_pitch * 4 + 255) / 256 * 256;
  f.blocks = (ffn + (nt ? 31 : 63)) / (nt ? 32 : 64);
  f.units_bytes = ((uint64_t)f.slots * f.blocks * 4 + 255) / 256 * 256;
  f.hidden_pitch = (hidden + 3) / 4 * 4;
  f.parts_bytes = (uint64_t)f.pieces * f.slots * f.hidden_pitch * 4;
  return f;
}

template <int DT, bool NT, bool ODD>
void launch_gate_up(const FewParams& p, const FewPlan& f, dim3 grid, hipStream_t stream) {
  if (f.up_rows == 1) {
    hipLaunchKernelGGL((few_gate_up_kernel<DT, NT, 1, ODD>), grid, dim3(gate_up_threads(NT)), 0, stream, p);
  } else {
    hipLaunchKernelGGL((few_gate_up_kernel<DT, NT, 2, ODD>), grid, dim3(gate_up_threads(NT)), 0, stream, p);
  }
}

template <int DT, bool NT, bool ODD>
void launch_down(const FewParams& p, const FewPlan& f, dim3 grid, hipStream_t stream) {
  switch (f.down_rows) {
    case 1: hipLaunchKernelGGL((few_down_kernel<DT, NT, 1, ODD>), grid, dim3(kFewThreads), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((few_down_kernel<DT, NT, 2, ODD>), grid, dim3(kFewThreads), 0, stream, p); break;
    default: hipLaunchKernelGGL((few_down_kernel<DT, NT, 4, ODD>), grid, dim3(kFewThreads), 0, stream, p); break;
  }
}

template <int DT, bool NT>
hipError_t launch_few(const FewTokensArgs& a, const FewPlan& f, hipStream_t stream) {
  FewParams p;
  p.a = a;
  p.slots = (int32_t)f.slots;
  p.ffn_pitch = (int32_t)f.ffn_pitch;
  p.hidden_pitch = (int32_t)f.hidden_pitch;
  p.parts_bytes = (uint32_t)f.parts_bytes;
  char* at = static_cast<char*>(a.scratch);
  p.arrivals = reinterpret_cast<int32_t*>(at);
  p.h = reinterpret_cast<uint16_t*>(at + f.arrivals_bytes);
  p.units = reinterpret_cast<int32_t*>(at + f.arrivals_bytes + f.h_bytes);
  p.blocks = (int32_t)f.blocks;
  p.parts = reinterpret_cast<float*>(at + f.arrivals_bytes + f.h_bytes + f.units_bytes);
  p.tiles = (int32_t)f.up_tiles;
  p.pieces = (int32_t)f.pieces;
  p.counters = (int32_t)f.down_tiles;
  p.shares = (int32_t)f.up_shares;
  const dim3 up((uint32_t)(f.named * f.up_tiles * f.up_shares)), down((uint32_t)(f.named * f.down_tiles * f.pieces * f.down_shares));
  if (NT && on_any_element(a.w13, a.x, a.hidden)) {
    launch_gate_up<DT, NT, NT>(p, f, up, stream);
  } else {
    launch_gate_up<DT, NT, false>(p, f, up, stream);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  p.tiles = (int32_t)f.down_tiles;
  p.shares = (int32_t)f.down_shares;
  if (NT && on_any_element(a.w2, nullptr, a.ffn)) {
    launch_down<DT, NT, NT>(p, f, down, stream);
  } else {
    launch_down<DT, NT, false>(p, f, down, stream);
  }
  return hipGetLastError();
}

}  // namespace

bool few_tokens_fits(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool trans_b) {
  const FewPlan f = few_plan(tokens, experts, top_k, hidden, ffn, trans_b);
  const int64_t most = (int64_t(1) << 32) / gate_up_threads(false);   // (threads of a launch are counted in 32 bits)
  return f.named * f.up_tiles * f.up_shares < most && f.named * f.down_tiles * f.pieces * f.down_shares < most && f.slots * f.ffn_pitch * 4 < (int64_t(1) << 32) && f.parts_bytes < (uint64_t(1) << 32);
}

uint64_t few_tokens_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool trans_b) {
  const FewPlan f = few_plan(tokens, experts, top_k, hidden, ffn, trans_b);
  return f.arrivals_bytes + f.h_bytes + f.units_bytes + f.parts_bytes;
}

hipError_t few_tokens(const FewTokensArgs& a, hipStream_t stream) {
  const FewPlan f = few_plan(a.tokens, a.experts, a.top_k, a.hidden, a.ffn, a.trans_b);
#define GG_LAUNCH(DT) (a.trans_b ? launch_few<DT, true>(a, f, stream) : launch_few<DT, false>(a, f, stream))
  return a.dt == kBF16 ? GG_LAUNCH(kBF16) : GG_LAUNCH(kF16);
#undef GG_LAUNCH
}

}  // namespace gg
