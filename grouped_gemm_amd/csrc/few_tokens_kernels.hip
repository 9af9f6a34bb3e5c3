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
#include "operators.hpp"

#include <math.h>

#include "gmm_kernel.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kFewWaves = 8;
constexpr int kFewThreads = kFewWaves * 64;
constexpr int kFewWords = (int)(kFewMaxExperts / 32);
static_assert(kFewWords <= 64, "");

// 8 elements on any boundary.
struct __attribute__((packed, aligned(2))) Packed8 {
  u32x4 v;
};
__device__ __forceinline__ u32x4 load8(const uint16_t* p) { return reinterpret_cast<const Packed8*>(p)->v; }

// Elements k .. k + 7 of a row of `depth`, zeros past its end; reads nothing outside the row.
__device__ __forceinline__ u32x4 load8_within(const uint16_t* row, int k, int depth) {
  if (k + 8 <= depth) return load8(row + k);
  u32x4 v = {0u, 0u, 0u, 0u};
  if (k >= depth) return v;
  if (depth >= 8) {   // the row's last 8, those before k shifted out
    const unsigned __int128 last = __builtin_bit_cast(unsigned __int128, load8(row + depth - 8));
    return __builtin_bit_cast(u32x4, last >> (16 * (k + 8 - depth)));
  }
  uint16_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k + i < depth ? row[k + i] : uint16_t(0);
  return __builtin_bit_cast(u32x4, e);
}

template <int DT>
__device__ __forceinline__ uint16_t round_bits(float v) {
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  else return __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ float widen_bits(uint16_t v) {
  if constexpr (DT == kBF16) return __builtin_bit_cast(float, (uint32_t)v << 16);
  else return (float)__builtin_bit_cast(_Float16, v);
}

struct FewParams {
  FewTokensArgs a;
  int32_t slots;         // tokens * top_k
  int32_t tiles;         // strips of this kernel
  int32_t pieces;        // of the depth of down
  int32_t counters;      // arrivals to clear for the second kernel
  int32_t ffn_pitch;     // elements from one row of high (and low) to the next
  int32_t* arrivals;     // [strips of down]
  uint16_t* high;        // [slots][ffn_pitch] h rounded to the element type,
  uint16_t* low;         // ... and what the rounding left: h is handed on with twice the bits of the type
  float* parts;          // [pieces][slots][hidden]
};

// Which experts are named, and the slots of one of them.
struct FewSchedule {
  uint32_t named[kFewWords];
  int32_t rows;
  int32_t expert;
  int32_t slot[kFewMaxSlots];
};

// All threads; the number of experts that are named.  Experts out of range are not.
__device__ __forceinline__ int find_named(const FewParams& p, FewSchedule& s) {
  if (threadIdx.x < kFewWords) s.named[threadIdx.x] = 0;
  if (threadIdx.x == 0) s.rows = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.slots; i += kFewThreads) {
    const uint32_t e = (uint32_t)p.a.chosen[i];
    if (e < (uint32_t)p.a.experts) atomicOr(&s.named[e / 32], 1u << (e % 32));
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  return __shfl(wave_prefix(lane < kFewWords ? __popc(s.named[lane]) : 0), 63);
}

// The which-th of the experts that are named, and its slots (in any order: a token's results do not depend on its place).
__device__ __forceinline__ void gather_slots(const FewParams& p, FewSchedule& s, int which) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    uint32_t word = lane < kFewWords ? s.named[lane] : 0u;
    const int upto = wave_prefix(__popc(word)), before = upto - __popc(word);
    if (which >= before && which < upto) {
      for (int i = before; i < which; ++i) word &= word - 1;
      s.expert = lane * 32 + __ffs(word) - 1;
    }
  }
  __syncthreads();
  const int expert = s.expert;
  for (int i = threadIdx.x; i < p.slots; i += kFewThreads)
    if (p.a.chosen[i] == expert) s.slot[atomicAdd(&s.rows, 1)] = i;
  __syncthreads();
}

// One wave's stream: its share of the depth of a strip of weights against up to 16 * MT rows.
//   NT   four tiles of 16 weight rows, two from `first` and two from `second` on; 64 deep at a time
//   NN   128 columns, in each lane 8 neighbouring ones; 32 deep at a time
// PARTS: the rows come as the sum of this many (high, or high and low).
template <int DT, bool NT, int MT, int PARTS>
struct Stream {
  static constexpr int DEPTH = NT ? 64 : 32;      // of a step
  static constexpr int TILES = NT ? 4 : 8;        // of 16 weight columns
  static constexpr int XS = NT ? 2 : 1;           // loads of a row per step

  struct Step {
    u32x4 w[8];
    u32x4 x[MT][PARTS][XS];
  };

  const uint16_t *first, *second;   // the same in all lanes: where the strip's columns begin, at depth 0
  uint32_t at[NT ? 4 : 1];          // this lane's offset from there, in bytes
  uint32_t pitch;                   // NN: bytes from one row of the depth to the next
  int width;                        // NN: columns this lane may read, 8 or (of a matrix narrower than 8) fewer
  const uint16_t* x[PARTS];         // the rows, the same in all lanes,
  uint32_t row[MT];                 // ... and this lane's of them, as offsets in bytes
  int depth;
  f32x4 acc[TILES][MT];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  __device__ __forceinline__ const uint16_t* lane_row(int p, int k, uint32_t offset) const {
    return reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(x[p] + k) + offset);
  }

  __device__ __forceinline__ void load(Step& s, int k) const {
    const int q = (threadIdx.x & 63) >> 4;
    if constexpr (NT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* base = reinterpret_cast<const char*>((i < 2 ? first : second) + k);
#pragma unroll
        for (int h = 0; h < 2; ++h) s.w[2 * i + h] = load8(reinterpret_cast<const uint16_t*>(base + at[i]) + 8 * h);
      }
    } else {
      const char* base = reinterpret_cast<const char*>(first) + (uint64_t)k * pitch;
#pragma unroll
      for (int i = 0; i < 8; ++i) s.w[i] = load8(reinterpret_cast<const uint16_t*>(base + (uint64_t)i * pitch + at[0]));
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int h = 0; h < XS; ++h) s.x[m][p][h] = load8(lane_row(p, k, row[m] + q * 16 * XS) + 8 * h);
  }

  // ... where the depth ends inside, or the matrix is narrower than a lane's columns
  __device__ __forceinline__ void load_within(Step& s, int k) const {
    const int q = (threadIdx.x & 63) >> 4;
    if constexpr (NT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t* base = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(i < 2 ? first : second) + at[i]);
#pragma unroll
        for (int h = 0; h < 2; ++h) s.w[2 * i + h] = load8_within(base - q * 16, k + q * 16 + 8 * h, depth);
      }
    } else {
      const char* base = reinterpret_cast<const char*>(first) + (uint64_t)k * pitch;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s.w[i] = u32x4{0u, 0u, 0u, 0u};
        if (k + q * 8 + i < depth) s.w[i] = load8_within(reinterpret_cast<const uint16_t*>(base + (uint64_t)i * pitch + at[0]), 0, width);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int h = 0; h < XS; ++h) s.x[m][p][h] = load8_within(lane_row(p, 0, row[m]), k + q * 8 * XS + 8 * h, depth);
  }

  __device__ __forceinline__ void multiply(const Step& s) {
    if constexpr (NT) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
              acc[i][m] = mfma_16x16x32<DT>(__builtin_bit_cast(bf16x8, s.w[2 * i + h]), __builtin_bit_cast(bf16x8, s.x[m][p][h]), acc[i][m]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(s.w[2 * i + 1][j / 2], s.w[2 * i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < PARTS; ++p)
            acc[j][m] = mfma_16x16x32<DT>(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, s.x[m][p][0]), acc[j][m]);
      }
    }
  }

  // Steps begin .. end - 1 of the depth, every kFewWaves-th of them; two in flight.
  __device__ __forceinline__ void run(int begin, int end) {
    const bool narrow = !NT && width < 8;
    const int whole = narrow ? begin : min(end, depth / DEPTH);   // steps that end inside the depth
    int step = begin + uniform((int)(threadIdx.x >> 6));
    Step s0, s1;
    if (step < whole) load(s0, step * DEPTH);
    if (step + kFewWaves < whole) load(s1, (step + kFewWaves) * DEPTH);
    while (step < whole) {
      multiply(s0);
      if (step + 2 * kFewWaves < whole) load(s0, (step + 2 * kFewWaves) * DEPTH);
      step += kFewWaves;
      if (step >= whole) break;
      multiply(s1);
      if (step + 2 * kFewWaves < whole) load(s1, (step + 2 * kFewWaves) * DEPTH);
      step += kFewWaves;
    }
    for (; step < end; step += kFewWaves) {
      load_within(s0, step * DEPTH);
      multiply(s0);
    }
  }
};

// The waves' sums through LDS, 4 KiB of each wave at a time: NT its four tiles, NN the first or second 64 of its columns.
template <bool NT>
struct Exchange {
  static constexpr int ROUNDS = NT ? 1 : 2;
  f32x4* lds;   // [kFewWaves][256]

  template <typename S>
  __device__ __forceinline__ void put(const S& s, int m, int round) const {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if constexpr (NT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) lds[wave * 256 + i * 64 + lane] = s.acc[i][m];
    } else {
      if ((lane >> 5) == round)
#pragma unroll
        for (int j = 0; j < 8; ++j) lds[wave * 256 + j * 32 + (lane & 31)] = s.acc[j][m];
    }
  }
  // Sum over the waves of weight column `column` (NT: of 64; NN: of 16 blocks of 8 lanes' columns, block i and column j of it) and row `token`
  __device__ __forceinline__ float get(int item, int r) const {
    const float* from = reinterpret_cast<const float*>(lds) + item * 4 + r;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) sum += from[w * 1024];
    return sum;
  }
  __device__ __forceinline__ float column_of_tiles(int column, int token) const {   // NT
    return get((column >> 4) * 64 + ((column >> 2) & 3) * 16 + token, column & 3);
  }
  __device__ __forceinline__ float column_of_block(int block, int j, int token) const {   // NN, block of this round's 8
    return get(j * 32 + (block >> 2) * 16 + token, block & 3);
  }
};

template <int DT, bool NT, int MT>
__global__ __launch_bounds__(kFewThreads, MT == 1 ? 4 : 2) void few_gate_up_kernel(FewParams p) {
  using S = Stream<DT, NT, MT, 1>;
  constexpr int COLUMNS = NT ? 32 : 64;   // of h
  __shared__ FewSchedule schedule;
  __shared__ f32x4 lds[kFewWaves * 256];
  const FewTokensArgs& a = p.a;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  if (blockIdx.x == 0)   // the second kernel's counters
    for (int i = threadIdx.x; i < p.counters; i += kFewThreads) p.arrivals[i] = 0;
  const int named = find_named(p, schedule);
  const int which = blockIdx.x / p.tiles, column0 = (blockIdx.x - which * p.tiles) * COLUMNS;
  if (which >= named) return;
  gather_slots(p, schedule, which);
  const int rows = uniform(schedule.rows), ffn = a.ffn, hidden = a.hidden;
  const uint16_t* w = static_cast<const uint16_t*>(a.w13) + (uint64_t)uniform(schedule.expert) * 2 * ffn * hidden;
  S s;
  s.x[0] = static_cast<const uint16_t*>(a.x);
  s.depth = hidden;
  s.width = 8;
  if constexpr (NT) {
    s.first = w + (uint64_t)column0 * hidden;
    s.second = s.first + (uint64_t)ffn * hidden;
#pragma unroll
    for (int i = 0; i < 4; ++i)   // (rows past the last: the last one's, not stored)
      s.at[i] = (uint32_t)(min(16 * (i & 1) + c, ffn - 1 - column0)) * (uint32_t)hidden * 2 + q * 32;
  } else {
    // lanes of even number have columns of gate, of odd number the same of up; blocks past the last column move back to it
    const int column = ffn < 8 ? 0 : min(column0 + c / 2 * 8, ffn - 8);
    s.width = min(ffn, 8);
    s.first = w;
    s.pitch = (uint32_t)ffn * 4;
    s.at[0] = q * 8 * s.pitch + (uint32_t)(column + (c & 1) * ffn) * 2;
  }
  const Exchange<NT> exchange{lds};
  for (int row0 = 0; row0 < rows; row0 += 16 * MT) {
#pragma unroll
    for (int m = 0; m < MT; ++m)   // (places past the last row: the last one's, not stored)
      s.row[m] = (uint32_t)(schedule.slot[min(row0 + 16 * m + c, rows - 1)] / a.top_k) * (uint32_t)hidden * 2;
    s.clear();
    s.run(0, (hidden + S::DEPTH - 1) / S::DEPTH);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (row0 + 16 * m >= rows) break;
#pragma unroll
      for (int round = 0; round < Exchange<NT>::ROUNDS; ++round) {
        __syncthreads();
        exchange.put(s, m, round);
        __syncthreads();
        const int token = threadIdx.x >> 5, n = threadIdx.x & 31;   // of 16 rows, of 32 columns
        float gate, up;
        int column;
        bool mine;
        if constexpr (NT) {
          gate = exchange.column_of_tiles(n, token);
          up = exchange.column_of_tiles(32 + n, token);
          column = column0 + n;
          mine = column < ffn;
        } else {
          const int block = n >> 3, start = column0 + round * 32 + block * 8;
          gate = exchange.column_of_block(2 * block, n & 7, token);
          up = exchange.column_of_block(2 * block + 1, n & 7, token);
          column = (ffn < 8 ? 0 : min(start, ffn - 8)) + (n & 7);
          mine = column >= start && column < ffn;   // (a block that moved back: its own columns only)
        }
        const int row = row0 + 16 * m + token;
        if (mine && row < rows) {
          const float h = gate / (1.0f + expf(-gate)) * up;
          const uint16_t high = round_bits<DT>(h);
          const float rest = h - widen_bits<DT>(high);
          const uint64_t to = (uint64_t)schedule.slot[row] * p.ffn_pitch + column;
          p.high[to] = high;
          p.low[to] = fabsf(rest) < INFINITY ? round_bits<DT>(rest) : uint16_t(0);   // (an infinite h has no rest)
        }
      }
    }
  }
}

template <int DT, bool NT, int MT>
__global__ __launch_bounds__(kFewThreads, 2) void few_down_kernel(FewParams p) {
  using S = Stream<DT, NT, MT, 2>;
  constexpr int COLUMNS = NT ? 64 : 128;
  __shared__ FewSchedule schedule;
  __shared__ f32x4 lds[kFewWaves * 256];
  __shared__ int32_t arrived;
  const FewTokensArgs& a = p.a;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int named = find_named(p, schedule), hidden = a.hidden, ffn = a.ffn;
  const int arrivals = named * p.pieces;
  int tile, left = 0;
  if (named > 0) {
    tile = blockIdx.x / arrivals;
    left = blockIdx.x - tile * arrivals;
  } else {
    tile = blockIdx.x;
  }
  if (tile >= p.tiles) return;
  const int column0 = tile * COLUMNS;
  if (named > 0) {
    const int which = left / p.pieces, piece = left - which * p.pieces;
    gather_slots(p, schedule, which);
    const int rows = uniform(schedule.rows);
    const uint16_t* w = static_cast<const uint16_t*>(a.w2) + (uint64_t)uniform(schedule.expert) * ffn * hidden;
    S s;
    s.x[0] = p.high, s.x[1] = p.low;
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
    const int steps = (ffn + S::DEPTH - 1) / S::DEPTH, begin = (int)((int64_t)steps * piece / p.pieces);
    const int end = (int)((int64_t)steps * (piece + 1) / p.pieces);
    const Exchange<NT> exchange{lds};
    float* parts = p.parts + (uint64_t)piece * p.slots * hidden;
    for (int row0 = 0; row0 < rows; row0 += 16 * MT) {
#pragma unroll
      for (int m = 0; m < MT; ++m) s.row[m] = (uint32_t)schedule.slot[min(row0 + 16 * m + c, rows - 1)] * (uint32_t)p.ffn_pitch * 2;
      s.clear();
      s.run(begin, end);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (row0 + 16 * m >= rows) break;
#pragma unroll
        for (int round = 0; round < Exchange<NT>::ROUNDS; ++round) {
          __syncthreads();
          exchange.put(s, m, round);
          __syncthreads();
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int token = half * 8 + (threadIdx.x >> 6), n = threadIdx.x & 63;   // of 16 rows, of 64 columns
            float y;
            int column;
            bool mine;
            if constexpr (NT) {
              y = exchange.column_of_tiles(n, token);
              column = column0 + n;
              mine = column < hidden;
            } else {
              const int start = column0 + round * 64 + (n >> 3) * 8;
              y = exchange.column_of_block(n >> 3, n & 7, token);
              column = (hidden < 8 ? 0 : min(start, hidden - 8)) + (n & 7);
              mine = column >= start && column < hidden;
            }
            const int row = row0 + 16 * m + token;
            if (mine && row < rows) {
              const int slot = schedule.slot[row];
              // (device scope: written to and read from where all XCDs see it, without a fence that empties whole L2s)
              __hip_atomic_store(&parts[(uint64_t)slot * hidden + column], y * a.weights[slot], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
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
  // The strip's sums, in the order of a token's experts and of the pieces.
  uint16_t* out = static_cast<uint16_t*>(a.out);
  const int columns = min(COLUMNS, hidden - column0);
  for (int i = threadIdx.x; i < a.tokens * COLUMNS; i += kFewThreads) {
    const int token = i / COLUMNS, n = i % COLUMNS;
    if (n >= columns) continue;
    float sum = 0.0f;
    for (int j = 0; j < a.top_k; ++j) {
      const int slot = token * a.top_k + j;
      if ((uint32_t)a.chosen[slot] >= (uint32_t)a.experts) continue;
      for (int piece = 0; piece < p.pieces; ++piece)
        sum += __hip_atomic_load(&p.parts[((uint64_t)piece * p.slots + slot) * hidden + column0 + n], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    out[(uint64_t)token * hidden + column0 + n] = round_bits<DT>(sum);
  }
}

struct FewPlan {
  int64_t slots, named, up_tiles, down_tiles, pieces, ffn_pitch;
  uint64_t arrivals_bytes, h_bytes, parts_bytes;
};

// Workgroups that keep the device busy: two rounds of two on each of 256 compute units.
constexpr int64_t kFewWorkgroups = 1024;

FewPlan few_plan(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool nt) {
  FewPlan f;
  f.slots = tokens * top_k;
  f.named = f.slots < experts ? f.slots : experts;   // at most
  f.up_tiles = (ffn + (nt ? 31 : 63)) / (nt ? 32 : 64);
  f.down_tiles = (hidden + (nt ? 63 : 127)) / (nt ? 64 : 128);
  f.ffn_pitch = (ffn + 7) / 8 * 8;
  // the depth of down in pieces where its strips alone are too few, each at least two steps of every wave
  const int64_t steps = (ffn + (nt ? 63 : 31)) / (nt ? 64 : 32);
  f.pieces = 1;
  while (f.pieces < 16 && f.named * f.down_tiles * f.pieces < kFewWorkgroups && steps >= 2 * f.pieces * 2 * kFewWaves) f.pieces *= 2;
  f.arrivals_bytes = (uint64_t)(f.down_tiles * 4 + 255) / 256 * 256;
  f.h_bytes = ((uint64_t)f.slots * f.ffn_pitch * 2 + 255) / 256 * 256;
  f.parts_bytes = (uint64_t)f.pieces * f.slots * hidden * 4;
  return f;
}

template <int DT, bool NT, int MT>
hipError_t launch_few(const FewTokensArgs& a, const FewPlan& f, hipStream_t stream) {
  FewParams p;
  p.a = a;
  p.slots = (int32_t)f.slots;
  p.ffn_pitch = (int32_t)f.ffn_pitch;
  char* at = static_cast<char*>(a.scratch);
  p.arrivals = reinterpret_cast<int32_t*>(at);
  p.high = reinterpret_cast<uint16_t*>(at + f.arrivals_bytes);
  p.low = reinterpret_cast<uint16_t*>(at + f.arrivals_bytes + f.h_bytes);
  p.parts = reinterpret_cast<float*>(at + f.arrivals_bytes + 2 * f.h_bytes);
  p.tiles = (int32_t)f.up_tiles;
  p.pieces = (int32_t)f.pieces;
  p.counters = (int32_t)f.down_tiles;
  hipLaunchKernelGGL((few_gate_up_kernel<DT, NT, MT>), dim3((uint32_t)(f.named * f.up_tiles)), dim3(kFewThreads), 0, stream, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  p.tiles = (int32_t)f.down_tiles;
  hipLaunchKernelGGL((few_down_kernel<DT, NT, MT>), dim3((uint32_t)(f.named * f.down_tiles * f.pieces)), dim3(kFewThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

bool few_tokens_fits(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool trans_b) {
  const FewPlan f = few_plan(tokens, experts, top_k, hidden, ffn, trans_b);
  const int64_t most = (int64_t(1) << 32) / kFewThreads;   // (threads of a launch are counted in 32 bits)
  return f.named * f.up_tiles < most && f.named * f.down_tiles * f.pieces < most && f.slots * f.ffn_pitch * 2 < (int64_t(1) << 32);
}

uint64_t few_tokens_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool trans_b) {
  const FewPlan f = few_plan(tokens, experts, top_k, hidden, ffn, trans_b);
  return f.arrivals_bytes + 2 * f.h_bytes + f.parts_bytes;
}

hipError_t few_tokens(const FewTokensArgs& a, hipStream_t stream) {
  const FewPlan f = few_plan(a.tokens, a.experts, a.top_k, a.hidden, a.ffn, a.trans_b);
  const bool one = a.tokens <= 16;   // rows of an expert fit one matrix tile (unless a token names an expert twice)
#define GG_LAUNCH(DT)                                                                                            \
  (a.trans_b ? (one ? launch_few<DT, true, 1>(a, f, stream) : launch_few<DT, true, 2>(a, f, stream))             \
             : (one ? launch_few<DT, false, 1>(a, f, stream) : launch_few<DT, false, 2>(a, f, stream)))
  return a.dt == kBF16 ? GG_LAUNCH(kBF16) : GG_LAUNCH(kF16);
#undef GG_LAUNCH
}

}  // namespace gg
