// Few rows against a stream of weights: what the operators that read each weight for a handful of rows are built on.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gmm_kernel.hpp"

namespace gg {

// Waves that share the depth of a strip of weights, in turns.
constexpr int kFewWaves = 4;
constexpr int kFewThreads = kFewWaves * 64;

// 8 elements on any boundary.
struct __attribute__((packed, aligned(2))) Packed8 {
  u32x4 v;
};
__device__ __forceinline__ u32x4 load8(const uint16_t* p) { return reinterpret_cast<const Packed8*>(p)->v; }

// ... at a base that all lanes share, and an offset of each in bytes.  The empty asm hides where the two come from: without it the compiler
// keeps one 64-bit address per load in vector registers from step to step.
__device__ __forceinline__ u32x4 load8_at(const void* base, uint32_t offset, int further = 0) {
  using Bytes = const __attribute__((address_space(1))) char*;
  using Eight = const __attribute__((address_space(1))) Packed8*;
  uint64_t at = (uint64_t)uniform_ptr(static_cast<const char*>(base));
  asm("" : "+s"(at), "+v"(offset));
  return ((Eight)((Bytes)at + offset + further))->v;
}
// ... one dword of them, on a boundary of 4 bytes
__device__ __forceinline__ uint32_t load_dword_at(const void* base, uint32_t offset) {
  using Bytes = const __attribute__((address_space(1))) char*;
  using Dword = const __attribute__((address_space(1))) uint32_t*;
  uint64_t at = (uint64_t)uniform_ptr(static_cast<const char*>(base));
  asm("" : "+s"(at), "+v"(offset));
  return *(Dword)((Bytes)at + offset);
}
__device__ __forceinline__ void store8(uint16_t* p, u32x4 v) { reinterpret_cast<Packed8*>(p)->v = v; }
__device__ __forceinline__ void store8_at(void* base, uint32_t offset, u32x4 v, int further = 0) {
  using Bytes = __attribute__((address_space(1))) char*;
  using Eight = __attribute__((address_space(1))) Packed8*;
  uint64_t at = (uint64_t)uniform_ptr(static_cast<const char*>(base));
  asm("" : "+s"(at), "+v"(offset));
  ((Eight)((Bytes)at + offset + further))->v = v;
}

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

// v in two numbers of the type: rounded, but not past the largest, and what that left: finite both where v is (float16's callers keep it below
// 2^15).  Of an infinity, and of NaN, the second is one.
template <int DT>
__device__ __forceinline__ void split(float v, uint32_t& high, uint32_t& low) {
  constexpr float LARGEST = DT == kBF16 ? 0x1.fep127f : 65504.0f;
  high = round_bits<DT>(__builtin_amdgcn_fmed3f(v, -LARGEST, LARGEST));
  low = round_bits<DT>(v - widen_bits<DT>((uint16_t)high));
}

// One wave's stream: its share of the depth of a strip of weights against up to 16 * MT rows.
//   NT   tiles of 16 weight rows, the first half of them from `first` and the others from `second` on; 64 deep at a time
//   NN   128 columns, in each lane 8 neighbouring ones; 32 deep at a time
// ODD (NT): rows may begin on any element.  Loads of 16 bytes that are not on a boundary of 4 take three times as long, so a lane loads from the
// boundary before its 16 elements on, one dword more, and shifts; each of those dwords holds an element of its own, so that nothing is read that
// could not be.  Without and with it, us: 8192 rows of 4097 against adapters of rank 64 117, 52 (of 4098: 41); gate and up of two experts, 4097 ->
// 14337, 202, 137 (of 4098: 101); one row 4.3, 4.4.  NN has whole rows of 256 bytes to an instruction, and loses an eighth.
// SCALED (float16): a row's elements are kept as multiples of a power of two of each block of them, and are brought to one that the whole row
// shares on their way into the instructions.
template <int DT, bool NT, int NT_TILES, int MT, bool ODD = false, bool SCALED = false>
struct Stream {
  static_assert(NT || !ODD, "");
  static_assert(DT == kF16 || !SCALED, "");
  static constexpr int BLOCK = NT ? 32 : 64;      // SCALED: elements of a block
  static constexpr int DEPTH = NT ? 64 : 32;      // of a step
  static constexpr int TILES = NT ? NT_TILES : 8;        // of 16 weight columns
  static constexpr int XS = NT ? 2 : 1;           // loads of a row per step

  struct Step {
    u32x4 w[NT ? 2 * TILES : 8];
    u32x4 x[MT][XS];
    uint32_t w_end[ODD ? TILES : 1], x_end[ODD ? MT : 1];
    int32_t unit[SCALED ? MT : 1];
  };

  const uint16_t *first, *second;   // the same in all lanes: where the strip's columns begin, at depth 0
  uint32_t at[NT ? TILES : 1];          // this lane's offset from there, in bytes
  uint32_t pitch;                   // NN: bytes from one row of the depth to the next
  int width;                        // NN: columns this lane may read, 8 or (of a matrix narrower than 8) fewer
  const uint16_t* x;                // the rows, the same in all lanes,
  uint32_t row[MT];                 // ... and where in them this lane's step 0 begins, in bytes (set_row)
  uint32_t w_turn[ODD ? TILES : 1], x_turn[ODD ? MT : 1];   // ODD: bytes from the boundary to there, 0 or 2 (`at` and `row` are the boundary's)
  const int32_t* units;             // SCALED: the exponents of the rows' blocks, the same in all lanes,
  uint32_t unit_row[SCALED ? MT : 1];   // ... where in them those of this lane's row begin, in bytes,
  int32_t row_unit[SCALED ? MT : 1];    // ... and the exponent that the row is brought to, none of its blocks' being larger
  int depth;
  f32x4 acc[TILES][MT];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  static __device__ __forceinline__ const uint16_t* boundary(const uint16_t* p) {
    return ODD ? reinterpret_cast<const uint16_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3)) : p;
  }
  static __device__ __forceinline__ void turn(const uint16_t* base, uint32_t& offset, uint32_t& bytes) {
    offset += (uint32_t)(reinterpret_cast<uintptr_t>(base) & 2);
    bytes = offset & 2;
    offset -= bytes;
  }
  // the lane's row of tile m begins `offset` bytes into x
  __device__ __forceinline__ void set_row(int m, uint32_t offset) {
    row[m] = offset + ((threadIdx.x & 63) >> 4) * 16 * XS;
    if constexpr (ODD) turn(x, row[m], x_turn[m]);
  }
  __device__ __forceinline__ const uint16_t* matrix(int i) const { return 2 * i < TILES ? first : second; }
  // once `at`, first and second are set
  __device__ __forceinline__ void set_weights() {
    if constexpr (ODD) {
#pragma unroll
      for (int i = 0; i < TILES; ++i) turn(matrix(i), at[i], w_turn[i]);
    }
  }

  __device__ __forceinline__ void load_weights(Step& s, int k) const {
    if constexpr (NT) {
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) s.w[2 * i + h] = load8_at(boundary(matrix(i)) + k, at[i], 16 * h);
      if constexpr (ODD) {   // (where nothing is to be shifted: the last dword again, not one past it)
#pragma unroll
        for (int i = 0; i < TILES; ++i) s.w_end[i] = load_dword_at(boundary(matrix(i)) + k, at[i] + 28 + 2 * w_turn[i]);
      }
    } else {
      const char* base = reinterpret_cast<const char*>(first) + (uint64_t)k * pitch;
#pragma unroll
      for (int i = 0; i < 8; ++i) s.w[i] = load8_at(base + (uint64_t)i * pitch, at[0]);
    }
  }
  __device__ __forceinline__ void load_rows(Step& s, int k) const {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < XS; ++h) s.x[m][h] = load8_at(boundary(x) + k, row[m], 16 * h);
    if constexpr (ODD) {
#pragma unroll
      for (int m = 0; m < MT; ++m) s.x_end[m] = load_dword_at(boundary(x) + k, row[m] + 28 + 2 * x_turn[m]);
    }
    if constexpr (SCALED) {   // (a lane's elements of a step lie in one block)
#pragma unroll
      for (int m = 0; m < MT; ++m) s.unit[m] = (int32_t)load_dword_at(units + (uint32_t)k / BLOCK, unit_row[m] + (NT ? (threadIdx.x & 32) / 8 : 0));
    }
  }

  // ... where the depth ends inside, or the matrix is narrower than a lane's columns
  __device__ __forceinline__ void load_within(Step& s, int k) const {
    const int q = (threadIdx.x & 63) >> 4;
    if constexpr (NT) {
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const uint16_t* base = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(boundary(matrix(i))) + at[i]);
        if constexpr (ODD) base += w_turn[i] / 2;
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
    for (int m = 0; m < MT; ++m) {
      const uint16_t* from = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(boundary(x)) + row[m]) - q * 8 * XS;
      if constexpr (ODD) from += x_turn[m] / 2;
#pragma unroll
      for (int h = 0; h < XS; ++h) s.x[m][h] = load8_within(from, k + q * 8 * XS + 8 * h, depth);
      if constexpr (SCALED) s.unit[m] = units[unit_row[m] / 4 + min(k + q * 8 * XS, depth - 1) / BLOCK];   // (of zeros past the end: the last one's)
    }
  }

  // ODD, of what load_weights and load_rows brought: from the boundary on -> from the lane's first element on
  static __device__ __forceinline__ void shift(u32x4& low, u32x4& high, uint32_t end, uint32_t bytes) {
    const uint32_t d[9] = {low[0], low[1], low[2], low[3], high[0], high[1], high[2], high[3], end};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      low[j] = __builtin_amdgcn_alignbyte(d[j + 1], d[j], bytes);
      high[j] = __builtin_amdgcn_alignbyte(d[j + 5], d[j + 4], bytes);
    }
  }
  __device__ __forceinline__ void shift(Step& s) const {
    if constexpr (ODD) {
#pragma unroll
      for (int i = 0; i < TILES; ++i) shift(s.w[2 * i], s.w[2 * i + 1], s.w_end[i], w_turn[i]);
#pragma unroll
      for (int m = 0; m < MT; ++m) shift(s.x[m][0], s.x[m][1], s.x_end[m], x_turn[m]);
    }
  }

  // SCALED: the rows' elements times 2^(their block's exponent - the row's), a power of two not above 1, in two factors: elements are below 2^15, and
  // down to 2^-39 of that the product is a number of float16, where the power itself is not.  Blocks of one row seldom need the second.
  __device__ __forceinline__ void scale(Step& s) const {
    if constexpr (SCALED) {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        auto times = [&](int power) {   // (below -24: to zero)
          const _Float16 factor = (_Float16)ldexpf(1.0f, power);
#pragma unroll
          for (int h = 0; h < XS; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t pair = s.x[m][h][j];
              s.x[m][h][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pair) * f16x2{factor, factor});
            }
        };
        const int power = s.unit[m] - row_unit[m];
        times(max(power, -14));
        if (__any(power < -14)) times(max(min(power + 14, 0), -26));
      }
    }
  }

  __device__ __forceinline__ void multiply(Step& s) {
    scale(s);
    if constexpr (NT) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[i][m] = mfma_16x16x32<DT>(__builtin_bit_cast(bf16x8, s.w[2 * i + h]), __builtin_bit_cast(bf16x8, s.x[m][h]), acc[i][m]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(s.w[2 * i + 1][j / 2], s.w[2 * i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[j][m] = mfma_16x16x32<DT>(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, s.x[m][0]), acc[j][m]);
      }
    }
  }

  // Steps begin .. end - 1 of the depth, every kFewWaves-th of them, two in flight.  The first two steps' weights are asked for by
  // prepare(), which needs neither `row` nor `x`: whose rows they meet may still have to be found out.
  Step s0, s1;
  int step, whole;   // the wave's next step, and the end of those that lie inside the depth

  // `wave`: of the kFewWaves that share the strip
  __device__ __forceinline__ void prepare(int wave, int begin, int end) {
    const bool narrow = !NT && width < 8;
    whole = narrow ? begin : min(end, depth / DEPTH);
    step = begin + wave;
    if (step < whole) load_weights(s0, step * DEPTH);
    if (step + kFewWaves < whole) load_weights(s1, (step + kFewWaves) * DEPTH);
  }
  // multiply, then ask for what comes two of the wave's steps later
  __device__ __forceinline__ void advance(Step& s) {
    shift(s);
    multiply(s);
    __builtin_amdgcn_sched_barrier(0);   // (steps do not mix: their registers would not suffice)
    load_weights(s, (step + 2 * kFewWaves) * DEPTH);
    load_rows(s, (step + 2 * kFewWaves) * DEPTH);
    step += kFewWaves;
    __builtin_amdgcn_sched_barrier(0);
  }
  // `meanwhile` is called once the first loads are under way (by all threads)
  template <typename Meanwhile>
  __device__ __forceinline__ void run(int end, Meanwhile meanwhile) {
    clear();
    if (step < whole) load_rows(s0, step * DEPTH);
    if (step + kFewWaves < whole) load_rows(s1, (step + kFewWaves) * DEPTH);
    meanwhile();
    // (the loop's loads are under no condition of their own, and its first turn, whose loads came in another order, is
    // outside it: the compiler then waits for a step's own loads only, not for all)
    if (step + 3 * kFewWaves < whole) {
      advance(s0);
      advance(s1);
      while (step + 3 * kFewWaves < whole) {
        advance(s0);
        advance(s1);
      }
    }
    if (step < whole) {   // one to three steps are left, two of them loaded
      const bool third = step + 2 * kFewWaves < whole;
      shift(s0);
      multiply(s0);
      if (third) {
        load_weights(s0, (step + 2 * kFewWaves) * DEPTH);
        load_rows(s0, (step + 2 * kFewWaves) * DEPTH);
      }
      step += kFewWaves;
      if (step < whole) {
        shift(s1);
        multiply(s1);
        step += kFewWaves;
      }
      if (third) {
        shift(s0);
        multiply(s0);
        step += kFewWaves;
      }
    }
    for (; step < end; step += kFewWaves) {
      load_within(s0, step * DEPTH);
      multiply(s0);
    }
  }
  __device__ __forceinline__ void run(int end) {
    run(end, [] {});
  }
};

// Whether rows of `depth` elements of these matrices begin elsewhere than on boundaries of 4 bytes: what ODD streams are for.
inline bool on_any_element(const void* p, const void* q, int64_t depth) {
  return ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 3) != 0 || depth % 2 != 0;
}

// The waves' sums through LDS, 4 KiB of each wave at a time: NT its tiles (up to four), NN the first or second 64 of its columns.
template <bool NT>
struct Exchange {
  static constexpr int ROUNDS = NT ? 1 : 2;
  f32x4* lds;   // [waves][256]

  template <typename S>
  __device__ __forceinline__ void put(const S& s, int m, int round) const {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if constexpr (NT) {
#pragma unroll
      for (int i = 0; i < S::TILES; ++i) lds[wave * 256 + i * 64 + lane] = s.acc[i][m];
    } else {
      if ((lane >> 5) == round)
#pragma unroll
        for (int j = 0; j < 8; ++j) lds[wave * 256 + j * 32 + (lane & 31)] = s.acc[j][m];
    }
  }
  // Sums over the kFewWaves from `wave` on; `token` is a row of the 16.
  __device__ __forceinline__ float get(int wave, int item, int r) const {
    const float* from = reinterpret_cast<const float*>(lds) + wave * 1024 + item * 4 + r;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) sum += from[w * 1024];
    return sum;
  }
  __device__ __forceinline__ float column_of_tiles(int column, int token) const {   // NT
    return get(0, (column >> 4) * 64 + ((column >> 2) & 3) * 16 + token, column & 3);
  }
  __device__ __forceinline__ float column_of_block(int wave, int block, int j, int token) const {   // NN, block of this round's 8
    return get(wave, j * 32 + (block >> 2) * 16 + token, block & 3);
  }
};

// Workgroups go to the 8 XCDs in turns; tasks are dealt so that each XCD has neighbouring ones, whose strips share pages and
// blocks of memory: 128 of 256 bytes of a row each, 2 x 235 MB: 94 us in plain order, 88 so.  A permutation of 0 .. tasks - 1.
__device__ __forceinline__ uint32_t task_of_block(uint32_t block, uint32_t tasks) {
  const uint32_t xcd = block % 8, each = tasks / 8, more = tasks % 8;
  return xcd * each + (xcd < more ? xcd : more) + block / 8;
}

}  // namespace gg
