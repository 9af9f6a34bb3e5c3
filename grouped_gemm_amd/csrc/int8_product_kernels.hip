// Grouped product of 8-bit integers where groups have few rows, or sizes and addresses are any:
//
//   c[r, n] = a_scales[r] * b_scales[e, n] * sum over k of a[r, k] * b[e, n, k],   e the group of row r
//
// The sums are exact (in 32 bits, up to a depth of 131071), so that neither the order nor the pieces they are made in matter.  They are scaled by
// the column's first: weights have scales of ordinary size, and where a row's is very large or small nothing in between leaves a float's range.
//
// Few rows are bound by reading b once.  A workgroup has a strip of 64 columns of a group's b, over the whole depth or a piece of it, and a
// window of up to 16, 32 or 64 of its rows; its four waves take the depth in turns, 128 deep at a time, each with its own loads from HBM
// straight into registers, where b is the matrix instruction's first operand: 16 columns against 16 rows.  No LDS and no barrier in the
// loop; the waves' sums are added up through LDS at its end.
//
// Workgroups of one strip and neighbouring windows are neighbours, so that groups of many rows find the strip in L2.
//
// 512 rows over 128 groups, 7168 -> 4096 (3.7 GB): 0.59 ms, 6.2 TB/s, faster than a copy, which writes too; 2 rows of 2 groups, 4096 -> 28672
// (235 MB): 46 us, of which a launch, the sizes and the first loads' way from memory take 6.6.
#include "operators.hpp"

#include <algorithm>

#include "few_rows.hpp"
#include "gmm_kernel.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kStrip = 64;     // columns
constexpr int kStep = 128;     // depth

struct Int8Params {
  Int8Args a;
  int32_t strips, pieces;
};

struct __attribute__((packed, aligned(1))) Packed16 {
  u32x4 v;
};
__device__ __forceinline__ u32x4 load16(const int8_t* p) { return reinterpret_cast<const Packed16*>(p)->v; }
// ... at a base that all lanes share, and an offset of each (as load8_at)
__device__ __forceinline__ u32x4 load16_at(const int8_t* base, uint32_t offset, int further) {
  using Bytes = const __attribute__((address_space(1))) char*;
  using Sixteen = const __attribute__((address_space(1))) Packed16*;
  uint64_t at = (uint64_t)uniform_ptr(reinterpret_cast<const char*>(base));
  asm("" : "+s"(at), "+v"(offset));
  return ((Sixteen)((Bytes)at + offset + further))->v;
}

// All of a row of fewer than 16, and zeros.
__device__ __noinline__ u32x4 load_short(const int8_t* row, int depth) {
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll 1
  for (int i = depth - 1; i >= 0; --i) {
#pragma unroll
    for (int d = 3; d > 0; --d) v[d] = v[d] << 8 | v[d - 1] >> 24;
    v[0] = v[0] << 8 | (uint8_t)row[i];
  }
  return v;
}
// Where elements k .. k + 15 are wanted of a row that ends before them, its last 16 are read (of a shorter row all): those before k are to meet
// zeros, one operand's are cleared.
__device__ __forceinline__ u32x4 without_before(u32x4 v, int k, int depth) {
  const int cut = k - min(k, max(depth - 16, 0));   // elements
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int gone = cut - 4 * d;
    v[d] &= gone <= 0 ? ~0u : (gone >= 4 ? 0u : ~0u << (8 * gone));
  }
  return v;
}

// One wave's stream: its share of the depth of a strip against up to 16 * MT rows.  A lane loads 32 neighbouring elements of a row of each
// operand, in two halves; which depth meets in which instruction is free as long as it is the same in both.
// ODD: rows may begin on any element.  Loads of 16 bytes that are not on a boundary of 4 are slow, so a lane takes what is from the boundary before
// its 32 elements on, and one dword more, and shifts; each dword that is loaded holds an element of the lane's own, so that nothing is read that could not be.
// The one more is the first of the lane that has the next 32 of the row, so that only the lanes with a step's last 32 load it, where there are registers
// for that (up to 32 rows; the other lanes' loads are out of range and reach no memory).  A load by all lanes costs as much as one of 16 bytes
// each: 8 rows of 8 groups, 4095 -> 14336 85 us, so 71 (4092: 57); 512 of 128, 2047 -> 1408 107 and 92.5 (2044: 78).  64 rows spill: 600 of 8, 1061 -> 2898 38 in place of 27.
template <int MT, bool ODD>
struct Int8Stream {
  static constexpr int TILES = kStrip / 16;
  struct Step {
    u32x4 w[TILES][2], x[MT][2];
    uint32_t w_end[ODD ? TILES : 1], x_end[ODD ? MT : 1];
  };

  const int8_t *w, *x;              // the strip and the window, the same in all lanes; ODD: the boundary before
  uint32_t w_at[TILES], x_at[MT];   // where in them this lane's elements of step 0 begin; ODD: ... of the boundary before
  uint32_t w_turn[ODD ? TILES : 1], x_turn[ODD ? MT : 1];   // ODD: elements from there
  static constexpr bool FROM_NEIGHBOUR = ODD && MT < 4;
  __amdgpu_buffer_rsrc_t w_ends, x_ends;                    // FROM_NEIGHBOUR: what the dwords behind are loaded by
  static constexpr uint32_t kNowhere = 0x80000000u;         // out of their range
  int depth;
  i32x4 acc[TILES][MT];

  static __device__ __forceinline__ const int8_t* boundary(const int8_t* p) {
    return ODD ? reinterpret_cast<const int8_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3)) : p;
  }
  // columns and rows past the last: the last one's, not stored
  __device__ __forceinline__ void setup(const int8_t* strip, int columns, const int8_t* window, int rows, int depth_) {
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    depth = depth_;
    w = boundary(strip), x = boundary(window);
    if constexpr (FROM_NEIGHBOUR) w_ends = make_rsrc(w, kNowhere - 1), x_ends = make_rsrc(x, kNowhere - 1);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      w_at[i] = (uint32_t)min(16 * i + c, columns - 1) * (uint32_t)depth + q * 32;
      if constexpr (ODD) turn(strip, w_at[i], w_turn[i]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      x_at[m] = (uint32_t)min(16 * m + c, rows - 1) * (uint32_t)depth + q * 32;
      if constexpr (ODD) turn(window, x_at[m], x_turn[m]);
    }
  }
  static __device__ __forceinline__ void turn(const int8_t* base, uint32_t& at, uint32_t& elements) {
    at += (uint32_t)(reinterpret_cast<uintptr_t>(base) & 3);
    elements = at & 3;
    at -= elements;
  }

  __device__ __forceinline__ void load(Step& s, int k) const {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.w[i][h] = load16_at(w + k, w_at[i], 16 * h);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.x[m][h] = load16_at(x + k, x_at[m], 16 * h);
    // (not where nothing is to be shifted: there may be nothing)
    if constexpr (FROM_NEIGHBOUR) {
      const bool last = (threadIdx.x & 63) >= 48;
#pragma unroll
      for (int i = 0; i < TILES; ++i) s.w_end[i] = __builtin_amdgcn_raw_buffer_load_b32(w_ends, last && w_turn[i] != 0 ? w_at[i] + 32 : kNowhere, k, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) s.x_end[m] = __builtin_amdgcn_raw_buffer_load_b32(x_ends, last && x_turn[m] != 0 ? x_at[m] + 32 : kNowhere, k, 0);
    } else if constexpr (ODD) {
#pragma unroll
      for (int i = 0; i < TILES; ++i) s.w_end[i] = load_dword_at(w + k, w_at[i] + (w_turn[i] != 0 ? 32 : 28));
#pragma unroll
      for (int m = 0; m < MT; ++m) s.x_end[m] = load_dword_at(x + k, x_at[m] + (x_turn[m] != 0 ? 32 : 28));
    }
  }
  // ... where the depth ends inside
  __device__ __forceinline__ void load_within(Step& s, int k) const {
    const int q = (threadIdx.x & 63) >> 4;
    auto each = [&](auto get) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k + q * 32 + 16 * h;
#pragma unroll
        for (int i = 0; i < TILES; ++i) s.w[i][h] = get(w + w_at[i] + (ODD ? w_turn[i] : 0u) - q * 32, at);
#pragma unroll
        for (int m = 0; m < MT; ++m) s.x[m][h] = without_before(get(x + x_at[m] + (ODD ? x_turn[m] : 0u) - q * 32, at), at, depth);
      }
    };
    if (depth >= 16) {
      each([&](const int8_t* row, int at) { return load16(row + min(at, depth - 16)); });
    } else {
      each([&](const int8_t* row, int) { return load_short(row, depth); });
    }
  }

  // ODD, of what load brought: from the boundary on -> from the lane's first element on
  static __device__ __forceinline__ void shift(u32x4 (&v)[2], uint32_t end, uint32_t elements) {
    if constexpr (FROM_NEIGHBOUR) {
      const int lane = threadIdx.x & 63;
      const uint32_t next = (uint32_t)__builtin_amdgcn_ds_bpermute((lane + 16) * 4, (int)v[0][0]);
      if (lane < 48) end = next;
    }
    const uint32_t d[9] = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3], end};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j / 4][j % 4] = __builtin_amdgcn_alignbyte(d[j + 1], d[j], elements);
  }
  __device__ __forceinline__ void shift(Step& s) const {
    if constexpr (ODD) {
#pragma unroll
      for (int i = 0; i < TILES; ++i) shift(s.w[i], s.w_end[i], w_turn[i]);
#pragma unroll
      for (int m = 0; m < MT; ++m) shift(s.x[m], s.x_end[m], x_turn[m]);
    }
  }
  __device__ __forceinline__ void multiply(const Step& s) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[i][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, s.w[i][h]), __builtin_bit_cast(i32x4, s.x[m][h]), acc[i][m], 0, 0, 0);
  }

  // Steps begin .. end - 1 of the depth, every kFewWaves-th of them, two in flight.
  __device__ __forceinline__ void run(int wave, int begin, int end) {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[i][m] = i32x4{0, 0, 0, 0};
    const int whole = min(end, depth / kStep);   // the end of the steps that lie inside the depth
    int step = begin + wave;
    Step s0, s1;
    if (step < whole) load(s0, step * kStep);
    if (step + kFewWaves < whole) load(s1, (step + kFewWaves) * kStep);
    auto advance = [&](Step& s) {   // multiply, then ask for what comes two of the wave's steps later
      shift(s);
      multiply(s);
      __builtin_amdgcn_sched_barrier(0);   // (steps do not mix: their registers would not suffice)
      load(s, (step + 2 * kFewWaves) * kStep);
      step += kFewWaves;
      __builtin_amdgcn_sched_barrier(0);
    };
    // (the loop's loads are under no condition of their own, and its first turn, whose loads came in another order, is outside it: the
    // compiler then waits for a step's own loads only, not for all)
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
      if (third) load(s0, (step + 2 * kFewWaves) * kStep);
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
      load_within(s0, step * kStep);
      multiply(s0);
    }
  }
};

// The groups of a launch, eight neighbouring ones to a lane: sizes are clamped and rows past the end dropped as the streaming kernels do.
struct Groups {
  static constexpr int OF_LANE = kMaxGroups / 64;
  uint32_t start[OF_LANE], rows[OF_LANE];   // rows of a
  uint32_t windows, before;                 // of this lane, and of those below it
  uint32_t all;                             // of all lanes
};
template <int WINDOW>
__device__ __forceinline__ Groups find_groups(const Int8Args& a, const HostSizes& hs) {
  const int lane = threadIdx.x & 63, per = (a.num_groups + 63) / 64;
  const uint32_t tokens = (uint32_t)a.tokens;
  int bad = 0;
  auto clamp = [&](int64_t v) {
    if (v < 0) bad |= kStatusNegativeSize;
    if (v > a.tokens) bad |= kStatusRowsPastEnd;
    return v < 0 ? 0u : (v > a.tokens ? tokens : (uint32_t)v);
  };
  auto add_sat = [](uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); };
  auto add = [](uint32_t x, uint32_t y) { return x + y; };
  uint32_t base = (uint32_t)a.row_base;
  if (a.sizes_dev != nullptr && a.first_group > 0) {
    uint32_t part = 0;
    for (int i = lane; i < a.first_group; i += 64) part = add_sat(part, clamp(a.sizes_dev[i]));
    base = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(part, add_sat), 63);
  }
  Groups g;
  int64_t given[Groups::OF_LANE];   // (asked for together; a lane without a group asks for the last one's)
  if (a.sizes_dev != nullptr) {
#pragma unroll
    for (int i = 0; i < Groups::OF_LANE; ++i)
      if (i < per) given[i] = a.sizes_dev[a.first_group + min(lane * per + i, a.num_groups - 1)];
  } else {
#pragma unroll
    for (int i = 0; i < Groups::OF_LANE; ++i)
      if (i < per) given[i] = hs.v[min(lane * per + i, a.num_groups - 1)];
  }
  uint32_t size[Groups::OF_LANE], sum = 0;
#pragma unroll
  for (int i = 0; i < Groups::OF_LANE; ++i) {
    size[i] = i < per && lane * per + i < a.num_groups ? clamp(given[i]) : 0u;
    sum = add_sat(sum, size[i]);
  }
  uint32_t run = wave_scan(sum, add_sat);
  if (add_sat(base, (uint32_t)__builtin_amdgcn_readlane((int)run, 63)) > tokens) bad |= kStatusRowsPastEnd;
  run = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)run, 0x138, 0xf, 0xf, false);   // wave_shr:1
  run = add_sat(base, run);
  g.windows = 0;
#pragma unroll
  for (int i = 0; i < Groups::OF_LANE; ++i) {
    g.start[i] = run < tokens ? run : tokens;
    const uint32_t left = tokens - g.start[i];
    g.rows[i] = size[i] < left ? size[i] : left;
    g.windows += (g.rows[i] + WINDOW - 1) / WINDOW;
    run = add_sat(run, size[i]);
  }
  const uint32_t upto = wave_scan(g.windows, add);
  g.before = upto - g.windows;
  g.all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  if (a.status != nullptr && blockIdx.x == 0 && threadIdx.x < 64) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) bad |= __shfl_xor(bad, d);
    if (lane == 0 && bad != 0) atomicOr(a.status, bad);
  }
  return g;
}

// The group that the u-th window belongs to, and where in it.
struct Window {
  int group, row0, rows, windows, first;   // rows of a: the group's first, and their number; windows of the group; the first of them among all
};
template <int WINDOW>
__device__ __forceinline__ Window find_window(const Int8Args& a, const Groups& g, uint32_t u) {
  const int lane = threadIdx.x & 63, per = (a.num_groups + 63) / 64;
  uint32_t at = g.before;
  Window w = {0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < Groups::OF_LANE; ++i) {
    const uint32_t n = (g.rows[i] + WINDOW - 1) / WINDOW;
    if (u >= at && u - at < n) w = {lane * per + i, (int)g.start[i], (int)g.rows[i], (int)n, (int)at};
    at += n;
  }
  const int from = __ffsll((unsigned long long)__ballot(u >= g.before && u - g.before < g.windows)) - 1;
  w.group = a.first_group + __builtin_amdgcn_readlane(w.group, from);
  w.row0 = __builtin_amdgcn_readlane(w.row0, from), w.rows = __builtin_amdgcn_readlane(w.rows, from);
  w.windows = __builtin_amdgcn_readlane(w.windows, from), w.first = __builtin_amdgcn_readlane(w.first, from);
  return w;
}

// (Two, three or four workgroups to a compute unit make no difference, 14336 -> 4096 for 2 rows: 23.7, 23.0, 23.8 us; 64 rows' sums take two.)
template <int MT, bool ODD>
__global__ __launch_bounds__(kFewThreads, MT == 1 ? 3 : 2) void int8_rows_kernel(Int8Params p, HostSizes hs) {
  constexpr int WINDOW = 16 * MT;
  __shared__ i32x4 lds[kFewWaves * 256];
  __shared__ int32_t arrived;
  const Int8Args& a = p.a;
  const int wave = uniform((int)(threadIdx.x >> 6)), depth = a.hidden_in, steps = (depth + kStep - 1) / kStep;
  const Groups groups = find_groups<WINDOW>(a, hs);
  const uint32_t of_window = (uint32_t)(p.strips * p.pieces), tasks = groups.all * of_window;   // (below 2^24: int8_rows_fit)
  if (blockIdx.x >= tasks) return;
  const uint32_t task = task_of_block(blockIdx.x, tasks);
  const Window at = find_window<WINDOW>(a, groups, task / of_window);
  // (of a group: piece by piece, window by window, strip by strip)
  const uint32_t in_group = task - (uint32_t)at.first * of_window, piece = in_group % (uint32_t)p.pieces, place = in_group / (uint32_t)p.pieces;
  const int strip = (int)(place / (uint32_t)at.windows), window = (int)place - strip * at.windows;
  const int column0 = strip * kStrip, columns = min(kStrip, a.hidden_out - column0);
  const int row0 = at.row0 + window * WINDOW, rows = min(WINDOW, at.rows - window * WINDOW);
  // A thread's results: column `mine` of rows first_row, first_row + kFewWaves, ...  Their scales come while the weights do (of 64 rows, which leave
  // no registers for them, when they are wanted).
  const int mine = threadIdx.x % kStrip, first_row = threadIdx.x / kStrip;
  static_assert(kFewThreads == kFewWaves * kStrip, "");
  const float of_column = a.b_scales[(int64_t)at.group * a.hidden_out + column0 + min(mine, columns - 1)];
  auto scale_of_row = [&](int i) { return a.a_scales[row0 + min(first_row + kFewWaves * i, rows - 1)]; };
  float of_row[MT < 4 ? 4 * MT : 1];
  if constexpr (MT < 4) {
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) of_row[i] = scale_of_row(i);
  }
  Int8Stream<MT, ODD> s;
  s.setup(a.b + ((int64_t)at.group * a.hidden_out + column0) * depth, columns, a.a + (int64_t)row0 * depth, rows, depth);
  s.run(wave, (int)((int64_t)steps * piece / p.pieces), (int)((int64_t)steps * (piece + 1) / p.pieces));
  auto store = [&](int i, int sum) {
    const float v = (float)sum * of_column * (MT < 4 ? of_row[MT < 4 ? i : 0] : scale_of_row(i));
    static_cast<uint16_t*>(a.c)[(int64_t)(row0 + first_row + kFewWaves * i) * a.hidden_out + column0 + mine] =
        a.to_f16 ? round_bits<kF16>(v) : round_bits<kBF16>(v);
  };
  int32_t* parts = a.parts + (int64_t)task / p.pieces * p.pieces * (WINDOW * kStrip);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (16 * m >= rows) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kStrip / 16; ++i) lds[wave * 256 + i * 64 + (threadIdx.x & 63)] = s.acc[i][m];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = first_row + kFewWaves * i;   // of the 16
      const int* from = reinterpret_cast<const int*>(lds) + ((mine >> 4) * 64 + ((mine >> 2) & 3) * 16 + row) * 4 + (mine & 3);
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) sum += from[w * 1024];
      if (16 * m + row >= rows || mine >= columns) continue;
      if (p.pieces == 1) {
        store(4 * m + i, sum);
      } else {
        __hip_atomic_store(parts + piece * (WINDOW * kStrip) + (16 * m + row) * kStrip + mine, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (p.pieces > 1) {
    // the last piece to arrive adds them up
    wait_vmcnt<0>();
    __syncthreads();
    if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(a.arrivals + task / p.pieces, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived == p.pieces - 1) {
      if (threadIdx.x == 0) __hip_atomic_store(a.arrivals + task / p.pieces, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // (as it was found)
#pragma unroll
      for (int i = 0; i < 4 * MT; ++i) {
        const int row = first_row + kFewWaves * i;
        if (row >= rows || mine >= columns) continue;
        int sum = 0;
        for (int q = 0; q < p.pieces; ++q)
          sum += __hip_atomic_load(parts + q * (WINDOW * kStrip) + row * kStrip + mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        store(i, sum);
      }
    }
  }
}

struct Int8Plan {
  int rows_of_window;   // in 16
  int64_t windows, strips, pieces;
};
constexpr int64_t kInt8Units = 256;   // compute units

// Windows at most: each group's last may be short.
Int8Plan int8_plan(int64_t tokens, int64_t num_groups, int64_t hidden_in, int64_t hidden_out, uint64_t workspace_bytes) {
  Int8Plan f;
  const int64_t named = std::max<int64_t>(1, std::min(tokens, num_groups));
  f.strips = (hidden_out + kStrip - 1) / kStrip;
  // Rows of a window by how many a group has on average (those that do not fit read the strip again), and fewer where such windows leave compute units.
  // us with 16, 32 and 64: 8 rows to a group (8 groups, 4096 -> 4096) 23, 24, 25; 16 31, 25, 27; 31 (64, 1023 -> 1407) 55, 46, 45; 375 (8, 2047 -> 1023)
  // 80, 60, 54; 67 (5, 2047 -> 1023: 368, 240 and 160 workgroups) 17, 14, 19; 13 (8, 1021 -> 513: 129, 99) 7.4, 8.0, 8.4.  (Pieces of the depth instead of fewer rows, where it is deep
  // enough: 1 group of 48, 4096 -> 4096 17.7 in place of 13.2, 9072 -> 5632 27.8 in place of 32.6; 8 of 12, 8192 -> 1024 25.3 and 22.4, 14336 -> 512 21.9 and 24.9.)
  f.rows_of_window = tokens <= 8 * named ? 1 : (tokens <= 24 * named ? 2 : 4);
  // (of n rows in a group, (n - 1) / window and one more)
  auto windows = [&] { return std::max<int64_t>(tokens - named, 0) / (16 * f.rows_of_window) + std::min(tokens, named); };
  while (f.rows_of_window > 1 && windows() * f.strips < kInt8Units * 3 / 4) f.rows_of_window /= 2;
  const int64_t window = 16 * f.rows_of_window;
  f.windows = windows();
  // Pieces of the depth while they are no more than the compute units, of at least four steps to a wave: b is read no faster by more workgroups,
  // and a piece is a sum to write and join.  us with whole depths, with up to 256, 512 and 1024 pieces: 1 row, 14336 -> 512 29.6, 11.9, 11.8, 11.9;
  // 2 rows of 2 groups, 8192 -> 1024 18.9, 11.6, 11.6, 11.6; 14336 -> 4096 29.9, 23.3, 23.0, 25.2; 4096 -> 8192 13.8, 13.7, 16.3, 16.3; 4 of 64 groups,
  // 7168 -> 2048 17.2, 15.4, 17.1, 17.0.  With two steps to a wave: 8 rows of 8 groups, 2048 -> 512 9.1 in place of 7.9, 2 of 8, 4096 -> 1024 9.7 in
  // place of 10.9; with eight 1, 14336 -> 512 15.8.
  const int64_t steps = (hidden_in + kStep - 1) / kStep, fit = kInt8Units / (f.windows * f.strips), deep = steps / (4 * kFewWaves);
  f.pieces = std::max<int64_t>(1, std::min({fit, deep, int64_t(16)}));
  const uint64_t need = kWsCounterBytes + (uint64_t)f.windows * f.strips * f.pieces * window * kStrip * 4;
  if (f.pieces > 1 && (need > workspace_bytes || f.windows * f.strips > kWsCounterBytes / 4)) f.pieces = 1;
  return f;
}

template <int MT>
void launch_rows(const Int8Params& p, const HostSizes& hs, uint32_t grid, bool odd, hipStream_t stream) {
  if (odd) {
    hipLaunchKernelGGL((int8_rows_kernel<MT, true>), dim3(grid), dim3(kFewThreads), 0, stream, p, hs);
  } else {
    hipLaunchKernelGGL((int8_rows_kernel<MT, false>), dim3(grid), dim3(kFewThreads), 0, stream, p, hs);
  }
}

}  // namespace

bool int8_rows_fit(int64_t tokens, int64_t num_groups, int64_t hidden_in, int64_t hidden_out) {
  const Int8Plan f = int8_plan(tokens, num_groups, hidden_in, hidden_out, ~uint64_t(0));
  return f.windows * f.strips * f.pieces < (int64_t(1) << 32) / kFewThreads;   // (threads of a launch are counted in 32 bits)
}

bool int8_rows_in_pieces(int64_t tokens, int64_t num_groups, int64_t hidden_in, int64_t hidden_out) {
  return int8_plan(tokens, num_groups, hidden_in, hidden_out, ~uint64_t(0)).pieces > 1;
}

hipError_t int8_rows(Int8Args a, const HostSizes& hs, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  const Int8Plan f = int8_plan(a.tokens, a.num_groups, a.hidden_in, a.hidden_out, workspace != nullptr ? workspace_bytes : 0);
  a.arrivals = static_cast<int32_t*>(workspace);
  a.parts = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + kWsCounterBytes);
  const Int8Params p = {a, (int32_t)f.strips, (int32_t)f.pieces};
  const uint32_t grid = (uint32_t)(f.windows * f.strips * f.pieces);
  const bool odd = (((reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b)) & 3) | (a.hidden_in & 3)) != 0;
  switch (f.rows_of_window) {
    case 1: launch_rows<1>(p, hs, grid, odd, stream); break;
    case 2: launch_rows<2>(p, hs, grid, odd, stream); break;
    default: launch_rows<4>(p, hs, grid, odd, stream); break;
  }
  return hipGetLastError();
}

}  // namespace gg
