// Low-rank adapters of many requests beside a shared projection: with l the adapter of row t,
//
//   v[t] = a_l x[t]   (a_l: rank x hidden_in)        out[t] = base[t] + scale_l * b_l v[t]   (b_l: hidden_out x rank)
//
// Bound by base and out for many rows, by the adapters' weights for rows of many adapters, and by the launches for one.
// Rows are taken in windows of 64 in their own order, and the rows of a window that share an adapter together: the
// rows of a prompt are neighbours, and the rows of a decode step are one window, so nothing has to be sorted.  A wave knows
// its window's rows from one load and a ballot for each adapter.
//
// v is kept in fp32, summed over pieces of the depth by its readers, and split there into two numbers of the
// element type (high, and what its rounding left), each multiplied by b_l: nothing of v is lost that the result could show.
#include "operators.hpp"

#include <math.h>

#include "few_rows.hpp"
#include "gmm_kernel.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kWindow = 64;

struct AdapterParams {
  AdapterArgs a;
  float* v;          // [pieces][rows][v_pitch]
  int32_t v_pitch;
  int32_t pieces;    // of the depth hidden_in
  int32_t splits;    // workgroups that share a window's adapters
  int32_t strips;    // of hidden_out
};

// The window's adapters one by one, in the order of their first rows: the rows of each as a mask of lanes.
struct Window {
  int32_t adapter;    // of this lane's row, -1 without one
  uint64_t left;      // rows not yet taken
  uint64_t none;      // rows without an adapter
  int32_t rows;

  __device__ __forceinline__ Window(const AdapterArgs& a, int64_t first) {
    const int lane = threadIdx.x & 63;
    rows = (int)(a.rows - first < kWindow ? a.rows - first : kWindow);
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
  // Lane i gets the number of the i-th row of `mine` in the window (lanes past the last: any).
  static __device__ __forceinline__ int list(uint64_t mine) {
    const int lane = threadIdx.x & 63, count = __popcll(mine);
    const int before = __popcll(mine & ((uint64_t(1) << lane) - 1));
    const bool in = (mine >> lane) & 1;
    // (rows of the mask go to the first lanes, the others behind them: every lane is written once)
    return __builtin_amdgcn_ds_permute(4 * (in ? before : count + lane - before), lane);
  }
};

// v of one piece of the depth.  TILES: of 16 rows of a_l; more than 64 of them are taken 64 at a time.
template <int DT, int TILES, int MT>
__global__ __launch_bounds__(kFewThreads, 2) void adapter_shrink_kernel(AdapterParams p) {
  using S = Stream<DT, true, TILES, MT>;
  __shared__ f32x4 lds[kFewWaves * 256];
  const AdapterArgs& a = p.a;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int64_t window = blockIdx.x / p.splits, first = window * kWindow;
  const int split = (int)(blockIdx.x - window * p.splits), piece = blockIdx.y;
  const int steps = (a.hidden_in + S::DEPTH - 1) / S::DEPTH;
  const int begin = (int)((int64_t)steps * piece / p.pieces), end = (int)((int64_t)steps * (piece + 1) / p.pieces);
  float* v = p.v + (uint64_t)piece * a.rows * p.v_pitch;
  Window w(a, first);
  S s;
  s.depth = a.hidden_in;
  s.width = 8;
  s.x = static_cast<const uint16_t*>(a.x) + (uint64_t)first * a.hidden_in;
  const Exchange<true> exchange{lds};
  for (int turn = 0; w.left != 0; turn = turn + 1 == p.splits ? 0 : turn + 1) {
    int which;
    const uint64_t mine = w.next(which);
    if (turn != split) continue;
    const int list = Window::list(mine), rows = __popcll(mine);
    const uint16_t* weights = static_cast<const uint16_t*>(a.a) + (uint64_t)which * a.rank * a.hidden_in;
    for (int r0 = 0; r0 < a.rank; r0 += 16 * TILES) {
      s.first = s.second = weights + (uint64_t)r0 * a.hidden_in;
#pragma unroll
      for (int i = 0; i < TILES; ++i)   // (rows past the last: the last one's, not stored)
        s.at[i] = (uint32_t)(min(16 * i + c, a.rank - 1 - r0)) * (uint32_t)a.hidden_in * 2 + q * 32;
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

// out for a strip of columns: each wave has 64 of them, a lane 16 neighbouring ones of one row of the 16 of a tile.
constexpr int kExpandWaves = 4;
constexpr int kExpandThreads = kExpandWaves * 64;
constexpr int kStrip = kExpandWaves * 64;
constexpr int kRankStep = 64;                  // ranks in LDS at a time
constexpr int kLowPitch = kRankStep + 8;       // (so that the 16 rows of a fragment start in different banks)

template <int DT>
__global__ __launch_bounds__(kExpandThreads, 2) void adapter_expand_kernel(AdapterParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t split_v[2][kWindow][kLowPitch];   // high, low
  __shared__ float unit[kWindow];
  const AdapterArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4, wave = tid >> 6;
  uint32_t block = blockIdx.x;
  const int strip = (int)(block % p.strips);
  block /= p.strips;
  const int split = (int)(block % p.splits);
  const int64_t first = (int64_t)(block / p.splits) * kWindow;
  const int column0 = strip * kStrip + wave * 64;   // of the wave
  const int own = column0 + q * 16;                 // the lane's first column
  const uint16_t* base = static_cast<const uint16_t*>(a.base);
  uint16_t* out = static_cast<uint16_t*>(a.out);
  const int columns = a.hidden_out;
  Window w(a, first);
  if (split == 0 && w.none != 0 && out != base) {   // rows without an adapter
    for (int r = wave; r < w.rows; r += kExpandWaves) {
      if (!((w.none >> r) & 1)) continue;
      const uint64_t at = (uint64_t)(first + r) * columns;
      for (int n = strip * kStrip + lane; n < min(columns, (strip + 1) * kStrip); n += 64) out[at + n] = base != nullptr ? base[at + n] : uint16_t(0);
    }
  }
  for (int turn = 0; w.left != 0; turn = turn + 1 == p.splits ? 0 : turn + 1) {
    int which;
    const uint64_t mine = w.next(which);
    if (turn != split) continue;
    const int list = Window::list(mine), rows = __popcll(mine);
    const uint16_t* weights = static_cast<const uint16_t*>(a.b) + (uint64_t)which * columns * a.rank;
    const float scale = a.scales != nullptr ? a.scales[which] : 1.0f;
    // the row of b_l that is this lane's row of tile i, so that a lane ends up with neighbouring columns
    uint32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = (uint32_t)min(column0 + (c >> 2) * 16 + i * 4 + (c & 3), columns - 1);
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int m = 0; m < 4; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // four threads have a row of v: 4 of every 16 ranks each
    const int row = tid >> 2, part = tid & 3;
    const float* v = p.v + (uint64_t)(first + __shfl(list, row)) * p.v_pitch;
    auto four = [&](int r) {
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
      if (row >= rows) return sum;
      for (int piece = 0; piece < p.pieces; ++piece) {
        const f32x4 one = *reinterpret_cast<const f32x4*>(v + (uint64_t)piece * a.rows * p.v_pitch + r);
        sum += one;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r + e >= a.rank) sum[e] = 0.0f;
      return sum;
    };
    float scaling = 1.0f;
    if constexpr (DT == kF16) {
      // v may be larger than the type holds: its row is scaled to below 1 by a power of two, exactly
      float most = 0.0f;
      for (int r = part * 4; r < a.rank; r += 16) {
        const f32x4 x = four(r);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[e]));
      }
      most = fmaxf(most, __shfl_xor(most, 1));
      most = fmaxf(most, __shfl_xor(most, 2));
      // (rows of zeros, and of infinities, which stay what they are)
      const int up = most > 0.0f && most < INFINITY ? min(max(ilogbf(most) + 1, -100), 120) : 0;
      scaling = ldexpf(1.0f, -up);
      __syncthreads();
      if (part == 0) unit[row] = ldexpf(1.0f, up);
    }
    for (int r0 = 0; r0 < a.rank; r0 += kRankStep) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kRankStep / 16; ++j) {
        const int r = j * 16 + part * 4;
        const f32x4 x = r0 + r < a.rank ? four(r0 + r) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        u32x2 high, low;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t h[2], l[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const float s = x[2 * e + o] * scaling;
            h[o] = round_bits<DT>(s);
            const float rest = s - widen_bits<DT>((uint16_t)h[o]);
            l[o] = fabsf(rest) < INFINITY ? round_bits<DT>(rest) : 0u;
          }
          high[e] = h[0] | h[1] << 16;
          low[e] = l[0] | l[1] << 16;
        }
        *reinterpret_cast<u32x2*>(&split_v[0][row][r]) = high;
        *reinterpret_cast<u32x2*>(&split_v[1][row][r]) = low;
      }
      __syncthreads();
      const int depth = min(kRankStep, a.rank - r0);
      for (int k = 0; k < depth; k += 32) {
        u32x4 b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = load8_within(weights + (uint64_t)at[i] * a.rank, r0 + k + q * 8, a.rank);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (16 * m >= rows) break;
#pragma unroll
          for (int part_of = 0; part_of < 2; ++part_of) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(&split_v[part_of][16 * m + c][k + q * 8]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[i][m] = mfma_16x16x32<DT>(__builtin_bit_cast(bf16x8, b[i]), __builtin_bit_cast(bf16x8, x), acc[i][m]);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (16 * m >= rows) break;
      const int of = 16 * m + c, from = __shfl(list, of);
      if (of >= rows || own >= columns) continue;
      const float s = DT == kF16 ? scale * unit[of] : scale;
      const uint64_t to = (uint64_t)(first + from) * columns + own;
      float y[16];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * i + e] = s * acc[i][m][e];
      if (own + 16 <= columns) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 have = {0u, 0u, 0u, 0u};
          if (base != nullptr) have = load8(base + to + 8 * h);
          u32x4 bits;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float lo = widen_bits<DT>((uint16_t)have[e]) + y[8 * h + 2 * e];
            const float hi = widen_bits<DT>((uint16_t)(have[e] >> 16)) + y[8 * h + 2 * e + 1];
            bits[e] = round_bits<DT>(lo) | (uint32_t)round_bits<DT>(hi) << 16;
          }
          store8(out + to + 8 * h, bits);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (own + e < columns) out[to + e] = round_bits<DT>((base != nullptr ? widen_bits<DT>(base[to + e]) : 0.0f) + y[e]);
      }
    }
  }
}

struct AdapterPlan {
  int64_t windows, v_pitch, pieces, shrink_splits, strips, expand_splits;
};

// Workgroups that keep the device busy.
constexpr int64_t kBusy = 1024;

AdapterPlan adapter_plan(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  AdapterPlan f;
  const int64_t most = num < kWindow ? (num < rows ? num : rows) : (rows < kWindow ? rows : kWindow);   // adapters of a window
  auto between = [](int64_t v, int64_t hi) { return v > hi ? (hi < 1 ? 1 : hi) : (v < 1 ? 1 : v); };
  f.windows = (rows + kWindow - 1) / kWindow;
  f.v_pitch = (rank + 3) / 4 * 4;
  f.shrink_splits = between(kBusy / f.windows, most);
  // the depth in pieces of at least one step of every wave
  f.pieces = between(between(hidden_in / (64 * kFewWaves), 8), kBusy / (f.windows * f.shrink_splits) < 1 ? 1 : kBusy / (f.windows * f.shrink_splits));
  f.strips = (hidden_out + kStrip - 1) / kStrip;
  f.expand_splits = between(kBusy / (f.windows * f.strips), most);
  return f;
}

template <int DT, int TILES>
void launch_shrink(const AdapterParams& p, const AdapterPlan& f, hipStream_t stream) {
  const dim3 grid((uint32_t)(f.windows * f.shrink_splits), (uint32_t)f.pieces);
  if (p.a.rows <= kWindow) {
    hipLaunchKernelGGL((adapter_shrink_kernel<DT, TILES, 1>), grid, dim3(kFewThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL((adapter_shrink_kernel<DT, TILES, 4>), grid, dim3(kFewThreads), 0, stream, p);
  }
}

template <int DT>
hipError_t launch_adapters(const AdapterArgs& a, hipStream_t stream) {
  const AdapterPlan f = adapter_plan(a.rows, a.num, a.rank, a.hidden_in, a.hidden_out);
  AdapterParams p;
  p.a = a;
  p.v = static_cast<float*>(a.scratch);
  p.v_pitch = (int32_t)f.v_pitch;
  p.pieces = (int32_t)f.pieces;
  p.strips = (int32_t)f.strips;
  p.splits = (int32_t)f.shrink_splits;
  if (a.rank <= 16) {
    launch_shrink<DT, 1>(p, f, stream);
  } else if (a.rank <= 32) {
    launch_shrink<DT, 2>(p, f, stream);
  } else {
    launch_shrink<DT, 4>(p, f, stream);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  p.splits = (int32_t)f.expand_splits;
  hipLaunchKernelGGL((adapter_expand_kernel<DT>), dim3((uint32_t)(f.windows * f.expand_splits * f.strips)), dim3(kExpandThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

bool adapters_fit(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  const AdapterPlan f = adapter_plan(rows, num, rank, hidden_in, hidden_out);
  const int64_t threads = int64_t(1) << 32;   // of a launch, which are counted in 32 bits
  return f.windows * f.shrink_splits * kFewThreads < threads && f.windows * f.expand_splits * f.strips * kExpandThreads < threads;
}

uint64_t adapters_scratch_bytes(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  const AdapterPlan f = adapter_plan(rows, num, rank, hidden_in, hidden_out);
  return (uint64_t)(f.pieces * rows * f.v_pitch) * sizeof(float);
}

hipError_t adapters(const AdapterArgs& a, hipStream_t stream) {
  return a.dt == kBF16 ? launch_adapters<kBF16>(a, stream) : launch_adapters<kF16>(a, stream);
}

}  // namespace gg
