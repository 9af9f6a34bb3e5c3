// Rows as 8-bit integers with a scale each, for products in them:
//
//   most = max |x| of the row;  scale = most / 127;  q = the integer nearest to 127 x / most, ties to even.
//
// x is a row as it is, or (with a row index) one that the index names, or silu(gate) * up of a row gate | up, computed in
// fp32 and not rounded in between.  q is what exact arithmetic gives: 127 x / most is computed in fp32, off by less than
// 2^-15 at its largest, and where that leaves open which integer is the nearest, 127 x - q most is looked at in 64
// bits, which hold it exactly.  scale is the fp32 quotient.  A row of zeros has a scale of 0.  An infinity in a row makes its scale
// infinite (infinities are +-127, all else 0), a NaN makes it NaN: products of such rows are not finite.
#include "operators.hpp"

#include <math.h>

#include <algorithm>

#include "few_rows.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

struct QuantizeParams {
  QuantizeArgs a;
  int32_t chunks;   // of 8 elements, of a row
};

struct Eight {
  float v[8];
};

// 8 elements from p on, in fp32.
template <int DT>
__device__ __forceinline__ Eight widen8(const void* row, int64_t at) {
  Eight e;
  if constexpr (DT == kF32) {
    struct __attribute__((packed, aligned(4))) Floats {
      float v[8];
    };
    const Floats f = *reinterpret_cast<const Floats*>(static_cast<const float*>(row) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = f.v[i];
  } else {
    const u32x4 raw = load8(static_cast<const uint16_t*>(row) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = widen_bits<DT>((uint16_t)(raw[i / 2] >> (16 * (i % 2))));
  }
  return e;
}
template <int DT>
__device__ __forceinline__ float widen1(const void* row, int64_t at) {
  if constexpr (DT == kF32) return static_cast<const float*>(row)[at];
  else return widen_bits<DT>(static_cast<const uint16_t*>(row)[at]);
}
// Chunk c of a row of `cols`: zeros past its end.
template <int DT>
__device__ __forceinline__ Eight chunk_of(const void* row, int c, int cols) {
  if (c * 8 + 8 <= cols) return widen8<DT>(row, c * 8);
  Eight e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = c * 8 + i < cols ? widen1<DT>(row, c * 8 + i) : 0.0f;
  return e;
}

template <int DT, bool GATED>
__device__ __forceinline__ Eight values_of(const void* row, int c, int cols) {
  Eight x = chunk_of<DT>(row, c, cols);
  if constexpr (GATED) {
    constexpr int BYTES = DT == kF32 ? 4 : 2;
    const Eight up = chunk_of<DT>(static_cast<const char*>(row) + (int64_t)cols * BYTES, c, cols);
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = x.v[i] / (1.0f + expf(-x.v[i])) * up.v[i];
  }
  return x;
}

// The bits of |x| are ordered as the numbers are, NaN above all.
__device__ __forceinline__ uint32_t size_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t most_of(const Eight& x, uint32_t most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t s = size_bits(x.v[i]);
    most = s > most ? s : most;
  }
  return most;
}

struct RowScale {
  float most, unit, inverse;   // unit: a power of two that x and most are multiplied with, so that 127 / most is a float
  bool finite;
};
__device__ __forceinline__ RowScale row_scale(uint32_t most_bits) {
  RowScale s;
  s.most = __builtin_bit_cast(float, most_bits);
  s.finite = most_bits < 0x7f800000u;
  s.unit = s.most < 0x1p-64f ? 0x1p64f : 1.0f;
  s.inverse = s.most > 0.0f ? 127.0f / (s.most * s.unit) : 0.0f;
  return s;
}

// Eight integers, a byte each.
__device__ __forceinline__ u32x2 round8(const Eight& x, const RowScale& s) {
  constexpr float MAGIC = 0x1.8p23f;   // beside it a float has no places behind the point, and its lowest byte is the integer's
  constexpr float OPEN = 0.5f - 0x1p-15f;
  uint32_t bits[8];
  if (!s.finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bits[i] = size_bits(x.v[i]) == 0x7f800000u ? (x.v[i] > 0.0f ? 127u : 129u) : 0u;
  } else {
    float furthest = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = x.v[i] * s.unit * s.inverse, m = t + MAGIC;
      bits[i] = __builtin_bit_cast(uint32_t, m);
      furthest = fmaxf(furthest, fabsf(t - (m - MAGIC)));
    }
    if (furthest > OPEN) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int q = (int)(bits[i] << 24) >> 24;
        const double rest = fma(-(double)q, (double)s.most, 127.0 * (double)x.v[i]), half = 0.5 * (double)s.most;
        const int odd = q & 1;
        if (rest > half || (rest == half && odd)) bits[i] = (uint32_t)(q + 1);
        if (rest < -half || (rest == -half && odd)) bits[i] = (uint32_t)(q - 1);
      }
    }
  }
  u32x2 packed;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t low = __builtin_amdgcn_perm(bits[4 * h + 1], bits[4 * h], 0x0c0c0400u);
    const uint32_t high = __builtin_amdgcn_perm(bits[4 * h + 3], bits[4 * h + 2], 0x04000c0cu);
    packed[h] = low | high;
  }
  return packed;
}

__device__ __forceinline__ void store_chunk(int8_t* row, int c, int cols, u32x2 v) {
  struct __attribute__((packed, aligned(1))) Bytes8 {
    u32x2 v;
  };
  if (c * 8 + 8 <= cols) {
    reinterpret_cast<Bytes8*>(row + c * 8)->v = v;
  } else {
    for (int i = 0; c * 8 + i < cols; ++i) row[c * 8 + i] = (int8_t)(v[i / 4] >> (8 * (i % 4)));
  }
}

// THREADS threads to a row, which hold HELD chunks of it each between the two passes; rows with more are read twice.
template <int DT, bool GATED, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void quantize_kernel(QuantizeParams p) {
  constexpr int BLOCK = THREADS < 256 ? 256 : THREADS, ROWS = BLOCK / THREADS, WAVES = THREADS / 64;
  constexpr int BYTES = DT == kF32 ? 4 : 2;
  __shared__ uint32_t of_wave[WAVES];
  const QuantizeArgs& a = p.a;
  const int t = threadIdx.x % THREADS;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    int64_t source = row;
    if (a.row_index != nullptr) source = a.row_index[row];
    const bool there = (uint64_t)source < (uint64_t)a.x_rows;
    const void* x = static_cast<const char*>(a.x) + (there ? source : 0) * a.x_stride * BYTES;
    const int cols = (int)a.cols, chunks = there ? p.chunks : 0;
    Eight held[HELD];
    uint32_t most = 0;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int c = t + h * THREADS;
      if (c < chunks) {
        held[h] = values_of<DT, GATED>(x, c, cols);
        most = most_of(held[h], most);
      }
    }
    for (int c = t + HELD * THREADS; c < chunks; c += THREADS) most = most_of(values_of<DT, GATED>(x, c, cols), most);
    most = group_max<64>(most);
    if constexpr (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) of_wave[t / 64] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) most = of_wave[w] > most ? of_wave[w] : most;
      __syncthreads();   // (read before the next row's are written)
    }
    const RowScale s = row_scale(most);
    int8_t* q = a.q + row * a.cols;
    if (t == 0) a.scales[row] = s.most / 127.0f;
    if (!there) {
      for (int c = t; c < p.chunks; c += THREADS) store_chunk(q, c, cols, u32x2{0u, 0u});
      continue;
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int c = t + h * THREADS;
      if (c < chunks) store_chunk(q, c, cols, round8(held[h], s));
    }
    for (int c = t + HELD * THREADS; c < chunks; c += THREADS) store_chunk(q, c, cols, round8(values_of<DT, GATED>(x, c, cols), s));
  }
}

template <int DT, bool GATED, int THREADS, int HELD>
hipError_t launch_rows(const QuantizeParams& p, hipStream_t stream) {
  constexpr int BLOCK = THREADS < 256 ? 256 : THREADS, ROWS = BLOCK / THREADS;
  const int64_t blocks = std::min<int64_t>((p.a.rows + ROWS - 1) / ROWS, 1 << 16);
  hipLaunchKernelGGL((quantize_kernel<DT, GATED, THREADS, HELD>), dim3((uint32_t)blocks), dim3(BLOCK), 0, stream, p);
  return hipGetLastError();
}

template <int DT, bool GATED>
hipError_t launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  QuantizeParams p;
  p.a = a;
  p.chunks = (int32_t)((a.cols + 7) / 8);
  if (p.chunks <= 64) return launch_rows<DT, GATED, 64, 1>(p, stream);
  if (p.chunks <= 128) return launch_rows<DT, GATED, 64, 2>(p, stream);
  if (p.chunks <= 256) return launch_rows<DT, GATED, 64, 4>(p, stream);
  if (p.chunks <= 512) return launch_rows<DT, GATED, 256, 2>(p, stream);
  if (p.chunks <= 1024) return launch_rows<DT, GATED, 256, 4>(p, stream);
  return launch_rows<DT, GATED, 256, 8>(p, stream);
}

}  // namespace

hipError_t quantize(const QuantizeArgs& a, hipStream_t stream) {
#define GG_LAUNCH(DT) (a.gated ? launch_quantize<DT, true>(a, stream) : launch_quantize<DT, false>(a, stream))
  if (a.dt == kF32) return GG_LAUNCH(kF32);
  return a.dt == kBF16 ? GG_LAUNCH(kBF16) : GG_LAUNCH(kF16);
#undef GG_LAUNCH
}

}  // namespace gg
