// Rows as 8-bit integers with a scale each, for products in them:
//
//   most = max |x| of the row;  scale = most / 127;  q = the integer nearest to 127 x / most, ties to even.
//
// x is a row as it is, or (with a row index) one that the index names, or silu(gate) * up of a row gate | up, computed in
// fp32 and not rounded in between.  scale is the fp32 quotient.  A row of zeros has a scale of 0.  An infinity in a row makes its scale infinite
// (infinities are +-127, all else 0), a NaN makes it NaN: products of such rows are not finite.
//
// q is what exact arithmetic gives, at one fused multiply-add for most elements (bound by reading and writing, the kernel has few instructions
// for each):
//   Two-byte x.  A tie is 254 x = (2 r + 1) most in whole numbers, so 127 divides most's significand, or it divides 2 r + 1 < 254, and then r is 63
//   and the tie goes to 64, away from zero.  Where 127 does not divide the significand, x times a number just above 127 / most, off by at
//   most 1.5 * 2^-23 of itself, rounds as it should: a value that is no tie is no nearer to one than 2^-20 of itself (x is a multiple of 2^-11 of its power
//   of two, most of its own, and |x| <= most), and the ties at 63.5 are pushed away from zero.
//   Otherwise 127 x / most comes out off by less than 2^-15, and where that leaves open which integer is the nearest, the sign of 127 x - (q +- 1/2) most
//   decides, which sums of floats whose errors are kept have exactly.
//   silu(gate) * up is off by more than any of that, and is rounded as it comes.
//
// Read once, written once: 16384 rows of 4096 bf16 in 30 us, 6.7 TB/s (where x is in the last level of cache in part; a copy from and to
// memory reaches 5.2), 8192 x 4096 in fp32 in 26 us, 6.5 TB/s; 24576 rows of 2048 that an index takes from 4096 in 23 us; silu(gate) * up, 8192 rows of
// 4096, in 29 us, 5.8 TB/s, by its arithmetic as much as by memory; one token in 2.8 us, next to an empty launch.
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
struct __attribute__((packed, aligned(4))) Floats8 {
  float v[8];
};

// What a thread holds of a row between the two passes: 8 elements, as they are or (gated) as they came out.
template <int DT, bool GATED>
struct Held {
  static constexpr bool FLOATS = DT == kF32 || GATED;
  std::conditional_t<FLOATS, Eight, u32x4> raw;
  __device__ __forceinline__ float value(int i) const {
    if constexpr (FLOATS) {
      return raw.v[i];
    } else if constexpr (DT == kBF16) {
      return __builtin_bit_cast(float, i % 2 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
    } else {
      return widen_bits<DT>((uint16_t)(raw[i / 2] >> (16 * (i % 2))));
    }
  }
};

// `count` elements of a row from `at` on, and zeros.
template <int DT>
__device__ __forceinline__ Held<DT, false> load_chunk(const void* row, int64_t at, int count = 8) {
  Held<DT, false> h;
  if constexpr (DT == kF32) {
    const float* from = static_cast<const float*>(row) + at;
    const Floats8 f = count == 8 ? *reinterpret_cast<const Floats8*>(from) : Floats8{};
#pragma unroll
    for (int i = 0; i < 8; ++i) h.raw.v[i] = count == 8 ? f.v[i] : (i < count ? from[i] : 0.0f);
  } else {
    const uint16_t* from = static_cast<const uint16_t*>(row) + at;
    if (count == 8) {
      h.raw = load8(from);
    } else {
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i < count ? from[i] : uint16_t(0);
      h.raw = __builtin_bit_cast(u32x4, e);
    }
  }
  return h;
}

// gate / (1 + exp(-gate)) * up.  The exponential by the hardware's power of two, with what rounding its argument lost put back: within two units in the
// last place.  The quotient as in the streaming kernel's epilogue: the hardware's reciprocal (of a quarter of the divisor, whose reciprocal is
// normal) and one correction by the remainder.
__device__ __forceinline__ float gated(float gate, float up) {
  constexpr float LOG2E = 0x1.715476p+0f, LOG2E_REST = 0x1.4ae0bep-26f, LN2 = 0x1.62e430p-1f;
  const float t = -gate * LOG2E, rest = __builtin_fmaf(-gate, LOG2E_REST, __builtin_fmaf(-gate, LOG2E, -t));
  const float power = __builtin_amdgcn_exp2f(t);
  const float e = fabsf(t) < 128.0f ? __builtin_fmaf(power, rest * LN2, power) : power;   // (past a float's range: 0 or infinity)
  const float d = 1.0f + e, inverse = 0.25f * __builtin_amdgcn_rcpf(0.25f * d);
  const float quotient = gate * inverse, remainder = __builtin_fmaf(-d, quotient, gate);
  return __builtin_fmaf(__builtin_fmaxf(remainder, -__FLT_MAX__), inverse, quotient) * up;
}

// What is loaded of a chunk, and what it is made into.
template <int DT, bool GATED>
struct Loaded {
  Held<DT, false> x, up;
  __device__ __forceinline__ void load(const void* row, int at, int cols, int count = 8) {
    x = load_chunk<DT>(row, at, count);
    if constexpr (GATED) up = load_chunk<DT>(row, (int64_t)cols + at, count);
  }
  __device__ __forceinline__ Held<DT, GATED> value() const {
    if constexpr (!GATED) {
      return x;
    } else {
      Held<DT, GATED> h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h.raw.v[i] = gated(x.value(i), up.value(i));
      return h;
    }
  }
};

// The bits of |x| are ordered as the numbers are, NaN above all.
__device__ __forceinline__ uint32_t size_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The largest of the elements' bits without their signs so far: two halves of two-byte types, one word of fp32.
template <int DT, bool GATED>
__device__ __forceinline__ uint32_t most_of(const Held<DT, GATED>& h, uint32_t most) {
  if constexpr (Held<DT, GATED>::FLOATS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, size_bits(h.raw.v[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most), __builtin_bit_cast(u16x2, h.raw[i] & 0x7fff7fffu)));
  }
  return most;
}

enum : int { kQuick, kExact, kOdd };   // one multiply-add; ties are looked at; an infinity or a NaN
struct RowScale {
  float most, inverse;
  float unit;   // kExact: a power of two that x and most are multiplied with, so that neither 127 / most nor 127 x leaves a float's range
  int way;      // the same in all threads of a row
};

// most_bits: as most_of gives them
template <int DT, bool GATED>
__device__ __forceinline__ RowScale row_scale(uint32_t most_bits) {
  RowScale s;
  bool divides = !GATED;   // 127 may divide the significand
  if constexpr (Held<DT, GATED>::FLOATS) {
    s.most = __builtin_bit_cast(float, most_bits);
  } else {
    s.most = widen_bits<DT>((uint16_t)most_bits);
    constexpr uint32_t IMPLICIT = DT == kBF16 ? 0x80u : 0x400u;
    divides = ((most_bits & (IMPLICIT - 1)) | (most_bits >= IMPLICIT ? IMPLICIT : 0u)) % 127u == 0;
  }
  const bool small = s.most < 0x1p-64f;
  s.way = !(s.most < INFINITY) ? kOdd : (divides || small ? kExact : kQuick);
  s.unit = s.way != kExact ? 1.0f : (small ? 0x1p64f : (s.most > 0x1p64f ? 0x1p-64f : 1.0f));
  s.inverse = s.most > 0.0f ? 127.0f / (s.most * s.unit) : 0.0f;
  if (s.way == kQuick && !GATED) s.inverse = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, s.inverse) + 1);
  return s;
}

constexpr float kMagic = 0x1.8p23f;   // beside it a float has no places behind the point, and its lowest byte is the integer's

__device__ __forceinline__ u32x2 pack8(const uint32_t (&bits)[8]) {
  u32x2 packed;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const uint32_t low = __builtin_amdgcn_perm(bits[4 * p + 1], bits[4 * p], 0x0c0c0400u);
    const uint32_t high = __builtin_amdgcn_perm(bits[4 * p + 3], bits[4 * p + 2], 0x04000c0cu);
    packed[p] = low | high;
  }
  return packed;
}
// Eight integers, a byte each.
template <int DT, bool GATED>
__device__ __forceinline__ u32x2 round_quick(const Held<DT, GATED>& h, const RowScale& s) {
  uint32_t bits[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bits[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(h.value(i), s.inverse, kMagic));
  return pack8(bits);
}
template <int DT, bool GATED>
__device__ __forceinline__ u32x2 round_exact(const Held<DT, GATED>& h, const RowScale& s) {
  uint32_t bits[8];
  float furthest = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = h.value(i) * s.unit, m = __builtin_fmaf(x, s.inverse, kMagic);
    bits[i] = __builtin_bit_cast(uint32_t, m);
    furthest = fmaxf(furthest, fabsf(__builtin_fmaf(x, s.inverse, kMagic - m)));
  }
  if (furthest > 0.5f - 0x1p-15f) {
    const float most = s.most * s.unit, half = 0.5f * most;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // 127 x = times + lost; times - q most is within half and 2^-15 of most, and a float; so is its difference from half
      const float x = h.value(i) * s.unit, q = __builtin_bit_cast(float, bits[i]) - kMagic;
      const float times = 127.0f * x, lost = __builtin_fmaf(127.0f, x, -times), rest = __builtin_fmaf(-q, most, times);
      const float above = (rest - half) + lost, below = (rest + half) + lost;
      const bool odd = (bits[i] & 1) != 0;
      if (above > 0.0f || (above == 0.0f && odd)) bits[i] += 1;
      if (below < 0.0f || (below == 0.0f && odd)) bits[i] -= 1;
    }
  }
  return pack8(bits);
}
template <int DT, bool GATED>
__device__ __forceinline__ u32x2 round_odd(const Held<DT, GATED>& h) {
  uint32_t bits[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bits[i] = size_bits(h.value(i)) == 0x7f800000u ? (h.value(i) > 0.0f ? 127u : 129u) : 0u;
  return pack8(bits);
}

template <int DT, bool GATED>
__device__ __forceinline__ u32x2 round_any(const Held<DT, GATED>& h, const RowScale& s) {
  return s.way == kOdd ? round_odd(h) : (s.way == kExact ? round_exact(h, s) : round_quick(h, s));
}

__device__ __forceinline__ void store8(int8_t* to, u32x2 v) {
  struct __attribute__((packed, aligned(1))) Bytes8 {
    u32x2 v;
  };
  reinterpret_cast<Bytes8*>(to)->v = v;
}

struct SourceRow {
  const void* x;
  bool there;   // the index names a row
};
template <int DT>
__device__ __forceinline__ SourceRow source_row(const QuantizeArgs& a, int64_t row) {
  int64_t source = row;
  if (a.row_index != nullptr) source = a.row_index[row];
  const bool there = (uint64_t)source < (uint64_t)a.x_rows;
  return {static_cast<const char*>(a.x) + (there ? source : 0) * a.x_stride * (DT == kF32 ? 4 : 2), there};
}

// THREADS threads to a row of at least 8, which hold HELD chunks of it each between the two passes; rows with more are read twice, and so are
// those that are not rounded in the way that most of their type are.  A row's last chunk is its last 8 elements: where it overlaps the one
// before, both write the same.  Threads without a chunk take the last one, and store nothing; waves without one leave out silu(gate) * up, which
// costs as much as its traffic (8192 rows of 5632, fp16: 41 us in place of 49.5; rows as they are lose 1 to 3 % by the branch, and go without).
template <int DT, bool GATED, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void quantize_kernel(QuantizeParams p) {
  constexpr int BLOCK = THREADS == 64 ? 256 : THREADS, ROWS = BLOCK / THREADS, WAVES = THREADS / 64;
  static_assert(ROWS == 1 || WAVES == 1, "rows of one workgroup meet at no barrier");
  __shared__ uint32_t of_wave[WAVES];
  const QuantizeArgs& a = p.a;
  const int t = threadIdx.x % THREADS, first = uniform(t / 64 * 64), cols = (int)a.cols;   // `first` of the wave
  for (int64_t row = (int64_t)blockIdx.x * ROWS + uniform((int)(threadIdx.x / THREADS)); row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    const SourceRow source = source_row<DT>(a, row);
    int8_t* q = a.q + row * a.cols;
    if (!source.there) {
      if (t == 0) a.scales[row] = 0.0f;
      for (int c = t; c < p.chunks; c += THREADS) store8(q + min(c * 8, cols - 8), u32x2{0u, 0u});
      continue;
    }
    Held<DT, GATED> held[HELD];
    uint32_t most = 0;
    {
      Loaded<DT, GATED> loaded[HELD];
#pragma unroll
      for (int h = 0; h < HELD; ++h) loaded[h].load(source.x, min((t + h * THREADS) * 8, cols - 8), cols);
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        if (GATED && first + h * THREADS >= p.chunks) break;
        held[h] = loaded[h].value();
        most = most_of(held[h], most);
      }
    }
    for (int c = t + HELD * THREADS; c < p.chunks; c += THREADS) {
      Loaded<DT, GATED> more;
      more.load(source.x, min(c * 8, cols - 8), cols);
      most = most_of(more.value(), most);
    }
    if constexpr (!Held<DT, GATED>::FLOATS) most = max(most & 0xffffu, most >> 16);
    most = group_max<64>(most);
    if constexpr (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) of_wave[t / 64] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) most = max(most, of_wave[w]);
      __syncthreads();   // (read before the next row's are written)
    }
    const RowScale s = row_scale<DT, GATED>((uint32_t)uniform((int)most));
    if (t == 0) a.scales[row] = s.most / 127.0f;
    constexpr int WAY = DT == kF32 && !GATED ? kExact : kQuick;
    if (s.way == WAY) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        if (GATED && first + h * THREADS >= p.chunks) break;
        const int c = t + h * THREADS;
        const u32x2 v = WAY == kExact ? round_exact(held[h], s) : round_quick(held[h], s);
        if (c < p.chunks) store8(q + min(c * 8, cols - 8), v);
      }
    }
#pragma unroll 1
    for (int c = t + (s.way == WAY ? HELD * THREADS : 0); c < p.chunks; c += THREADS) {
      Loaded<DT, GATED> more;
      more.load(source.x, min(c * 8, cols - 8), cols);
      store8(q + min(c * 8, cols - 8), round_any(more.value(), s));
    }
  }
}

// Rows of fewer than 8, a thread to each.
template <int DT, bool GATED>
__global__ __launch_bounds__(256) void quantize_short_kernel(QuantizeParams p) {
  const QuantizeArgs& a = p.a;
  const int cols = (int)a.cols;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (int64_t)gridDim.x * 256) {
    const SourceRow source = source_row<DT>(a, row);
    u32x2 v = {0u, 0u};
    float scale = 0.0f;
    if (source.there) {
      Loaded<DT, GATED> loaded;
      loaded.load(source.x, 0, cols, cols);
      const Held<DT, GATED> h = loaded.value();
      uint32_t most = most_of(h, 0u);
      if constexpr (!Held<DT, GATED>::FLOATS) most = max(most & 0xffffu, most >> 16);
      const RowScale s = row_scale<DT, GATED>(most);
      v = round_any(h, s);
      scale = s.most / 127.0f;
    }
    a.scales[row] = scale;
    for (int i = 0; i < cols; ++i) a.q[row * cols + i] = (int8_t)(v[i / 4] >> (8 * (i % 4)));
  }
}

template <int DT, bool GATED, int THREADS, int HELD>
hipError_t launch_rows(const QuantizeParams& p, hipStream_t stream) {
  constexpr int BLOCK = THREADS == 64 ? 256 : THREADS, ROWS = BLOCK / THREADS;
  const int64_t blocks = std::min<int64_t>((p.a.rows + ROWS - 1) / ROWS, 1 << 16);
  hipLaunchKernelGGL((quantize_kernel<DT, GATED, THREADS, HELD>), dim3((uint32_t)blocks), dim3(BLOCK), 0, stream, p);
  return hipGetLastError();
}

template <int DT, bool GATED>
hipError_t launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  QuantizeParams p;
  p.a = a;
  p.chunks = (int32_t)((a.cols + 7) / 8);
  if (a.cols < 8) {
    hipLaunchKernelGGL((quantize_short_kernel<DT, GATED>), dim3((uint32_t)std::min<int64_t>((a.rows + 255) / 256, 1 << 16)), dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  // Threads to a row and chunks to a thread: more threads where there are few rows to fill the device with or a row is long, fewer, which meet at no
  // barrier or a small one, elsewhere.  In us, one call after the other, x partly in the last level of cache:
  //   up to 256 chunks, 256 x 1 / the lines below: 512 x 2048 bf16 2.9 / 3.8, 2048 x 2048 4.1 / 4.3, 8192 x 2048 11.0 / 10.5, 8192 x 1024 8.1 / 5.6;
  //   128 x 2 / 64 x 4: 4096 x 2048 6.0 / 6.9, 16384 x 2048 17.3 / 18.3; silu(gate) * up 8192 x 2048 17.2 / 15.7, 24576 x 1408 40.5 / 37.6;
  //   up to 512, 512 x 1 / 256 x 2: 512 x 4096 3.2 / 4.0, 1024 x 4096 4.2 / 4.5, 8192 x 4096 18.3 / 16.8;
  //   up to 1024, 512 x 2 / 256 x 4: 8192 x 8192 30.3 / 31.8, 1024 x 8192 5.8 / 6.9; 1024 x 1: 36.3 and 6.9;
  //   more, 1024 x 2 / 512 x 4 / 256 x 8: 8192 x 14336 62.6 / 62.4 / 64.9, in fp32 100 / 107 / 111, 512 x 14336 6.1 / 6.6 / 8.7; silu(gate) * up,
  //   whose waves without a chunk do less, 4096 x 9000 48 / 35.7 / 34.9, 4096 x 14336 56 / 54 / 56, 64 x 14336 5.1 / 5.0 / 5.9.
  if (p.chunks <= 64) return launch_rows<DT, GATED, 64, 1>(p, stream);
  if (p.chunks <= 256 && a.rows <= 2048) return launch_rows<DT, GATED, 256, 1>(p, stream);
  if (p.chunks <= 128) return launch_rows<DT, GATED, 64, 2>(p, stream);
  if (p.chunks <= 256) return launch_rows<DT, GATED, GATED ? 64 : 128, GATED ? 4 : 2>(p, stream);
  if (p.chunks <= 512) return a.rows <= 1024 ? launch_rows<DT, GATED, 512, 1>(p, stream) : launch_rows<DT, GATED, 256, 2>(p, stream);
  if (p.chunks <= 1024) return launch_rows<DT, GATED, 512, 2>(p, stream);
  return launch_rows<DT, GATED, GATED ? 512 : 1024, GATED ? 4 : 2>(p, stream);
}

}  // namespace

hipError_t quantize(const QuantizeArgs& a, hipStream_t stream) {
#define GG_LAUNCH(DT) (a.gated ? launch_quantize<DT, true>(a, stream) : launch_quantize<DT, false>(a, stream))
  if (a.dt == kF32) return GG_LAUNCH(kF32);
  return a.dt == kBF16 ? GG_LAUNCH(kBF16) : GG_LAUNCH(kF16);
#undef GG_LAUNCH
}

}  // namespace gg
