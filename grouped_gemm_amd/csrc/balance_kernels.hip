// The balance loss of a router and its z-loss, over packed sequences, and their gradient.  For sequence s of T_s counted tokens, T in all:
//
//   mass[s, e] = sum over its tokens of p[t, e];  counts[s, e] = its tokens' choices of e
//   balance = sum over s of T_s / T * sum over e of f[s, e] * mass[s, e] / T_s,  f[s, e] = experts * counts[s, e] / (top_k * T_s)
//   z = 1 / T * sum over t of (log of the sum over e of exp(l[t, e]))^2
//
// with p = softmax(l), or sigmoid(l) divided by its sum.  So balance = 1 / T * sum of share * mass, share = f of the two quotients that do
// not depend on the logits, and the gradient of a logit is
//
//   1 / T * (g p (slope) (share - <share, p>) + 2 h lse softmax),   slope = 1, or 1 - sigmoid(l).
//
// Forward: workgroups take neighbouring tokens; for each sequence in them (a "unit") they sum p in registers and choices in LDS, and write
// one row of partial sums.  The second kernel adds up a sequence's units in their order, and its last workgroup the sequences: no
// atomic adds floats, the same bits on every call.  The units of workgroup c and sequence s are number c + s, since the two only grow.
#include "operators.hpp"

#include <math.h>

#include <algorithm>

#include "gmm_kernel.hpp"
#include "logits.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kBalanceThreads = 256;
constexpr int64_t kBalanceBlocks = 1024;
constexpr int kSumColumns = 64;   // of the second kernel's workgroups

struct BalanceParams {
  BalanceArgs a;
  int32_t chunk;     // tokens of a workgroup
  int32_t tiles;     // of kSumColumns experts
  float* mass;       // [units][experts]
  int32_t* counts;   // [units][experts]
  float* z;          // [units]
  int32_t* tokens;   // [units] counted ones
  float* loss;       // [sequences][tiles]
  float* sequence_z;           // [sequences]
  int32_t* sequence_tokens;    // [sequences]
  int32_t* arrived;
};

__device__ __forceinline__ int64_t offset_of(const int32_t* offsets, int64_t tokens, int s) {
  if (offsets == nullptr) return s == 0 ? 0 : tokens;
  const int64_t at = offsets[s];
  return at < 0 ? 0 : (at > tokens ? tokens : at);
}

// The sequence that token t is in, or the last one that begins before it; -1: none.  By all lanes of a wave: 64 offsets at a time.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int sequences, int64_t t) {
  if (offsets == nullptr) return 0;
  const int lane = threadIdx.x & 63;
  int low = 0, n = sequences + 1;   // the first of the offsets not yet known to be at t or before, and how many are open
  while (n > 0) {
    const int step = (n + 63) / 64, at = lane * step;
    const int before = __popcll(__ballot(at < n && offsets[low + at] <= t));
    if (before == 0) break;
    if (step == 1) {
      low += before;
      break;
    }
    const int from = (before - 1) * step + 1;
    n = min(step - 1, n - from);
    low += from;
  }
  return uniform(low) - 1;
}

// A token's exponentials, in the lanes of its group: softmax and the score, as multiples of what is common to all.
template <int DT, int G, int VPL>
struct Scores {
  float x[VPL], softmax[VPL], score[VPL];
  float lse;

  __device__ __forceinline__ void compute(const Row<typename Logit<DT>::T, VPL>& raw, bool sigmoids) {
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      x[v] = Logit<DT>::widen(raw.v[v]);
      top = fmaxf(top, x[v]);
    }
    top = group_reduce<G>(top, [](float p, float q) { return fmaxf(p, q); });
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      softmax[v] = quick_exp(x[v] - base);
      sum += softmax[v];
    }
    sum = group_sum<G>(sum);
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    lse = sum == 0.0f ? 0.0f : base + logf(sum);   // (no expert is open to the token: it adds nothing)
#pragma unroll
    for (int v = 0; v < VPL; ++v) softmax[v] *= scale;
    if (!sigmoids) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) score[v] = softmax[v];
      return;
    }
    // (of sigmoids that are all too small for a float, what is left of them relative to the largest)
    const float least = fminf(base, 0.0f);
    float all = 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      score[v] = (x[v] >= 0.0f ? 1.0f : quick_exp(x[v] - least)) * __builtin_amdgcn_rcpf(1.0f + quick_exp(-fabsf(x[v])));
      all += score[v];
    }
    all = group_sum<G>(all);
    const float over = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
    for (int v = 0; v < VPL; ++v) score[v] *= over;
  }
};

template <int DT, int G, int VPL>
__global__ __launch_bounds__(kBalanceThreads) void balance_units_kernel(BalanceParams p) {
  constexpr int GROUPS = kBalanceThreads / G, COLUMNS = G * VPL;
  __shared__ float rows[GROUPS * COLUMNS];
  __shared__ int32_t chosen[COLUMNS];
  __shared__ float of_group_z[GROUPS];
  __shared__ int32_t of_group_tokens[GROUPS];
  const BalanceArgs& a = p.a;
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.arrived = 0;
  const int64_t first = (int64_t)blockIdx.x * p.chunk, last = min(first + p.chunk, a.tokens);
  int64_t at = first;
  for (int s = max(sequence_of(a.offsets, a.sequences, at), 0); s < a.sequences && at < last; ++s) {
    const int64_t begin = max(offset_of(a.offsets, a.tokens, s), at), end = min(offset_of(a.offsets, a.tokens, s + 1), last);
    if (begin >= last) break;
    if (begin >= end) continue;
    at = end;
    const int64_t unit = (int64_t)blockIdx.x + s;
    for (int e = threadIdx.x; e < a.experts; e += kBalanceThreads) chosen[e] = 0;
    __syncthreads();
    for (int64_t i = begin * a.top_k + threadIdx.x; i < end * a.top_k; i += kBalanceThreads) {
      const uint32_t e = (uint32_t)a.chosen[i];
      if (e < (uint32_t)a.experts && (a.mask == nullptr || a.mask[i / a.top_k] != 0)) atomicAdd(&chosen[e], 1);
    }
    float mass[VPL], z = 0.0f;
    int32_t tokens = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) mass[v] = 0.0f;
    for (int64_t t = begin + group; t < end; t += GROUPS) {
      if (a.mask != nullptr && a.mask[t] == 0) continue;
      Scores<DT, G, VPL> scores;
      scores.compute(load_logits<DT, VPL>(a.logits, t, a.experts, column), a.sigmoid);
#pragma unroll
      for (int v = 0; v < VPL; ++v) mass[v] += scores.score[v];
      z += scores.lse * scores.lse;
      ++tokens;
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v) rows[group * COLUMNS + column + v] = mass[v];
    if (l == 0) of_group_z[group] = z, of_group_tokens[group] = tokens;
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kBalanceThreads) {
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) sum += rows[g * COLUMNS + e];
      p.mass[unit * a.experts + e] = sum;
      p.counts[unit * a.experts + e] = chosen[e];
    }
    if (threadIdx.x == 0) {
      float sum = 0.0f;
      int32_t all = 0;
      for (int g = 0; g < GROUPS; ++g) sum += of_group_z[g], all += of_group_tokens[g];
      p.z[unit] = sum, p.tokens[unit] = all;
    }
    __syncthreads();   // (LDS is read before the next unit's sums)
  }
}

template <typename T>
__device__ __forceinline__ void store_shared(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T load_shared(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum over all threads of a workgroup, in every thread.
template <int THREADS, typename T>
__device__ __forceinline__ T block_sum(T v, T* lds) {
  v = group_reduce<64>(v, [](T p, T q) { return p + q; });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  T sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) sum += lds[w];
  return sum;
}

// A sequence's sums over its units, kSumColumns experts to a workgroup, whose waves take the units in turns.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void balance_sums_kernel(BalanceParams p) {
  constexpr int WAVES = THREADS / 64;
  __shared__ float mass_of[WAVES][64];
  __shared__ int32_t count_of[WAVES][64];
  __shared__ float sums[WAVES];
  __shared__ int32_t whole[WAVES];
  __shared__ int32_t arrived;
  const BalanceArgs& a = p.a;
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x / 64));
  const int64_t tasks = (int64_t)a.sequences * p.tiles;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int s = (int)(task / p.tiles), tile = (int)(task - (int64_t)s * p.tiles), e = tile * kSumColumns + lane;
    const int64_t begin = offset_of(a.offsets, a.tokens, s), end = offset_of(a.offsets, a.tokens, s + 1);
    const int64_t from = begin / p.chunk + s, to = begin < end ? (end - 1) / p.chunk + s + 1 : from;   // units
    float mass = 0.0f, z = 0.0f;
    int32_t count = 0, tokens = 0;
    if (e < a.experts) {
      for (int64_t u = from + wave; u < to; u += WAVES) mass += p.mass[u * a.experts + e], count += p.counts[u * a.experts + e];
    }
    for (int64_t u = from + threadIdx.x; u < to; u += THREADS) z += p.z[u], tokens += p.tokens[u];
    mass_of[wave][lane] = mass, count_of[wave][lane] = count;
    z = block_sum<THREADS>(z, sums);   // (barriers inside)
    tokens = block_sum<THREADS>(tokens, whole);
    float loss = 0.0f;
    if (wave == 0) {
      mass = 0.0f, count = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) mass += mass_of[w][lane], count += count_of[w][lane];
      const float share = tokens > 0 ? (float)count * (float)a.experts / ((float)a.top_k * (float)tokens) : 0.0f;
      if (e < a.experts) {
        a.counts[(int64_t)s * a.experts + e] = count;
        a.share[(int64_t)s * a.experts + e] = share;
        loss = share * mass;
      }
      loss = group_sum<64>(loss);
      if (lane == 0) {
        store_shared(p.loss + task, loss);
        if (tile == 0) store_shared(p.sequence_z + s, z), store_shared(p.sequence_tokens + s, tokens);
      }
    }
    __syncthreads();   // (LDS is read before the next task's sums)
  }
  // the last workgroup to arrive adds up the sequences
  wait_vmcnt<0>();
  __syncthreads();
  if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(p.arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != (int)gridDim.x - 1) return;
  float loss = 0.0f, z = 0.0f;
  int32_t tokens = 0;
  for (int64_t i = threadIdx.x; i < tasks; i += THREADS) loss += load_shared(p.loss + i);
  for (int i = threadIdx.x; i < a.sequences; i += THREADS) z += load_shared(p.sequence_z + i), tokens += load_shared(p.sequence_tokens + i);
  loss = block_sum<THREADS>(loss, sums);
  z = block_sum<THREADS>(z, sums);
  tokens = block_sum<THREADS>(tokens, whole);
  if (threadIdx.x == 0) {
    const float inverse = tokens > 0 ? 1.0f / (float)tokens : 0.0f;
    *a.balance = loss * inverse;
    *a.z = z * inverse;
    *a.inverse = inverse;
  }
}

// The gradient, one pass: workgroups take neighbouring tokens, a sequence's shares stay in registers.
template <int DT, int G, int VPL>
__global__ __launch_bounds__(kBalanceThreads) void balance_backward_kernel(BalanceBackwardArgs a, int chunk) {
  using T = typename Logit<DT>::T;
  constexpr int GROUPS = kBalanceThreads / G;
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL;
  const int64_t first = (int64_t)blockIdx.x * chunk, last = min(first + chunk, a.tokens);
  const float inverse = *a.inverse;
  const float of_balance = a.balance_grad != nullptr ? *a.balance_grad * inverse : 0.0f, of_z = a.z_grad != nullptr ? *a.z_grad * 2.0f * inverse : 0.0f;
  int s = sequence_of(a.offsets, a.sequences, first), held = -1;   // `held`: whose shares are here
  int64_t begin = s >= 0 && s < a.sequences ? offset_of(a.offsets, a.tokens, s) : a.tokens;
  int64_t end = s < a.sequences ? offset_of(a.offsets, a.tokens, s + 1) : a.tokens;   // (before the first sequence: it begins there)
  if (s >= a.sequences) begin = end = a.tokens;
  float share[VPL];
  for (int64_t t = first + group; t < last; t += GROUPS) {
    while (t >= end && s + 1 < a.sequences) {
      ++s;
      begin = offset_of(a.offsets, a.tokens, s), end = offset_of(a.offsets, a.tokens, s + 1);
    }
    Row<T, VPL> out;
    if (t < begin || t >= end || (a.mask != nullptr && a.mask[t] == 0)) {   // (not counted)
#pragma unroll
      for (int v = 0; v < VPL; ++v) out.v[v] = Logit<DT>::narrow(0.0f);
    } else {
      if (held != s) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) share[v] = column + v < a.experts ? a.share[(int64_t)s * a.experts + column + v] : 0.0f;
        held = s;
      }
      Scores<DT, G, VPL> scores;
      scores.compute(load_logits<DT, VPL>(a.logits, t, a.experts, column), a.sigmoid);
      float dot = 0.0f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) dot += scores.score[v] * share[v];
      dot = group_sum<G>(dot);
      const float of_softmax = of_z * scores.lse;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const float slope = a.sigmoid ? quick_sigmoid(-scores.x[v]) : 1.0f;
        out.v[v] = Logit<DT>::narrow(of_balance * scores.score[v] * slope * (share[v] - dot) + of_softmax * scores.softmax[v]);
      }
    }
    T* to = static_cast<T*>(a.logits_grad) + t * a.experts + column;
    if (column + VPL <= a.experts) {
      *reinterpret_cast<Row<T, VPL>*>(to) = out;
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (column + v < a.experts) to[v] = out.v[v];
    }
  }
}

// Tokens of a workgroup: at least a round, and no more than kBalanceBlocks workgroups.
int64_t chunk_of(int64_t tokens, int64_t experts) {
  const int64_t round = kBalanceThreads / (experts <= 256 ? 16 : 64), each = (tokens + kBalanceBlocks - 1) / kBalanceBlocks;
  return std::max(round, (each + round - 1) / round * round);
}
int64_t units_of(int64_t tokens, int64_t experts, int64_t sequences) {
  const int64_t chunk = chunk_of(tokens, experts);
  return (tokens + chunk - 1) / chunk + sequences;
}

struct BalanceScratch {
  int64_t units, tiles;
  uint64_t mass, counts, z, tokens, loss, sequence_z, sequence_tokens, bytes;   // where they are, behind the counter
};
BalanceScratch scratch_of(int64_t tokens, int64_t experts, int64_t sequences) {
  BalanceScratch b;
  b.units = units_of(tokens, experts, sequences);
  b.tiles = (experts + kSumColumns - 1) / kSumColumns;
  uint64_t at = 16;
  auto take = [&](int64_t words) {
    const uint64_t here = at;
    at += (uint64_t)words * 4;
    return here;
  };
  b.mass = take(b.units * experts), b.counts = take(b.units * experts), b.z = take(b.units), b.tokens = take(b.units);
  b.loss = take(sequences * b.tiles), b.sequence_z = take(sequences), b.sequence_tokens = take(sequences);
  b.bytes = at;
  return b;
}

template <int DT, int G, int VPL>
hipError_t launch_balance(const BalanceArgs& a, hipStream_t stream) {
  const BalanceScratch b = scratch_of(a.tokens, a.experts, a.sequences);
  char* at = static_cast<char*>(a.scratch);
  BalanceParams p;
  p.a = a;
  p.chunk = (int32_t)chunk_of(a.tokens, a.experts);
  p.tiles = (int32_t)b.tiles;
  p.arrived = reinterpret_cast<int32_t*>(at);
  p.mass = reinterpret_cast<float*>(at + b.mass), p.counts = reinterpret_cast<int32_t*>(at + b.counts);
  p.z = reinterpret_cast<float*>(at + b.z), p.tokens = reinterpret_cast<int32_t*>(at + b.tokens);
  p.loss = reinterpret_cast<float*>(at + b.loss), p.sequence_z = reinterpret_cast<float*>(at + b.sequence_z);
  p.sequence_tokens = reinterpret_cast<int32_t*>(at + b.sequence_tokens);
  // (without tokens the first kernel still clears the counter)
  const int64_t chunks = std::max<int64_t>(1, (a.tokens + p.chunk - 1) / p.chunk);
  hipLaunchKernelGGL((balance_units_kernel<DT, G, VPL>), dim3((uint32_t)chunks), dim3(kBalanceThreads), 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const uint32_t blocks = (uint32_t)std::max<int64_t>(1, std::min<int64_t>(a.sequences * b.tiles, 2048));
  if (chunks > 8 * a.sequences) {
    hipLaunchKernelGGL(balance_sums_kernel<1024>, dim3(blocks), dim3(1024), 0, stream, p);
  } else {
    hipLaunchKernelGGL(balance_sums_kernel<256>, dim3(blocks), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

template <int DT, int G, int VPL>
hipError_t launch_balance_backward(const BalanceBackwardArgs& a, hipStream_t stream) {
  const int64_t chunk = chunk_of(a.tokens, a.experts);
  hipLaunchKernelGGL((balance_backward_kernel<DT, G, VPL>), dim3((uint32_t)((a.tokens + chunk - 1) / chunk)), dim3(kBalanceThreads), 0, stream, a, (int)chunk);
  return hipGetLastError();
}

}  // namespace

uint64_t balance_scratch_bytes(int64_t tokens, int64_t experts, int64_t sequences) { return scratch_of(tokens, experts, sequences).bytes; }

#define GG_BY_EXPERTS(DT, launch, a, stream)                          \
  do {                                                                \
    if ((a).experts <= 64) return launch<DT, 16, 4>(a, stream);       \
    if ((a).experts <= 128) return launch<DT, 16, 8>(a, stream);      \
    if ((a).experts <= 256) return launch<DT, 16, 16>(a, stream);     \
    if ((a).experts <= 512) return launch<DT, 64, 8>(a, stream);      \
    return launch<DT, 64, 16>(a, stream);                             \
  } while (0)

hipError_t balance(const BalanceArgs& a, hipStream_t stream) {
  if (a.dt == kF32) GG_BY_EXPERTS(kF32, launch_balance, a, stream);
  if (a.dt == kBF16) GG_BY_EXPERTS(kBF16, launch_balance, a, stream);
  GG_BY_EXPERTS(kF16, launch_balance, a, stream);
}

hipError_t balance_backward(const BalanceBackwardArgs& a, hipStream_t stream) {
  if (a.dt == kF32) GG_BY_EXPERTS(kF32, launch_balance_backward, a, stream);
  if (a.dt == kBF16) GG_BY_EXPERTS(kBF16, launch_balance_backward, a, stream);
  GG_BY_EXPERTS(kF16, launch_balance_backward, a, stream);
}

}  // namespace gg
