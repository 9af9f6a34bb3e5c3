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
// Workgroups that the tokens are cut into, at most: four to a compute unit, all there at once.  Units / sums / backward in us with 512, 1024 and
// 2048: 65536 x 256, bf16, sigmoid, 64 sequences 18.2 / 7.3 / 25.1, 16.3 / 8.1 / 24.7, 17.9 / 10.4 / 29.7; softmax 14.5 / 7.3 / 23.3, 13.4 / 8.1 /
// 22.6, 14.9 / 10.4 / 28.0; 32768 x 128, 16 sequences 7.3 / 6.9 / 10.0, 6.7 / 9.0 / 9.8, 7.9 / 8.2 / 12.4; 65536 x 64, fp32, 8 9.2 / 7.2 / 10.0, 8.3 / 8.1 /
// 9.0, 9.2 / 9.2 / 8.6.
constexpr int64_t kBalanceBlocks = 1024;
// Units of a sequence, on average, up to which a wave adds them up, and needs no barrier for it.  All three kernels, wave / workgroup: 65536 x 64, 8192 sequences
// (1.1 units) 85 / 102 us; 4096 x 64, 512 25.7 / 29.7; 65536 x 256, 64 sequences (17) 57.5 / 52.
constexpr int64_t kWaveUnits = 8;

struct BalanceParams {
  BalanceArgs a;
  int32_t chunk;     // tokens of a workgroup
  int32_t tiles;     // of the second kernel's columns of experts
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
    const int step = (n - 1) / 64 + 1, at = lane * step;   // (of up to 2^31 - 1)
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

// A token's scores, in the lanes of its group, by one exponential (and, of sigmoids, one reciprocal) to a logit: with E = exp(x - top), softmax is E
// over its sum, and sigmoid(x) = E / (E + exp(-top)), 1 - sigmoid(x) = exp(-top) / (E + exp(-top)).  Where top is negative both divisors are
// taken times exp(top), which leaves sigmoids that are all too small for a float their proportions, and the division by their sum takes out
// again.  Above kFarTop sigmoids are computed by themselves: E, and a sigmoid with it, ends 87 below top, up to there at sigmoids of exp(-67), beyond at
// such as show (top 59: 4e-13).  (65536 x 256 logits, bf16, most tokens' largest above it: 62 us in place of 53, all three kernels.)
//
// top * log2 e is rounded, by at most half a unit in its last place, and each power of two comes out times two to that: a factor that all of a token's share, and
// that p and lse lose again, as long as it is near one.  Past kNoPower, where it is 2^(1/16) at most (at 3e9 it would be 2^72 or 2^-72, at
// 1e10 past a float's range), differences from top are taken first, which floats of that size have nearly exactly.
constexpr float kFarTop = 20.0f;
constexpr float kNoPower = 0x1p20f;

template <int DT, bool SIGMOID, int G, int VPL>
struct Scores {
  float e[VPL];                   // exponentials: softmax / of_softmax
  float s[SIGMOID ? VPL : 1];     // p / of_score (softmax: e),
  float slope[SIGMOID ? VPL : 1];   // ... and (1 - sigmoid) / of_slope
  float of_softmax, of_score, of_slope, lse;

  __device__ __forceinline__ float score(int v) const { return SIGMOID ? s[v] : e[v]; }

  __device__ __forceinline__ void compute(const Row<typename Logit<DT>::T, VPL>& raw) {
    constexpr float LOG2E = 1.44269504f;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      e[v] = Logit<DT>::widen(raw.v[v]);
      top = fmaxf(top, e[v]);
    }
    top = group_reduce<G>(top, [](float p, float q) { return fmaxf(p, q); });
    const float base = top == -INFINITY ? 0.0f : top;
    float base2 = base * LOG2E;
    auto bring_near = [&]() {
      if (__builtin_expect(__any(fabsf(base) > kNoPower), 0)) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) e[v] -= base;
        base2 = 0.0f;
      }
    };
    auto power = [&](float x) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, LOG2E, -base2)); };
    float sum = 0.0f, all = 0.0f;
    if constexpr (SIGMOID) {
      if (__builtin_expect(__any(base > kFarTop), 0)) {
        of_slope = 1.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          const float x = e[v], least = fminf(base, 0.0f);
          s[v] = (x >= 0.0f ? 1.0f : quick_exp(x - least)) * __builtin_amdgcn_rcpf(1.0f + quick_exp(-fabsf(x)));
          slope[v] = quick_sigmoid(-x);
        }
        bring_near();
#pragma unroll
        for (int v = 0; v < VPL; ++v) e[v] = power(e[v]);
      } else {
        const float less = __builtin_amdgcn_exp2f(-fabsf(base2)), of_e = base < 0.0f ? less : 1.0f;
        of_slope = base < 0.0f ? 1.0f : less;
        bring_near();
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          e[v] = power(e[v]);
          slope[v] = __builtin_amdgcn_rcpf(__builtin_fmaf(e[v], of_e, of_slope));
          s[v] = e[v] * slope[v];
        }
      }
#pragma unroll
      for (int v = 0; v < VPL; ++v) all += s[v];
      all = group_sum<G>(all);
    } else {
      bring_near();
#pragma unroll
      for (int v = 0; v < VPL; ++v) e[v] = power(e[v]);
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v) sum += e[v];
    sum = group_sum<G>(sum);
    // (no expert is open to the token: it adds nothing)
    of_softmax = sum == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum);
    lse = sum == 0.0f ? 0.0f : base + logf(sum);
    of_score = !SIGMOID ? of_softmax : (all == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(all));
  }
};

// A token's logits, asked for one turn ahead.
template <int DT, int G, int VPL>
struct NextToken {
  const void* logits;
  const uint8_t* mask;
  int experts, column;
  Row<typename Logit<DT>::T, VPL> raw;
  bool counted;
  __device__ __forceinline__ NextToken(const void* logits_, const uint8_t* mask_, int experts_, int column_)
      : logits(logits_), mask(mask_), experts(experts_), column(column_) {}
  __device__ __forceinline__ void ask(int64_t t, int64_t end) {
    if (t >= end) return;
    raw = load_logits<DT, VPL>(logits, t, experts, column);
    counted = mask == nullptr || mask[t] != 0;
  }
};

// (Four workgroups to a compute unit leave 128 registers.  Sigmoids of fp16, 16 to a lane, do not fit beside the next token's logits: 2 registers spill here with
// more than 512 experts, 4 in the gradient with 129 to 256 and 8 with more than 512.  65536 x 256, fp16 55 us, bf16 52, all three kernels.)
template <int DT, bool SIGMOID, int G, int VPL>
__global__ __launch_bounds__(kBalanceThreads, 4) void balance_units_kernel(BalanceParams p) {
  constexpr int GROUPS = kBalanceThreads / G, COLUMNS = G * VPL;
  __shared__ float rows[GROUPS * COLUMNS];
  __shared__ int32_t chosen[COLUMNS];
  __shared__ float of_group_z[GROUPS];
  __shared__ int32_t of_group_tokens[GROUPS];
  const BalanceArgs& a = p.a;
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.arrived = 0;
  const int64_t first = (int64_t)blockIdx.x * p.chunk, last = min(first + p.chunk, a.tokens);
  // (the first token's logits come while its sequence is looked for; they are asked for again where it begins later)
  NextToken<DT, G, VPL> next(a.logits, a.mask, a.experts, column);
  next.ask(first + group, last);
  int64_t at = first;
  bool empty = false;
  for (int s = max(sequence_of(a.offsets, a.sequences, at), 0); s < a.sequences && at < last; ++s) {
    const int64_t begin = max(offset_of(a.offsets, a.tokens, s), at), end = min(offset_of(a.offsets, a.tokens, s + 1), last);
    if (begin >= last) break;
    if (begin >= end) {   // behind a second empty one all that follow are left out at once
      if (empty) s = max(s, sequence_of(a.offsets, a.sequences, begin) - 1);
      empty = !empty;
      continue;
    }
    empty = false;
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
    if (begin != first) next.ask(begin + group, end);
    for (int64_t t = begin + group; t < end; t += GROUPS) {
      const auto raw = next.raw;
      const bool counted = next.counted;
      next.ask(t + GROUPS, end);
      if (!counted) continue;
      Scores<DT, SIGMOID, G, VPL> scores;
      scores.compute(raw);
#pragma unroll
      for (int v = 0; v < VPL; ++v) mass[v] = __builtin_fmaf(scores.score(v), scores.of_score, mass[v]);
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

// A sequence's sums over its units, COLUMNS experts at a time, by TEAM threads (a wave, or all), which take the units in turns.
template <int THREADS, int TEAM, int COLUMNS>
__global__ __launch_bounds__(THREADS) void balance_sums_kernel(BalanceParams p) {
  constexpr int WAVES = THREADS / 64, TURNS = TEAM / COLUMNS, IN_FLIGHT = 8;
  static_assert(TEAM == 64 || TEAM == THREADS, "");
  __shared__ float mass_of[TEAM == 64 ? 1 : TURNS][COLUMNS];
  __shared__ int32_t count_of[TEAM == 64 ? 1 : TURNS][COLUMNS];
  __shared__ float sums[WAVES];
  __shared__ int32_t whole[WAVES];
  __shared__ int32_t arrived;
  const BalanceArgs& a = p.a;
  const int member = threadIdx.x % TEAM, column = member % COLUMNS, turn = member / COLUMNS;
  const int64_t tasks = (int64_t)a.sequences * p.tiles;
  for (int64_t task = (int64_t)blockIdx.x * (THREADS / TEAM) + uniform((int)(threadIdx.x / TEAM)); task < tasks; task += (int64_t)gridDim.x * (THREADS / TEAM)) {
    const int s = (int)(task / p.tiles), tile = (int)(task - (int64_t)s * p.tiles), e = tile * COLUMNS + column;
    const int64_t begin = offset_of(a.offsets, a.tokens, s), end = offset_of(a.offsets, a.tokens, s + 1);
    const int64_t from = begin / p.chunk + s, to = begin < end ? (end - 1) / p.chunk + s + 1 : from;   // units
    float mass = 0.0f, z = 0.0f;
    int32_t count = 0, tokens = 0;
    if (e < a.experts && from < to) {
      for (int64_t u = from + turn; u < to; u += IN_FLIGHT * TURNS) {
        float m[IN_FLIGHT];
        int32_t n[IN_FLIGHT];
#pragma unroll
        for (int f = 0; f < IN_FLIGHT; ++f) {
          const int64_t at = min(u + f * TURNS, to - 1) * a.experts + e;
          m[f] = p.mass[at], n[f] = p.counts[at];
        }
#pragma unroll
        for (int f = 0; f < IN_FLIGHT; ++f)
          if (u + f * TURNS < to) mass += m[f], count += n[f];
      }
    }
    for (int64_t u = from + member; u < to; u += TEAM) z += p.z[u], tokens += p.tokens[u];
    if constexpr (TEAM == 64) {
      z = group_sum<64>(z);
      tokens = group_reduce<64>(tokens, [](int p, int q) { return p + q; });
#pragma unroll
      for (int d = COLUMNS; d < 64; d <<= 1) mass += __shfl_xor(mass, d), count += __shfl_xor(count, d);
    } else {
      mass_of[turn][column] = mass, count_of[turn][column] = count;
      z = block_sum<THREADS>(z, sums);   // (barriers inside)
      tokens = block_sum<THREADS>(tokens, whole);
      mass = 0.0f, count = 0;
      if (turn == 0)
#pragma unroll
        for (int w = 0; w < TURNS; ++w) mass += mass_of[w][column], count += count_of[w][column];
    }
    if (member < 64) {
      const float share = tokens > 0 ? (float)count * (float)a.experts / ((float)a.top_k * (float)tokens) : 0.0f;
      float loss = 0.0f;
      if (turn == 0 && e < a.experts) {
        a.counts[(int64_t)s * a.experts + e] = count;
        a.share[(int64_t)s * a.experts + e] = share;
        loss = share * mass;
      }
      loss = group_sum<64>(loss);
      if (member == 0) {
        store_shared(p.loss + task, loss);
        if (tile == 0) store_shared(p.sequence_z + s, z), store_shared(p.sequence_tokens + s, tokens);
      }
    }
    if constexpr (TEAM != 64) __syncthreads();   // (LDS is read before the next task's sums)
  }
  // the last workgroup to arrive adds up the sequences
  wait_vmcnt<0>();
  __syncthreads();
  if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(p.arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != (int)gridDim.x - 1) return;
  float loss = 0.0f, z = 0.0f;
  int32_t tokens = 0;
  for (int64_t first = threadIdx.x; first < tasks; first += IN_FLIGHT * THREADS) {
    float of_loss[IN_FLIGHT], of_z[IN_FLIGHT];
    int32_t of_tokens[IN_FLIGHT];
#pragma unroll
    for (int f = 0; f < IN_FLIGHT; ++f) {
      of_loss[f] = load_shared(p.loss + min(first + f * THREADS, tasks - 1));
      const int64_t s = min(first + f * THREADS, (int64_t)a.sequences - 1);
      of_z[f] = load_shared(p.sequence_z + s), of_tokens[f] = load_shared(p.sequence_tokens + s);
    }
#pragma unroll
    for (int f = 0; f < IN_FLIGHT; ++f) {
      if (first + f * THREADS < tasks) loss += of_loss[f];
      if (first + f * THREADS < a.sequences) z += of_z[f], tokens += of_tokens[f];
    }
  }
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

// VPL neighbouring results to any element of a row, the last lane's only as far as the row goes.  (In words: element by element each would be a
// store of its own, 16 in place of 2 for 256 experts, bf16: 27 us instead of 25 for 65536 tokens.)
template <int DT, int VPL>
__device__ __forceinline__ void store_logits(void* logits, int64_t token, int experts, int column, const float (&value)[VPL]) {
  using T = typename Logit<DT>::T;
  constexpr int WORDS = VPL * (int)sizeof(T) / 4;
  T* to = static_cast<T*>(logits) + token * experts + column;
  if (column + VPL <= experts) {
    using Words = __attribute__((ext_vector_type(WORDS < 4 ? WORDS : 4))) uint32_t;
    struct __attribute__((packed, aligned(sizeof(T)))) Packed {
      Words v;
    };
    uint32_t word[WORDS];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) word[w] = Logit<DT>::narrow(value[w]);
    } else {
#pragma unroll
      for (int w = 0; w < WORDS; w += 2) {
        const u32x2 four = round4<DT>(value[2 * w], value[2 * w + 1], value[2 * w + 2], value[2 * w + 3]);
        word[w] = four[0], word[w + 1] = four[1];
      }
    }
#pragma unroll
    for (int w = 0; w < WORDS; w += 4) {
      Words v;
#pragma unroll
      for (int i = 0; i < (WORDS < 4 ? WORDS : 4); ++i) v[i] = word[w + i];
      reinterpret_cast<Packed*>(reinterpret_cast<uint32_t*>(to) + w)->v = v;
    }
  } else {
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (column + v < experts) to[v] = Logit<DT>::narrow(value[v]);
  }
}

// The gradient, one pass: workgroups take neighbouring tokens, a sequence's shares stay in registers.
template <int DT, bool SIGMOID, int G, int VPL>
__global__ __launch_bounds__(kBalanceThreads, 4) void balance_backward_kernel(BalanceBackwardArgs a, int chunk) {
  constexpr int GROUPS = kBalanceThreads / G;
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL;
  const int64_t first = (int64_t)blockIdx.x * chunk, last = min(first + chunk, a.tokens);
  NextToken<DT, G, VPL> next(a.logits, a.mask, a.experts, column);
  next.ask(first + group, last);
  const float inverse = *a.inverse;
  const float of_balance = a.balance_grad != nullptr ? *a.balance_grad * inverse : 0.0f, of_z = a.z_grad != nullptr ? *a.z_grad * 2.0f * inverse : 0.0f;
  int s = sequence_of(a.offsets, a.sequences, first), held = -1;   // `held`: whose shares are here
  int64_t begin = s >= 0 && s < a.sequences ? offset_of(a.offsets, a.tokens, s) : a.tokens;
  int64_t end = s < a.sequences ? offset_of(a.offsets, a.tokens, s + 1) : a.tokens;   // (before the first sequence: it begins there)
  if (s >= a.sequences) begin = end = a.tokens;
  auto enter = [&](int sequence) {
    s = sequence;
    begin = offset_of(a.offsets, a.tokens, s), end = offset_of(a.offsets, a.tokens, s + 1);
  };
  float share[VPL];
  for (int64_t t = first + group; t < last; t += GROUPS) {
    const auto raw = next.raw;
    const bool counted = next.counted;
    next.ask(t + GROUPS, last);
    for (int further = 0; t >= end && s + 1 < a.sequences && further < 4; ++further) enter(s + 1);
    if (t >= end && s + 1 < a.sequences) {   // far from here: those that are left are halved
      int low = s + 1, high = a.sequences - 1;
      while (low < high) {
        const int middle = low + (high - low + 1) / 2;   // (their sum may pass 31 bits)
        if (offset_of(a.offsets, a.tokens, middle) <= t) low = middle;
        else high = middle - 1;
      }
      enter(low);
    }
    float grad[VPL];
    if (t < begin || t >= end || !counted) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) grad[v] = 0.0f;
    } else {
      if (held != s) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) share[v] = column + v < a.experts ? a.share[(int64_t)s * a.experts + column + v] : 0.0f;
        held = s;
      }
      Scores<DT, SIGMOID, G, VPL> scores;
      scores.compute(raw);
      float dot = 0.0f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) dot = __builtin_fmaf(scores.score(v), share[v], dot);
      dot = group_sum<G>(dot) * scores.of_score;
      const float of_score = of_balance * scores.of_score, of_softmax = of_z * scores.lse * scores.of_softmax;
      if constexpr (SIGMOID) {
        const float factor = of_score * scores.of_slope, rest = -dot * factor;
#pragma unroll
        for (int v = 0; v < VPL; ++v) grad[v] = scores.s[v] * scores.slope[v] * __builtin_fmaf(share[v], factor, rest);
        // (without a gradient of z its softmax stays out: that of a row with +inf is NaN, the balance of its sigmoids is not)
        if (a.z_grad != nullptr) {
#pragma unroll
          for (int v = 0; v < VPL; ++v) grad[v] = __builtin_fmaf(of_softmax, scores.e[v], grad[v]);
        }
      } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) grad[v] = scores.e[v] * __builtin_fmaf(share[v] - dot, of_score, of_softmax);
      }
    }
    store_logits<DT, VPL>(a.logits_grad, t, a.experts, column, grad);
  }
}

// Tokens of a workgroup: at least a round (a token to each group of lanes), and no more than kBalanceBlocks workgroups.  A workgroup takes its sequences one after the
// other, about 1.6 us each, so that where they are shorter than a round it has as many tokens as they have on average.  (All three kernels, with / without that
// and the searches behind empty sequences: 50 tokens x 9, 50 sequences 19 / 94 us; 13 x 111, 69 19 / 62; 280 x 74, 109 23 / 37; 5088 x 4, 111 27 / 28.)
int64_t chunk_of(int64_t tokens, int64_t experts, int64_t sequences) {
  const int64_t round = kBalanceThreads / (experts <= 16 ? 4 : (experts <= 256 ? 16 : 64)), each = (tokens + kBalanceBlocks - 1) / kBalanceBlocks;
  if (each > round) return (each + round - 1) / round * round;
  const int64_t average = sequences > 0 ? (tokens + sequences - 1) / sequences : tokens;
  return std::max<int64_t>({std::min(round, average), each, 1});
}
int64_t units_of(int64_t tokens, int64_t experts, int64_t sequences) {
  const int64_t chunk = chunk_of(tokens, experts, sequences);
  return (tokens + chunk - 1) / chunk + sequences;
}

struct BalanceScratch {
  int64_t units, tiles;
  int columns;          // of the second kernel's workgroups
  int threads, team;    // ... of these workgroups, and of those that take a sequence's tile
  uint64_t mass, counts, z, tokens, loss, sequence_z, sequence_tokens, bytes;   // where they are, behind the counter
};
BalanceScratch scratch_of(int64_t tokens, int64_t experts, int64_t sequences) {
  BalanceScratch b;
  b.units = units_of(tokens, experts, sequences);
  b.threads = b.units > 65 * sequences ? 1024 : 256;
  b.team = b.units <= kWaveUnits * sequences ? 64 : b.threads;
  // Where a sequence has more than 64 units, 1024 threads take them, so that each has few to wait for, and 32 columns, so that more workgroups do
  // (all three kernels of 65536 x 256, one sequence: 50.6 us with 64 columns, 48.0 with 32, 49.0 with 16, 49.7 with 8).  Otherwise whole rows of
  // 64 columns are better, as one workgroup takes each sequence's tile (64 sequences: 53.2, with 16 columns 62.8).  Few experts leave
  // wider tiles idle lanes (65536 x 8, 16 sequences: 28.6 with 64 columns, 24.5 with 16, the units' kernel being what it was).
  b.columns = experts <= 16 ? 16 : (b.threads == 1024 ? 32 : 64);
  b.tiles = (experts + b.columns - 1) / b.columns;
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

template <int DT, bool SIGMOID, int G, int VPL>
hipError_t launch_balance(const BalanceArgs& a, hipStream_t stream) {
  const BalanceScratch b = scratch_of(a.tokens, a.experts, a.sequences);
  char* at = static_cast<char*>(a.scratch);
  BalanceParams p;
  p.a = a;
  p.chunk = (int32_t)chunk_of(a.tokens, a.experts, a.sequences);
  p.tiles = (int32_t)b.tiles;
  p.arrived = reinterpret_cast<int32_t*>(at);
  p.mass = reinterpret_cast<float*>(at + b.mass), p.counts = reinterpret_cast<int32_t*>(at + b.counts);
  p.z = reinterpret_cast<float*>(at + b.z), p.tokens = reinterpret_cast<int32_t*>(at + b.tokens);
  p.loss = reinterpret_cast<float*>(at + b.loss), p.sequence_z = reinterpret_cast<float*>(at + b.sequence_z);
  p.sequence_tokens = reinterpret_cast<int32_t*>(at + b.sequence_tokens);
  // (without tokens the first kernel still clears the counter)
  const int64_t chunks = std::max<int64_t>(1, (a.tokens + p.chunk - 1) / p.chunk);
  hipLaunchKernelGGL((balance_units_kernel<DT, SIGMOID, G, VPL>), dim3((uint32_t)chunks), dim3(kBalanceThreads), 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int64_t teams = b.threads / b.team, tasks = a.sequences * b.tiles;
  const dim3 blocks((uint32_t)std::max<int64_t>(1, std::min<int64_t>((tasks + teams - 1) / teams, 2048))), threads(b.threads);
  const bool few = b.columns == 16;
  if (b.threads == 1024) {
    if (few) hipLaunchKernelGGL((balance_sums_kernel<1024, 1024, 16>), blocks, threads, 0, stream, p);
    else hipLaunchKernelGGL((balance_sums_kernel<1024, 1024, 32>), blocks, threads, 0, stream, p);
  } else if (b.team == 64) {
    if (few) hipLaunchKernelGGL((balance_sums_kernel<256, 64, 16>), blocks, threads, 0, stream, p);
    else hipLaunchKernelGGL((balance_sums_kernel<256, 64, 64>), blocks, threads, 0, stream, p);
  } else {
    if (few) hipLaunchKernelGGL((balance_sums_kernel<256, 256, 16>), blocks, threads, 0, stream, p);
    else hipLaunchKernelGGL((balance_sums_kernel<256, 256, 64>), blocks, threads, 0, stream, p);
  }
  return hipGetLastError();
}

template <int DT, bool SIGMOID, int G, int VPL>
hipError_t launch_balance_backward(const BalanceBackwardArgs& a, hipStream_t stream) {
  const int64_t chunk = chunk_of(a.tokens, a.experts, a.sequences);
  hipLaunchKernelGGL((balance_backward_kernel<DT, SIGMOID, G, VPL>), dim3((uint32_t)((a.tokens + chunk - 1) / chunk)), dim3(kBalanceThreads), 0, stream, a, (int)chunk);
  return hipGetLastError();
}

}  // namespace

uint64_t balance_scratch_bytes(int64_t tokens, int64_t experts, int64_t sequences) { return scratch_of(tokens, experts, sequences).bytes; }

// The fewest lanes that hold a token's logits, 16 each at most: more of them leave lanes idle, and each reduction takes more steps.  (16 lanes
// for up to 16 experts, as up to 64: 65536 x 8, 16 sequences, 28.6 us in place of 20.9; 8192 x 8, 20.0 in place of 18.4.)
#define GG_BY_EXPERTS(DT, SIGMOID, launch, a, stream)                   \
  do {                                                                  \
    if ((a).experts <= 16) return launch<DT, SIGMOID, 4, 4>(a, stream);      \
    if ((a).experts <= 64) return launch<DT, SIGMOID, 16, 4>(a, stream);     \
    if ((a).experts <= 128) return launch<DT, SIGMOID, 16, 8>(a, stream);    \
    if ((a).experts <= 256) return launch<DT, SIGMOID, 16, 16>(a, stream);   \
    if ((a).experts <= 512) return launch<DT, SIGMOID, 64, 8>(a, stream);    \
    return launch<DT, SIGMOID, 64, 16>(a, stream);                           \
  } while (0)
#define GG_BY_TYPE(SIGMOID, launch, a, stream)                              \
  do {                                                                      \
    if ((a).dt == kF32) GG_BY_EXPERTS(kF32, SIGMOID, launch, a, stream);    \
    if ((a).dt == kBF16) GG_BY_EXPERTS(kBF16, SIGMOID, launch, a, stream);  \
    GG_BY_EXPERTS(kF16, SIGMOID, launch, a, stream);                        \
  } while (0)

hipError_t balance(const BalanceArgs& a, hipStream_t stream) {
  if (a.sigmoid) GG_BY_TYPE(true, launch_balance, a, stream);
  GG_BY_TYPE(false, launch_balance, a, stream);
}

hipError_t balance_backward(const BalanceBackwardArgs& a, hipStream_t stream) {
  if (a.sigmoid) GG_BY_TYPE(true, launch_balance_backward, a, stream);
  GG_BY_TYPE(false, launch_balance_backward, a, stream);
}

}  // namespace gg
