// The router: scores of each token's experts, the top_k of them, and the order that sorts the chosen rows by expert.
//
//   s = softmax(l) or sigmoid(l); the top_k largest logits are chosen, ties by the lower index;
//   w_j = s[e_j], divided by the sum over the chosen where `normalize` is set;  mass[e] = sum over tokens of s[e].
//
// A token all of whose logits are -inf has scores and weights of zero (and, as every token, top_k chosen experts).  NaN
// counts as larger than any number; the weights of its token are then NaN, as the formulas give them.
//
// Sorting is by counting, in a fixed order: a workgroup counts its tokens' experts, the counts are summed over
// the workgroups before each, and the rows are placed by how many earlier rows of the same expert there are.
//
// Choosing is bound by the vector units' issue: every logit is read once, but takes an exponential (four times the time of an addition), and a
// subtraction and half a maximum for each of the top_k.  65536 tokens of 256 experts, bf16, sigmoid, top 8: choosing 26 us (33.6 MB: 1.3 TB/s;
// vector instructions in 81 % of the cycles), summing the counts 5, placing 524288 rows 11 (latency of scattered 4-byte stores), the gradient 26 (67
// MB and the chosen: 2.7 TB/s; vector instructions in half of the cycles, memory's latency in the others: a token's loads follow one another, see
// there).  Few tokens are bound by the launches: one token 3.8 us in one, 8192 of 64 experts 5 + 4 + 4 and 4.
#include "operators.hpp"

#include <math.h>

#include <type_traits>

#include "gmm_kernel.hpp"
#include "logits.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kRouteThreads = 512;
constexpr int kRouteWaves = kRouteThreads / 64;
// Workgroups that choose and place, at most: two on each of 256 compute units; a column of their counts is 8 words for each lane of the wave
// that sums it.  Choosing, summing, placing for 65536 tokens of 256 experts with 256, 512, 1024: 29 + 4.7 + 12, 27 + 4.8 + 13, 28 + 7 + 13 us (placing now 11).
constexpr int kRouteBlocks = 512;
// Up to this many tokens and chosen rows one workgroup does everything in one launch.  That and three launches (their sum, without what lies
// between them), us: 1 token of 64 experts 3.6, 8.6; 64 of 64 5.0, 9.6; 64 of 256 7.4, 12; 128 of 64 8.8, 10.0; 256 of 64 14.7, 11.1; 256 of 256
// 30, 13.
constexpr int kSmallTokens = 64, kSmallSlots = 2048;

// Whole numbers ordered as the floats are: -0 equal to +0, NaN above all, 0 below all.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.0f);
  const uint32_t key = bits ^ ((bits & 0x80000000u) ? 0xffffffffu : 0x80000000u);
  return x != x ? 0xffffffffu : key;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// ... and of the bits of a two-byte type, in the upper half, with the lane's columns below in falling order: with key_of_lane() added, no two
// keys of a token are equal.  Two elements at a time; -0 and NaN, which few tokens have, are looked for first and made +0 and one NaN.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

template <int DT, int VPL>
__device__ __forceinline__ void unique_keys(const uint16_t (&bits)[VPL], uint32_t (&key)[VPL]) {
  constexpr uint16_t INFINITE = DT == kBF16 ? 0x7f80 : 0x7c00;
  u16x2 pair[VPL / 2], most = {0, 0}, least = {0xffff, 0xffff};
#pragma unroll
  for (int i = 0; i < VPL / 2; ++i) {
    pair[i] = u16x2{bits[2 * i], bits[2 * i + 1]};
    most = __builtin_elementwise_max(most, pair[i] & (uint16_t)0x7fff);
    least = __builtin_elementwise_min(least, pair[i] ^ (uint16_t)0x8000);
  }
  if (__any(most.x > INFINITE || most.y > INFINITE || least.x == 0 || least.y == 0)) {
#pragma unroll
    for (int i = 0; i < VPL / 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint16_t one = pair[i][e];
        pair[i][e] = one == 0x8000 ? uint16_t(0) : ((one & 0x7fff) > INFINITE ? uint16_t(0x7fff) : one);
      }
  }
#pragma unroll
  for (int i = 0; i < VPL / 2; ++i) {
    const u16x2 sign = __builtin_bit_cast(u16x2, __builtin_bit_cast(i16x2, pair[i]) >> (int16_t)15);
    const uint32_t both = __builtin_bit_cast(uint32_t, pair[i] ^ (sign | (uint16_t)0x8000));
    key[2 * i] = both << 16 | (uint32_t)(VPL - 1 - 2 * i);
    key[2 * i + 1] = (both & 0xffff0000u) | (uint32_t)(VPL - 2 - 2 * i);
  }
}
template <int VPL>
__device__ __forceinline__ uint32_t key_of_lane(int column) { return (uint32_t)(0xffff - column - (VPL - 1)); }
template <int DT>
__device__ __forceinline__ float unique_key_value(uint32_t key) {
  if constexpr (DT == kF32) return 0.0f;
  else return Logit<DT>::widen((typename Logit<DT>::T)((key >> 16) ^ ((key >> 31) ? 0x8000u : 0xffffu)));
}

struct RouteParams {
  RouteArgs a;
  int32_t chunk;           // tokens of a workgroup
  int32_t blocks;
  int32_t* counts;         // [experts][blocks] chosen rows of each workgroup; then those of the workgroups before it
  float* mass_parts;       // [experts][blocks]
};

// Chooses for tokens first + group, first + group + groups, ... below last: a group of G lanes has one token,
// each lane VPL neighbouring columns.  One round of a maximum over the group for each of the top_k.
// counts[e] (in LDS) is raised for each chosen row, slots (in LDS, or null) receive the experts of the rows from `first`
// on, mass the lane's share of the scores' sums.
template <int DT, int G, int VPL>
__device__ __forceinline__ void choose(const RouteArgs& a, int64_t first, int64_t last, int32_t* counts, int32_t* slots, float (&mass)[VPL]) {
#pragma unroll
  for (int v = 0; v < VPL; ++v) mass[v] = 0.0f;
  constexpr int KR = G == 16 ? 2 : 1;   // chosen experts a lane may hold: numbers l and l + 16
  static_assert(KR * G >= kRouteMaxTopK, "");
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL, k = a.top_k;
  const bool all_scores = a.mass != nullptr || !(a.normalize || a.sigmoid);
  for (int64_t t = first + group; t < last; t += kRouteThreads / G) {
    const auto raw = load_logits<DT, VPL>(a.logits, t, a.experts, column);
    constexpr bool UNIQUE = DT != kF32;
    float x[VPL];
    uint32_t key[VPL];   // (columns past the last are -inf, and behind all of the same: top_k others go before them)
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      x[v] = Logit<DT>::widen(raw.v[v]);
      if constexpr (!UNIQUE) key[v] = order_key(x[v]);
    }
    if constexpr (UNIQUE) unique_keys<DT>(raw.v, key);
    uint32_t chosen_key[KR], top_key = 0u, last = 0u;
    int index[KR];
#pragma unroll
    for (int r = 0; r < KR; ++r) chosen_key[r] = 0u, index[r] = 0;
    for (int j = 0; j < k; ++j) {
      uint32_t best, at = ~0u;
      if constexpr (UNIQUE) {
        // the largest below the last: modulo 2^32, the differences of those below are larger than all others, and in their order
        const uint32_t from = last - key_of_lane<VPL>(column);
        best = key[0] - from;
#pragma unroll
        for (int v = 1; v < VPL; ++v) best = max(best, key[v] - from);
        best = group_max<G>(best) + last;
        last = best;
      } else {
        best = key[0];
#pragma unroll
        for (int v = 1; v < VPL; ++v) best = max(best, key[v]);
        best = group_max<G>(best);
#pragma unroll
        for (int v = VPL - 1; v >= 0; --v) at = key[v] == best ? (uint32_t)(column + v) : at;
        at = group_min<G>(at);
#pragma unroll
        for (int v = 0; v < VPL; ++v) key[v] = at == (uint32_t)(column + v) ? 0u : key[v];
      }
      if (j == 0) top_key = best;
#pragma unroll
      for (int r = 0; r < KR; ++r)
        if (r * G <= j && j == l + r * G) chosen_key[r] = best, index[r] = (int)at;
    }
    auto decode = [](uint32_t key) { return UNIQUE ? unique_key_value<DT>(key) : key_value(key); };
    const float top = decode(top_key);
    float value[KR];
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      value[r] = decode(chosen_key[r]);
      if (UNIQUE) index[r] = 0xffff - (int)(chosen_key[r] & 0xffffu);
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float share[KR], scale = 0.0f;
    if (all_scores) {
      if (a.sigmoid) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) mass[v] += quick_sigmoid(x[v]);
      } else {
        float s[VPL], sum = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          s[v] = quick_exp(x[v] - base);
          sum += s[v];
        }
        sum = group_sum<G>(sum);
        scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int v = 0; v < VPL; ++v) mass[v] += s[v] * scale;
      }
    }
    if (a.normalize) {
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        share[r] = 0.0f;
        if (r * G >= k) continue;   // (the same in all lanes)
        share[r] = a.sigmoid ? scaled_sigmoid(value[r], base) : expf(value[r] - base);
        if (l + r * G >= k) share[r] = 0.0f;
        sum += share[r];
      }
      sum = group_sum<G>(sum);
#pragma unroll
      for (int r = 0; r < KR; ++r) share[r] = sum == 0.0f ? 0.0f : share[r] / sum;
    } else {
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        share[r] = 0.0f;
        if (r * G < k) share[r] = a.sigmoid ? sigmoid(value[r]) : expf(value[r] - base) * scale;
      }
    }
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      const int j = l + r * G;
      if (j >= k) continue;
      a.weights[t * k + j] = share[r];
      a.chosen[t * k + j] = index[r];
      if (slots != nullptr) slots[(t - first) * k + j] = index[r];
      atomicAdd(&counts[index[r]], 1);
    }
  }
}

// The workgroup's share of the scores' sums: waves' shares through LDS ([kRouteWaves][experts]), added up in their order.
template <int G, int VPL, typename Store>
__device__ __forceinline__ void sum_mass(float (&mass)[VPL], float* parts, int experts, Store store) {
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, column = threadIdx.x % G * VPL;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    if constexpr (G == 16) {
      mass[v] += __shfl_xor(mass[v], 16);
      mass[v] += __shfl_xor(mass[v], 32);
    }
    if (lane < G && column + v < experts) parts[wave * experts + column + v] = mass[v];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kRouteThreads) {
    float sum = 0.0f;
    for (int w = 0; w < kRouteWaves; ++w) sum += parts[w * experts + e];
    store(e, sum);
  }
}

// Lanes of the wave whose expert is the same; `bits` bits of it matter.
__device__ __forceinline__ uint64_t same_expert(int e, int bits, uint64_t valid) {
  uint64_t same = valid;
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((e >> b) & 1);
    same &= (e >> b) & 1 ? set : ~set;
  }
  return same;
}

// Places n chosen rows, expert(i) being that of the i-th: the waves take shares of them in order.  `next` is LDS,
// [kRouteWaves][experts]; start(e) is where the workgroup's first row of expert e goes.  first_slot: number of its first row.
template <typename Expert, typename Start>
__device__ __forceinline__ void place(int n, int experts, int top_k, int64_t first_slot, int32_t* next, Expert expert, Start start,
                                      int32_t* row_index, int32_t* order) {
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, bits = 32 - __clz(experts - 1 > 0 ? experts - 1 : 1);
  const int share = ((n + kRouteWaves - 1) / kRouteWaves + 63) / 64 * 64;
  const int begin = wave * share, end = begin + share < n ? begin + share : n;
  int32_t* mine = next + wave * experts;
  for (int i = threadIdx.x; i < kRouteWaves * experts; i += kRouteThreads) next[i] = 0;
  __syncthreads();
  for (int i = begin + lane; i < end; i += 64) atomicAdd(&mine[expert(i)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kRouteThreads) {
    int at = start(e);
    for (int w = 0; w < kRouteWaves; ++w) {
      const int count = next[w * experts + e];
      next[w * experts + e] = at;
      at += count;
    }
  }
  __syncthreads();
  for (int i0 = begin; i0 < end; i0 += 64) {   // (whole waves)
    const int i = i0 + lane;
    const bool valid = i < end;
    const int e = valid ? expert(i) : 0;
    const uint64_t same = same_expert(e, bits, __ballot(valid));
    if (!valid) continue;
    const int first = __ffsll((unsigned long long)same) - 1;
    const int before = __popcll(same & ((uint64_t(1) << lane) - 1));
    int at = 0;
    if (lane == first) at = atomicAdd(&mine[e], __popcll(same));
    at = __shfl(at, first) + before;
    const int64_t slot = first_slot + i;
    order[at] = (int32_t)slot;
    row_index[at] = (int32_t)(slot / top_k);
  }
}

// Exclusive prefix sums of the experts' counts, in LDS; all threads, ends with a barrier.
template <typename Count>
__device__ __forceinline__ void expert_starts(int experts, int32_t* starts, Count count) {
  __shared__ int32_t totals[kRouteWaves];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  int before = 0;
  for (int e0 = 0; e0 < experts; e0 += kRouteThreads) {
    const int e = e0 + (int)threadIdx.x, mine = e < experts ? count(e) : 0, upto = wave_prefix(mine);
    if (lane == 63) totals[wave] = upto;
    __syncthreads();
    int at = before + upto - mine;
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) {
      at += w < wave ? totals[w] : 0;
      before += totals[w];
    }
    if (e < experts) starts[e] = at;
    __syncthreads();
  }
}

// Everything in one workgroup, for the few tokens of a decode step, where a second launch would cost more than the rest.
template <int DT, int G, int VPL>
__global__ __launch_bounds__(kRouteThreads) void route_small_kernel(RouteArgs a) {
  extern __shared__ int32_t lds[];
  int32_t *counts = lds, *starts = counts + a.experts, *slots = starts + a.experts, *next = slots + kSmallSlots;
  const int tid = threadIdx.x;
  for (int e = tid; e < a.experts; e += kRouteThreads) counts[e] = 0;
  __syncthreads();
  float mass[VPL];
  choose<DT, G, VPL>(a, 0, a.tokens, counts, slots, mass);
  if (a.mass != nullptr) {
    sum_mass<G, VPL>(mass, reinterpret_cast<float*>(next), a.experts, [&](int e, float sum) { a.mass[e] = sum; });
  }
  __syncthreads();
  for (int e = tid; e < a.experts; e += kRouteThreads) a.batch_sizes[e] = counts[e];
  expert_starts(a.experts, starts, [&](int e) { return counts[e]; });
  place((int)a.tokens * a.top_k, a.experts, a.top_k, 0, next, [&](int i) { return slots[i]; }, [&](int e) { return starts[e]; },
        a.row_index, a.order);
}

template <int DT, int G, int VPL>
__global__ __launch_bounds__(kRouteThreads) void route_choose_kernel(RouteParams p) {
  extern __shared__ int32_t lds[];
  const RouteArgs& a = p.a;
  int32_t* counts = lds;
  const int tid = threadIdx.x;
  for (int e = tid; e < a.experts; e += kRouteThreads) counts[e] = 0;
  __syncthreads();
  float mass[VPL];
  const int64_t first = (int64_t)blockIdx.x * p.chunk, last = first + p.chunk < a.tokens ? first + p.chunk : a.tokens;
  choose<DT, G, VPL>(a, first, last, counts, nullptr, mass);
  if (a.mass != nullptr) {
    sum_mass<G, VPL>(mass, reinterpret_cast<float*>(counts + a.experts), a.experts,
                     [&](int e, float sum) { p.mass_parts[(int64_t)e * p.blocks + blockIdx.x] = sum; });
  }
  __syncthreads();
  for (int e = tid; e < a.experts; e += kRouteThreads) p.counts[(int64_t)e * p.blocks + blockIdx.x] = counts[e];
}

// One wave for each expert: its count in all workgroups, and in those before each.
__global__ __launch_bounds__(256) void route_scan_kernel(RouteParams p) {
  const int e = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (e >= p.a.experts) return;
  constexpr int EACH = kRouteBlocks / 64;
  int32_t* column = p.counts + (int64_t)e * p.blocks;
  int count[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int b = lane * EACH + i;
    count[i] = b < p.blocks ? column[b] : 0;
    sum += count[i];
  }
  const int upto = wave_prefix(sum);
  int at = upto - sum;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int b = lane * EACH + i;
    if (b < p.blocks) column[b] = at;
    at += count[i];
  }
  if (lane == 63) p.a.batch_sizes[e] = upto;
  if (p.a.mass != nullptr) {
    const float* parts = p.mass_parts + (int64_t)e * p.blocks;
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int b = i * 64 + lane;
      m += b < p.blocks ? parts[b] : 0.0f;
    }
    m = group_sum<64>(m);
    if (lane == 0) p.a.mass[e] = m;
  }
}

__global__ __launch_bounds__(kRouteThreads) void route_place_kernel(RouteParams p) {
  extern __shared__ int32_t lds[];
  const RouteArgs& a = p.a;
  int32_t *starts = lds, *next = lds + a.experts;
  // (asked for before anything waits: where this workgroup's rows of the thread's experts begin)
  constexpr int EACH = (int)kRouteMaxExperts / kRouteThreads;
  int own[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = i * kRouteThreads + (int)threadIdx.x;
    own[i] = e < a.experts ? p.counts[(int64_t)e * p.blocks + blockIdx.x] : 0;
  }
  expert_starts(a.experts, starts, [&](int e) { return (int)a.batch_sizes[e]; });
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = i * kRouteThreads + (int)threadIdx.x;
    if (e < a.experts) starts[e] += own[i];   // (its own thread's only, here and in place())
  }
  const int64_t first = (int64_t)blockIdx.x * p.chunk, last = first + p.chunk < a.tokens ? first + p.chunk : a.tokens;
  const int32_t* chosen = a.chosen + first * a.top_k;
  place((int)(last - first) * a.top_k, a.experts, a.top_k, first * a.top_k, next, [&](int i) { return chosen[i]; },
        [&](int e) { return starts[e]; }, a.row_index, a.order);
}

// Gradient of the logits, one pass: with g the gradients of the chosen weights and m those of the mass,
//   softmax  s (u - <u, s>), u = m, and g at the chosen where the weights are the scores themselves;
//   sigmoid  s (1 - s) u;
//   normalized weights q = w add q_j (g_j - <g, q>) at the chosen (times 1 - s_j with the sigmoid).
// What falls on the chosen columns goes to their lanes through LDS, one row of it for each group.
constexpr int kBackThreads = 256;
constexpr int64_t kBackBlocks = 1024;   // (65536 tokens of 256 experts, 512, 768, 1024, 1280, 2048: 30, 27, 26, 33, 33 us; of 64: 17, 13, 12, 12, 12)

template <int DT, int G, int VPL>
__global__ __launch_bounds__(kBackThreads, 4) void route_backward_kernel(RouteBackwardArgs a) {
  using T = typename Logit<DT>::T;
  constexpr int KR = G == 16 ? 2 : 1, GROUPS = kBackThreads / G, PITCH = VPL + 4;   // (of a lane's columns in LDS: 16 lanes start in different banks)
  __shared__ __attribute__((aligned(16))) float rows[GROUPS * G * PITCH];
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL, k = a.top_k;
  float *row = rows + group * G * PITCH, *own = row + l * PITCH;
  float m[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) m[v] = a.mass_grad != nullptr && column + v < a.experts ? a.mass_grad[column + v] : 0.0f;
  // The next token's rows are read ahead, but what is made of them here waits for them here: `chosen` is compared, and two-byte rows are taken apart.
  // With the chosen logits, which are gathered from memory, a token has three waits for memory, one after the other.
  Row<T, VPL> next_raw;
  int next_index[KR];
  float next_grad[KR];
  auto ask = [&](int64_t t) {
    if (t >= a.tokens) return;
    next_raw = load_logits<DT, VPL>(a.logits, t, a.experts, column);
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      const int j = l + r * G;
      next_index[r] = j < k ? a.chosen[t * k + j] : -1;
      if ((uint32_t)next_index[r] >= (uint32_t)a.experts) next_index[r] = -1;   // (names no expert: no gradient)
      next_grad[r] = j < k && a.weights_grad != nullptr ? a.weights_grad[t * k + j] : 0.0f;
    }
  };
  const int64_t stride = (int64_t)gridDim.x * GROUPS;
  int64_t t = (int64_t)blockIdx.x * GROUPS + group;
  ask(t);
  for (; t < a.tokens; t += stride) {
    const auto raw = next_raw;
    float value[KR], grad[KR];   // what falls on the chosen columns
    int index[KR];
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      index[r] = next_index[r];
      grad[r] = index[r] >= 0 ? next_grad[r] : 0.0f;
      value[r] = index[r] >= 0 ? Logit<DT>::widen(static_cast<const T*>(a.logits)[t * a.experts + index[r]]) : -INFINITY;
    }
    ask(t + stride);
    auto x = [&](int v) { return Logit<DT>::widen(raw.v[v]); };
    float top = -INFINITY;   // of all columns, or, for sigmoids, of the chosen
    if (a.sigmoid) {
#pragma unroll
      for (int r = 0; r < KR; ++r) top = fmaxf(top, value[r]);
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v) top = fmaxf(top, x(v));
    }
    top = group_reduce<G>(top, [](float p, float q) { return fmaxf(p, q); });
    const float base = top == -INFINITY ? 0.0f : top;
    if (a.normalize) {
      float q[KR], sum = 0.0f, dot = 0.0f;
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        q[r] = 0.0f;
        if (r * G >= k) continue;   // (the same in all lanes)
        if (index[r] >= 0) q[r] = a.sigmoid ? scaled_sigmoid(value[r], base) : expf(value[r] - base);
        sum += q[r];
      }
      sum = group_sum<G>(sum);
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        q[r] = sum == 0.0f ? 0.0f : q[r] / sum;
        dot += q[r] * grad[r];
      }
      dot = group_sum<G>(dot);
#pragma unroll
      for (int r = 0; r < KR; ++r)
        if (r * G < k) grad[r] = q[r] * (grad[r] - dot) * (a.sigmoid ? sigmoid(-value[r]) : 1.0f);
    }
    // (a row belongs to one wave, whose LDS accesses stay in order)
#pragma unroll
    for (int v = 0; v < VPL; ++v) own[v] = 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < KR; ++r)
      if (index[r] >= 0) row[index[r] / VPL * PITCH + index[r] % VPL] = grad[r];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // (scores are computed where they are needed, of the softmax twice: registers are what this kernel is short of)
    Row<T, VPL> out;
    auto finish = [&](auto normalized) {
      auto gradient = [&](int v) { return normalized ? m[v] : m[v] + own[v]; };   // of the column's score
      auto rest = [&](int v) { return normalized ? own[v] : 0.0f; };
      if (normalized && a.mass_grad == nullptr) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) out.v[v] = Logit<DT>::narrow(own[v]);
      } else if (a.sigmoid) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          // s (1 - s), the same for x and -x, without the difference, which would lose all of a small one
          const float e = quick_exp(-fabsf(x(v))), score = __builtin_amdgcn_rcpf(1.0f + e);
          out.v[v] = Logit<DT>::narrow(rest(v) + score * (e * score) * gradient(v));
        }
      } else {
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          const float s = quick_exp(x(v) - base);
          sum += s;
          dot += s * gradient(v);
        }
        sum = group_sum<G>(sum);
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        dot = group_sum<G>(dot) * scale;
#pragma unroll
        for (int v = 0; v < VPL; ++v) out.v[v] = Logit<DT>::narrow(rest(v) + quick_exp(x(v) - base) * scale * (gradient(v) - dot));
      }
    };
    if (a.normalize) finish(std::true_type());
    else finish(std::false_type());
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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

int tokens_of_round(int64_t experts) { return kRouteThreads / (experts <= 256 ? 16 : 64); }

bool is_small(int64_t tokens, int64_t top_k) { return tokens <= kSmallTokens && tokens * top_k <= kSmallSlots; }

// Tokens of a workgroup: at least a round, and no more than kRouteBlocks workgroups.
int64_t tokens_of_block(int64_t tokens, int64_t experts) {
  const int64_t round = tokens_of_round(experts), each = (tokens + kRouteBlocks - 1) / kRouteBlocks;
  return each < round ? round : (each + round - 1) / round * round;
}

int64_t route_blocks(int64_t tokens, int64_t experts) {
  const int64_t chunk = tokens_of_block(tokens, experts);
  return (tokens + chunk - 1) / chunk;
}

template <int DT, int G, int VPL>
hipError_t launch_route(const RouteArgs& a, hipStream_t stream) {
  const size_t row = (size_t)a.experts * sizeof(int32_t), waves = kRouteWaves * row;
  if (is_small(a.tokens, a.top_k)) {
    hipLaunchKernelGGL((route_small_kernel<DT, G, VPL>), dim3(1), dim3(kRouteThreads), 2 * row + kSmallSlots * sizeof(int32_t) + waves,
                       stream, a);
    return hipGetLastError();
  }
  RouteParams p;
  p.a = a;
  p.chunk = (int32_t)tokens_of_block(a.tokens, a.experts);
  p.blocks = (int32_t)route_blocks(a.tokens, a.experts);
  p.counts = static_cast<int32_t*>(a.scratch);
  p.mass_parts = reinterpret_cast<float*>(p.counts + (int64_t)a.experts * p.blocks);
  hipLaunchKernelGGL((route_choose_kernel<DT, G, VPL>), dim3(p.blocks), dim3(kRouteThreads), row + (a.mass != nullptr ? waves : 0), stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(route_scan_kernel, dim3((a.experts + 3) / 4), dim3(256), 0, stream, p);
  err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(route_place_kernel, dim3(p.blocks), dim3(kRouteThreads), row + waves, stream, p);
  return hipGetLastError();
}

template <int DT, int G, int VPL>
hipError_t launch_backward(const RouteBackwardArgs& a, hipStream_t stream) {
  constexpr int64_t GROUPS = kBackThreads / G;
  const int64_t blocks = (a.tokens + GROUPS - 1) / GROUPS;
  hipLaunchKernelGGL((route_backward_kernel<DT, G, VPL>), dim3((uint32_t)(blocks < kBackBlocks ? blocks : kBackBlocks)), dim3(kBackThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

uint64_t route_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k) {
  return is_small(tokens, top_k) ? 0 : (uint64_t)(2 * experts * route_blocks(tokens, experts)) * sizeof(int32_t);
}

// Lanes of a token and columns of a lane by the number of experts: as few lanes as hold the token, since each round of the choice costs an
// exchange over them.  16 and 64 lanes, us: choosing for 65536 tokens of 256 experts 37, 79, their gradient 35, 62; 8192 of 128 6.4, 10.6 and
// 6.9, 8.4; 8192 of 64 5.2, 8.8 and 4.6, 5.2.
#define GG_BY_EXPERTS(DT, launch, a, stream)                          \
  do {                                                                \
    if ((a).experts <= 64) return launch<DT, 16, 4>(a, stream);       \
    if ((a).experts <= 128) return launch<DT, 16, 8>(a, stream);      \
    if ((a).experts <= 256) return launch<DT, 16, 16>(a, stream);     \
    if ((a).experts <= 512) return launch<DT, 64, 8>(a, stream);      \
    return launch<DT, 64, 16>(a, stream);                             \
  } while (0)

hipError_t route(const RouteArgs& a, hipStream_t stream) {
  if (a.dt == kF32) GG_BY_EXPERTS(kF32, launch_route, a, stream);
  if (a.dt == kBF16) GG_BY_EXPERTS(kBF16, launch_route, a, stream);
  GG_BY_EXPERTS(kF16, launch_route, a, stream);
}

hipError_t route_backward(const RouteBackwardArgs& a, hipStream_t stream) {
  if (a.dt == kF32) GG_BY_EXPERTS(kF32, launch_backward, a, stream);
  if (a.dt == kBF16) GG_BY_EXPERTS(kBF16, launch_backward, a, stream);
  GG_BY_EXPERTS(kF16, launch_backward, a, stream);
}

}  // namespace gg
