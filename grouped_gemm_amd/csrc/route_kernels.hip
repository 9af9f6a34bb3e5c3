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
#include "operators.hpp"

#include <math.h>

#include "gmm_kernel.hpp"
#include "wave_ops.hpp"

namespace gg {
namespace {

constexpr int kRouteThreads = 512;
constexpr int kRouteWaves = kRouteThreads / 64;
// Workgroups that choose and place: two on each of 256 compute units; a column of their counts is 8 words for each lane
// of the wave that sums it.
constexpr int kRouteBlocks = 512;
// Up to this many tokens and chosen rows one workgroup does everything in one launch.
constexpr int kSmallTokens = 64, kSmallSlots = 2048;

template <int DT>
struct Logit;
template <>
struct Logit<kF32> {
  using T = uint32_t;
  static __device__ __forceinline__ float widen(T v) { return __builtin_bit_cast(float, v); }
  static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(uint32_t, v); }
};
template <>
struct Logit<kBF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float widen(T v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
  static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct Logit<kF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float widen(T v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// VPL neighbouring elements on any boundary (rows of any length): CDNA takes wide accesses on any boundary of an element.
template <typename T, int VPL>
struct __attribute__((packed, aligned(sizeof(T)))) Row {
  T v[VPL];
};

// Whole numbers ordered as the floats are: -0 equal to +0, NaN above all, 0 below all.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.0f);
  const uint32_t key = bits ^ ((bits & 0x80000000u) ? 0xffffffffu : 0x80000000u);
  return x != x ? 0xffffffffu : key;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __builtin_bit_cast(float, key ^ ((key & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// ... and of the 16 bits of a two-byte type.
template <int DT>
__device__ __forceinline__ uint32_t short_key(float x) {
  const uint32_t bits = Logit<DT>::narrow(x + 0.0f);   // (exact)
  const uint32_t key = (bits ^ ((bits & 0x8000u) ? 0xffffu : 0x8000u)) & 0xffffu;
  return x != x ? 0xffffu : key;
}
template <int DT>
__device__ __forceinline__ float short_key_value(uint32_t key) {
  if constexpr (DT == kF32) return 0.0f;
  return Logit<DT>::widen((typename Logit<DT>::T)(key ^ ((key & 0x8000u) ? 0x8000u : 0xffffu)));
}

// The exponential by the hardware's power of two, off by 2^-24 |x| and a unit in the last place: for the scores of all experts, whose
// sums and gradients that does not show in.  The chosen weights are computed with the full functions.
__device__ __forceinline__ float quick_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float quick_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + quick_exp(-x)); }
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.0f) - log1pf(expf(-fabsf(x))); }

struct RouteParams {
  RouteArgs a;
  int32_t chunk;           // tokens of a workgroup
  int32_t blocks;
  int32_t* counts;         // [experts][blocks] chosen rows of each workgroup; then those of the workgroups before it
  float* mass_parts;       // [experts][blocks]
};

// The VPL logits of one lane, columns l * VPL .. of its token; columns past the last read as -inf.
template <int DT, int VPL>
__device__ __forceinline__ void load_logits(const void* logits, int64_t token, int experts, int column, float* x) {
  using T = typename Logit<DT>::T;
  const T* from = static_cast<const T*>(logits) + token * experts + column;
  if (column + VPL <= experts) {
    const Row<T, VPL> r = *reinterpret_cast<const Row<T, VPL>*>(from);
#pragma unroll
    for (int v = 0; v < VPL; ++v) x[v] = Logit<DT>::widen(r.v[v]);
  } else {
#pragma unroll
    for (int v = 0; v < VPL; ++v) x[v] = column + v < experts ? Logit<DT>::widen(from[v]) : -INFINITY;
  }
}

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
    float x[VPL];
    load_logits<DT, VPL>(a.logits, t, a.experts, column, x);
    // Two-byte logits leave room for their column below, so that no two keys are equal.
    constexpr bool UNIQUE = DT != kF32;
    uint32_t key[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      key[v] = column + v < a.experts ? order_key(x[v]) : 0u;
      if (UNIQUE && column + v < a.experts) key[v] = (short_key<DT>(x[v]) << 16) | (uint32_t)(0xffff - (column + v));
    }
    float value[KR];
    int index[KR];
#pragma unroll
    for (int r = 0; r < KR; ++r) value[r] = 0.0f, index[r] = 0;
    float top = 0.0f;
    for (int j = 0; j < k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int v = 1; v < VPL; ++v) best = best > key[v] ? best : key[v];
      best = group_max<G>(best);
      uint32_t at = ~0u;
      float found;
      if constexpr (UNIQUE) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) key[v] = key[v] == best ? 0u : key[v];
        at = 0xffffu - (best & 0xffffu);
        found = short_key_value<DT>(best >> 16);
      } else {
#pragma unroll
        for (int v = VPL - 1; v >= 0; --v) at = key[v] == best ? (uint32_t)(column + v) : at;
        at = group_min<G>(at);
#pragma unroll
        for (int v = 0; v < VPL; ++v) key[v] = at == (uint32_t)(column + v) ? 0u : key[v];
        found = key_value(best);
      }
      if (j == 0) top = found;
#pragma unroll
      for (int r = 0; r < KR; ++r)
        if (j == l + r * G) value[r] = found, index[r] = (int)at;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float share[KR], scale = 0.0f;
    if (all_scores) {   // (the sigmoid's own sum is not used)
      float s[VPL], sum = 0.0f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        s[v] = a.sigmoid ? quick_sigmoid(x[v]) : quick_exp(x[v] - base);
        sum += s[v];
      }
      sum = group_sum<G>(sum);
      scale = a.sigmoid ? 1.0f : (sum == 0.0f ? 0.0f : 1.0f / sum);
#pragma unroll
      for (int v = 0; v < VPL; ++v) mass[v] += s[v] * scale;
    }
    if (a.normalize) {
      // (of sigmoids by their logarithms: their sum may be too small for a float)
      const float log_top = a.sigmoid ? log_sigmoid(base) : 0.0f;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        share[r] = expf(a.sigmoid ? log_sigmoid(value[r]) - log_top : value[r] - base);
        if (l + r * G >= k) share[r] = 0.0f;
        sum += share[r];
      }
      sum = group_sum<G>(sum);
#pragma unroll
      for (int r = 0; r < KR; ++r) share[r] = sum == 0.0f ? 0.0f : share[r] / sum;
    } else {
#pragma unroll
      for (int r = 0; r < KR; ++r) share[r] = a.sigmoid ? sigmoid(value[r]) : expf(value[r] - base) * scale;
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

// Exclusive prefix sums of the experts' counts, in LDS, by the first wave; ends with a barrier.
template <typename Count>
__device__ __forceinline__ void expert_starts(int experts, int32_t* starts, Count count) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
      const int mine = e0 + lane < experts ? count(e0 + lane) : 0;
      const int upto = wave_prefix(mine);
      if (e0 + lane < experts) starts[e0 + lane] = before + upto - mine;
      before += __shfl(upto, 63);
    }
  }
  __syncthreads();
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
  expert_starts(a.experts, starts, [&](int e) { return (int)a.batch_sizes[e]; });
  const int64_t first = (int64_t)blockIdx.x * p.chunk, last = first + p.chunk < a.tokens ? first + p.chunk : a.tokens;
  const int32_t* chosen = a.chosen + first * a.top_k;
  place((int)(last - first) * a.top_k, a.experts, a.top_k, first * a.top_k, next, [&](int i) { return chosen[i]; },
        [&](int e) { return starts[e] + p.counts[(int64_t)e * p.blocks + blockIdx.x]; }, a.row_index, a.order);
}

// Gradient of the logits, one pass: with g the gradients of the chosen weights and m those of the mass,
//   softmax  s (u - <u, s>), u = m, and g at the chosen where the weights are the scores themselves;
//   sigmoid  s (1 - s) u;
//   normalized weights q = w add q_j (g_j - <g, q>) at the chosen (times 1 - s_j with the sigmoid).
// What falls on the chosen columns goes to their lanes through LDS, one row of it for each group.
constexpr int kBackThreads = 256;

template <int DT, int G, int VPL>
__global__ __launch_bounds__(kBackThreads) void route_backward_kernel(RouteBackwardArgs a) {
  using T = typename Logit<DT>::T;
  constexpr int KR = G == 16 ? 2 : 1, GROUPS = kBackThreads / G, WIDTH = G * VPL;
  __shared__ __attribute__((aligned(16))) float rows[GROUPS * WIDTH];
  const int group = threadIdx.x / G, l = threadIdx.x % G, column = l * VPL, k = a.top_k;
  float* row = rows + group * WIDTH;
  float m[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) m[v] = a.mass_grad != nullptr && column + v < a.experts ? a.mass_grad[column + v] : 0.0f;
  const bool dense = a.mass_grad != nullptr || !a.normalize;
  for (int64_t t = (int64_t)blockIdx.x * GROUPS + group; t < a.tokens; t += (int64_t)gridDim.x * GROUPS) {
    float x[VPL];
    load_logits<DT, VPL>(a.logits, t, a.experts, column, x);
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) top = fmaxf(top, x[v]);
    top = group_reduce<G>(top, [](float p, float q) { return fmaxf(p, q); });
    const float base = top == -INFINITY ? 0.0f : top;
    // what falls on the chosen columns
    float value[KR], grad[KR];
    int index[KR];
#pragma unroll
    for (int r = 0; r < KR; ++r) {
      const int j = l + r * G;
      index[r] = j < k ? a.chosen[t * k + j] : -1;
      if ((uint32_t)index[r] >= (uint32_t)a.experts) index[r] = -1;   // (names no expert: no gradient)
      grad[r] = index[r] >= 0 && a.weights_grad != nullptr ? a.weights_grad[t * k + j] : 0.0f;
      value[r] = index[r] >= 0 ? Logit<DT>::widen(static_cast<const T*>(a.logits)[t * a.experts + index[r]]) : -INFINITY;
    }
    if (a.normalize) {
      const float log_top = a.sigmoid ? log_sigmoid(base) : 0.0f;
      float q[KR], sum = 0.0f, dot = 0.0f;
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        q[r] = index[r] >= 0 ? expf(a.sigmoid ? log_sigmoid(value[r]) - log_top : value[r] - base) : 0.0f;
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
      for (int r = 0; r < KR; ++r) grad[r] = q[r] * (grad[r] - dot) * (a.sigmoid ? sigmoid(-value[r]) : 1.0f);
    }
    // (a row belongs to one wave, whose LDS accesses stay in order)
#pragma unroll
    for (int v = 0; v < VPL; ++v) row[column + v] = 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < KR; ++r)
      if (index[r] >= 0) row[index[r]] = grad[r];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float at[VPL], out[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) at[v] = row[column + v];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int v = 0; v < VPL; ++v) out[v] = a.normalize ? at[v] : 0.0f;
    if (dense) {
      float s[VPL], sum = 0.0f, dot = 0.0f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        at[v] = m[v] + (a.normalize ? 0.0f : at[v]);
        s[v] = a.sigmoid ? quick_sigmoid(x[v]) : quick_exp(x[v] - base);
        sum += s[v];
        dot += s[v] * at[v];
      }
      if (!a.sigmoid) {
        sum = group_sum<G>(sum);
        dot = group_sum<G>(dot);
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        dot *= scale;
#pragma unroll
        for (int v = 0; v < VPL; ++v) out[v] += s[v] * scale * (at[v] - dot);
      } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) out[v] += s[v] * quick_sigmoid(-x[v]) * at[v];   // (1 - s would lose all of a small difference)
      }
    }
    T* to = static_cast<T*>(a.logits_grad) + t * a.experts + column;
    if (column + VPL <= a.experts) {
      Row<T, VPL> r;
#pragma unroll
      for (int v = 0; v < VPL; ++v) r.v[v] = Logit<DT>::narrow(out[v]);
      *reinterpret_cast<Row<T, VPL>*>(to) = r;
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        if (column + v < a.experts) to[v] = Logit<DT>::narrow(out[v]);
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
  hipLaunchKernelGGL((route_backward_kernel<DT, G, VPL>), dim3((uint32_t)(blocks < 2048 ? blocks : 2048)), dim3(kBackThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

uint64_t route_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k) {
  return is_small(tokens, top_k) ? 0 : (uint64_t)(2 * experts * route_blocks(tokens, experts)) * sizeof(int32_t);
}

// Lanes of a token and columns of a lane by the number of experts.
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
