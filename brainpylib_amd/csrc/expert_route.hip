// Routing of tokens to experts: the choice of the experts (expert_topk), the sort of the chosen pairs by expert
// (expert_sort), and the rows' way to the experts (expert_dispatch) and back (expert_combine), with their gradients.
// A mixture's routing is a sparse tokens x experts matrix with k nonzeros a row; expert_sort turns it into index arrays
// by expert as coo_to_csr does by row, and the two ways are products of it with dense rows.
#include <type_traits>

#include "expert.h"

namespace {

using namespace bpl;

constexpr uint32_t kNone = 0xffffffffu;  // -1 in the index arrays

// ---- all-reductions within aligned groups of G lanes: DPP within rows of 16, then exchanges across rows -------------
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
template <int G, typename OP>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, OP op) {
  v = op(v, dpp<0xB1>(v));   // lane ^ 1
  v = op(v, dpp<0x4E>(v));   // lane ^ 2
  v = op(v, dpp<0x141>(v));  // mirrored in 8 (the halves hold equal values by now)
  if (G > 8) v = op(v, dpp<0x140>(v));  // mirrored in 16
  if (G > 16) v = op(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16, kWave)));
  if (G > 32) v = op(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32, kWave)));
  return v;
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int G>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
  return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
template <int G>
__device__ __forceinline__ float group_add(float v) {
  return __uint_as_float(group_reduce<G>(
      __float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// ---- expert_topk ----------------------------------------------------------------------------------------------------
// k turns of: the largest key of a lane's 8 logits, of the row's lanes, the lowest place that holds it, that place's key to 0.
// A row to as few lanes as hold it, so that a wave takes 1 to 8 rows at once and most exchanges are DPP moves.  Bound by
// instructions, 50 a turn and wave: 32,771 rows of 128 float logits, k = 8, 11.4 us (1.5 TB/s), its gradient 10.6 us.
// Keys whose order as whole numbers is that of the logits: NaN above every number, -0 equal to 0, and 0 for -inf (and
// for what is beyond the row or taken already), which is never chosen.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t key = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x != x ? 0xffffffffu : key == 0x007fffffu ? 0u : key;
}
__device__ __forceinline__ float of_key(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// V consecutive logits of a row to a lane, G lanes to a row.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T *__restrict__ row, uint32_t first, uint32_t experts, float (&x)[V]) {
  constexpr int kPer = static_cast<int>(Piece<T>::kElems);
  static_assert(V % kPer == 0, "whole pieces");
  if (first + V <= experts) {
#pragma unroll
    for (int j = 0; j < V; j += kPer) {
      const typename Piece<T>::type v = *reinterpret_cast<const typename Piece<T>::type *>(row + first + j);
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[j + i] = static_cast<float>(v[i]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = first + j < experts ? static_cast<float>(row[first + j]) : -__builtin_inff();
  }
}

template <typename T, int V, int G>
__global__ __launch_bounds__(256) void topk_kernel(const T *__restrict__ logits, const uint8_t *__restrict__ mask,
                                                   float *__restrict__ weights, uint32_t *__restrict__ chosen,
                                                   uint32_t tokens, uint32_t experts, uint32_t k, bool normalize) {
  constexpr uint32_t kRows = 256 / G;
  const uint32_t lane = threadIdx.x % G;
  for (uint32_t t0 = blockIdx.x * kRows; t0 < tokens; t0 += gridDim.x * kRows) {
    const uint32_t t = t0 + threadIdx.x / G;
    const bool live = t < tokens && (mask == nullptr || mask[t] != 0);
    float x[V];
    uint32_t key[V];
    if (live) {
      load_logits<T, V>(logits + static_cast<size_t>(t) * experts, lane * V, experts, x);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = -__builtin_inff();
    }
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = key_of(x[j]);
    uint32_t most = 0, my_key = 0, my_expert = kNone;
    for (uint32_t r = 0; r < k; ++r) {
      uint32_t best = key[0];
#pragma unroll
      for (int j = 1; j < V; ++j) best = key[j] > best ? key[j] : best;
      best = group_max<G>(best);
      uint32_t at = kNone;
#pragma unroll
      for (int j = V - 1; j >= 0; --j) at = key[j] == best ? lane * V + j : at;
      at = group_min<G>(at);
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = at == lane * V + j ? 0u : key[j];
      if (r == 0) most = best;
      if (lane == r) {
        my_key = best;
        my_expert = best != 0 ? at : kNone;
      }
    }
    const float top = of_key(most);
    const bool mine = my_key != 0;
    const float e = mine ? expf(of_key(my_key) - top) : 0.f;
    float total;
    if (normalize) {
      total = group_add<G>(e);
    } else {
      total = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) total += expf(x[j] - top);
      total = group_add<G>(total);
    }
    if (t < tokens && lane < k) {
      weights[static_cast<size_t>(t) * k + lane] = mine ? e / total : 0.f;
      chosen[static_cast<size_t>(t) * k + lane] = my_expert;
    }
  }
}

// Normalized: d_e = w_e (g_e - sum w g) at the chosen, 0 elsewhere, without the logits.  Else, with p the softmax over all
// experts: d_e = p_e ([e chosen] g_e - sum w g).
template <typename T, int V, int G>
__global__ __launch_bounds__(256) void topk_gradient_kernel(const T *__restrict__ logits, const uint32_t *__restrict__ chosen,
                                                            const float *__restrict__ weights, const float *__restrict__ ct,
                                                            T *__restrict__ grad, uint32_t tokens, uint32_t experts,
                                                            uint32_t k, bool normalize) {
  constexpr uint32_t kRows = 256 / G;
  constexpr int kPer = static_cast<int>(Piece<T>::kElems);
  const uint32_t lane = threadIdx.x % G;
  const int group = static_cast<int>(threadIdx.x % kWave) / G * G;
  for (uint32_t t0 = blockIdx.x * kRows; t0 < tokens; t0 += gridDim.x * kRows) {
    const uint32_t t = t0 + threadIdx.x / G;
    uint32_t expert = kNone;
    float w = 0.f, g = 0.f;
    if (t < tokens && lane < k) {
      const size_t p = static_cast<size_t>(t) * k + lane;
      expert = chosen[p];
      if (expert < experts) {  // (a place without an expert has no gradient, whatever stands in the cotangent there)
        w = weights[p];
        g = ct[p];
      }
    }
    const float inner = group_add<G>(w * g);
    const bool any = __shfl(static_cast<int>(expert), group, kWave) != -1;
    const float own = normalize ? w * (g - inner) : w * g;
    float d[V];
    if (normalize || !any) {
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = 0.f;
    } else {
      float x[V];
      load_logits<T, V>(logits + static_cast<size_t>(t) * experts, lane * V, experts, x);
      float top = x[0];
      uint32_t best = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const uint32_t key = key_of(x[j]);
        best = key > best ? key : best;
      }
      top = of_key(group_max<G>(best));
      float total = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = expf(x[j] - top);
        total += d[j];
      }
      const float scale = -inner / group_add<G>(total);
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] *= scale;
    }
    for (uint32_t r = 0; r < k; ++r) {
      const uint32_t e = static_cast<uint32_t>(__shfl(static_cast<int>(expert), group + static_cast<int>(r), kWave));
      const float v = __shfl(own, group + static_cast<int>(r), kWave);
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] += e == lane * V + j ? v : 0.f;
    }
    if (t < tokens) {
      T *const row = grad + static_cast<size_t>(t) * experts;
#pragma unroll
      for (int j = 0; j < V; j += kPer) {
        typename Piece<T>::type v;
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = static_cast<T>(d[j + i]);
        if (lane * V + j < experts) store_piece<T>(row, lane * V + j, experts, v);
      }
    }
  }
}

// f(lanes to a row, logits to a lane): 8 logits to a lane and as few lanes as hold the row and its k places.
template <typename FN>
void by_row_shape(uint32_t experts, uint32_t k, FN f) {
  if (experts <= 64 && k <= 8)
    f(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  else if (experts <= 128 && k <= 16)
    f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
  else if (experts <= 256 && k <= 32)
    f(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
  else if (experts <= 512)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
  else
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

unsigned capped(uint64_t blocks, uint64_t most = 1u << 20) { return static_cast<unsigned>(blocks < most ? blocks : most); }

bool topk_limits(const char *target, const bpl_expert_descriptor &d) {
  if (!expert_limits(target, d)) return false;
  if (d.per_token < 1 || d.per_token > d.experts) {
    set_error("%s: 1 to %u experts a token, got %u", target, d.experts, d.per_token);
    return false;
  }
  return true;
}

template <typename T>
void topk(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !topk_limits(target, d) || d.tokens == 0) return;
  const auto *mask = d.flags & BPL_EXPERT_MASKED ? static_cast<const uint8_t *>(buffers[1]) : nullptr;
  by_row_shape(d.experts, d.per_token, [&](auto lanes, auto values) {
    constexpr int G = decltype(lanes)::value, V = decltype(values)::value;
    hipLaunchKernelGGL((topk_kernel<T, V, G>), dim3(capped(div_up(d.tokens, 256 / G))), dim3(256), 0, stream,
                       static_cast<const T *>(buffers[0]), mask, static_cast<float *>(buffers[2]),
                       static_cast<uint32_t *>(buffers[3]), d.tokens, d.experts, d.per_token,
                       (d.flags & BPL_EXPERT_NORMALIZE) != 0);
  });
  check_launch(target);
}

template <typename T>
void topk_gradient(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !topk_limits(target, d) || d.tokens == 0) return;
  by_row_shape(d.experts, d.per_token, [&](auto lanes, auto values) {
    constexpr int G = decltype(lanes)::value, V = decltype(values)::value;
    hipLaunchKernelGGL((topk_gradient_kernel<T, V, G>), dim3(capped(div_up(d.tokens, 256 / G))), dim3(256), 0, stream,
                       static_cast<const T *>(buffers[0]), static_cast<const uint32_t *>(buffers[1]),
                       static_cast<const float *>(buffers[2]), static_cast<const float *>(buffers[3]),
                       static_cast<T *>(buffers[4]), d.tokens, d.experts, d.per_token,
                       (d.flags & BPL_EXPERT_NORMALIZE) != 0);
  });
  check_launch(target);
}

// ---- expert_sort ----------------------------------------------------------------------------------------------------
// A stable counting sort.  Workgroup b takes a range of the pairs, its waves consecutive parts of it: counts of every
// (workgroup, expert) by one launch (none where one workgroup takes all), then every workgroup adds up the counts before
// its own, scans the experts and ranks its pairs 64 at a time, in their order.  What is dropped counts as one more
// expert behind the last.  No atomics but in counts, so the result never depends on an order.
// Bound by the chain of its steps, not by bytes: 524,296 pairs over 256 experts 14.1 us, in two
// launches of 3.1 and 11.8 (14.8 with eight rows of counts and no next steps under way).
constexpr uint32_t kSortThreads = 512, kSortWaves = kSortThreads / kWave;
constexpr uint32_t kSortPairs = 2048;  // to a workgroup, at least
constexpr uint32_t kSortOne = 8192;    // so many pairs one workgroup takes alone
constexpr uint32_t kSortMostGroups = 256;
constexpr uint32_t kSortRows = 20;      // rows of counts that a thread requests together
constexpr uint32_t kSortAtOnce = 4;    // steps of 64 pairs whose experts a wave requests together

struct SortShape {
  uint32_t groups, pairs;  // workgroups, pairs to each (a multiple of kSortThreads)
};
SortShape sort_shape(uint32_t pairs) {
  SortShape s;
  s.groups = pairs <= kSortOne ? 1u : div_up(pairs, kSortPairs);
  if (s.groups > kSortMostGroups) s.groups = kSortMostGroups;
  s.pairs = (div_up(pairs, s.groups) + kSortThreads - 1) / kSortThreads * kSortThreads;
  if (s.pairs == 0) s.pairs = kSortThreads;
  s.groups = pairs == 0 ? 1u : div_up(pairs, s.pairs);
  return s;
}
// A workgroup's row of counts: one for each expert and one for what is dropped, in whole quads.
__host__ __device__ inline uint32_t sort_bins(uint32_t experts) { return (experts + 4u) / 4u * 4u; }

// The experts of a wave's pairs from `first + i0` on, kSortAtOnce steps of 64.
struct SortSteps {
  uint32_t e[kSortAtOnce];
};
__device__ __forceinline__ SortSteps sort_load(const uint32_t *__restrict__ chosen, uint64_t first, uint32_t i0, uint32_t part,
                                               uint32_t pairs) {
  SortSteps s;
#pragma unroll
  for (uint32_t j = 0; j < kSortAtOnce; ++j) {
    const uint32_t i = i0 + j * kWave;
    const uint64_t p = first + i + threadIdx.x % kWave;
    s.e[j] = i < part && p < pairs ? chosen[p] : 0u;
  }
  return s;
}
// f(pair, expert, whether there is a pair) for a wave's pairs from `first` on, 64 a step; `now`: the first steps' experts.  The
// next ones are requested before these are worked on.
template <typename FN>
__device__ __forceinline__ void sort_steps(const uint32_t *__restrict__ chosen, uint64_t first, uint32_t part, uint32_t pairs,
                                           uint32_t experts, SortSteps now, FN f) {
  for (uint32_t i0 = 0; i0 < part; i0 += kSortAtOnce * kWave) {
    const SortSteps next = sort_load(chosen, first, i0 + kSortAtOnce * kWave, part, pairs);
#pragma unroll
    for (uint32_t j = 0; j < kSortAtOnce; ++j) {
      const uint64_t p = first + i0 + j * kWave + threadIdx.x % kWave;
      if (i0 + j * kWave < part) f(p, now.e[j] < experts ? now.e[j] : experts, p < pairs);
    }
    now = next;
  }
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const uint32_t *__restrict__ chosen, uint32_t *__restrict__ counts,
                                                                  uint32_t pairs, uint32_t experts, uint32_t share) {
  __shared__ uint32_t count[kMostExperts + 4];
  const uint32_t bins = sort_bins(experts);
  const uint32_t part = share / kSortWaves;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * share + threadIdx.x / kWave * part;
  const SortSteps ahead = sort_load(chosen, first, 0, part, pairs);
  for (uint32_t e = threadIdx.x; e < bins; e += kSortThreads) count[e] = 0;
  __syncthreads();
  sort_steps(chosen, first, part, pairs, experts, ahead, [&](uint64_t, uint32_t e, bool there) {
    if (there) atomicAdd(&count[e], 1u);
  });
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < bins; e += kSortThreads) counts[static_cast<size_t>(blockIdx.x) * bins + e] = count[e];
}

__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const uint32_t *__restrict__ chosen, const uint32_t *__restrict__ counts,
                                                                  uint32_t *__restrict__ indptr, uint32_t *__restrict__ order,
                                                                  uint32_t *__restrict__ position, uint32_t pairs,
                                                                  uint32_t experts, uint32_t share, uint32_t groups) {
  // next[wave][expert]: first the wave's counts, then the place of its next pair of that expert
  extern __shared__ uint32_t lds[];
  uint32_t *const next = lds;
  const uint32_t bins = sort_bins(experts);
  uint32_t *const total = next + kSortWaves * bins, *const before = total + bins;
  __shared__ uint32_t wave_total[kSortWaves];
  const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  uint32_t *const mine = next + wave * bins;
  const uint32_t part = share / kSortWaves;  // (a multiple of 64)
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * share + wave * part;
  const SortSteps ahead = sort_load(chosen, first, 0, part, pairs);
  for (uint32_t i = threadIdx.x; i < (kSortWaves + 2) * bins; i += kSortThreads) next[i] = 0;
  __syncthreads();
  if (groups != 1) {
    // four experts to a lane, lanes side by side; sets of them share the workgroups' counts
    const uint32_t quads = bins / 4, sets = kSortThreads / quads, set = threadIdx.x / quads, quad = threadIdx.x % quads;
    if (set < sets) {
      uint4 all = make_uint4(0, 0, 0, 0), below = all;
      const uint4 *const from = reinterpret_cast<const uint4 *>(counts) + quad;
      // (a share to a set, kSortRows rows of it requested together: what is beyond is not read one by one)
      const uint32_t rows = (groups + sets - 1) / sets, b0 = set * rows, b1 = b0 + rows < groups ? b0 + rows : groups;
      for (uint32_t b = b0; b < b1; b += kSortRows) {
        uint4 c[kSortRows];
#pragma unroll
        for (uint32_t j = 0; j < kSortRows; ++j)
          c[j] = b + j < b1 ? from[static_cast<size_t>(b + j) * quads] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t j = 0; j < kSortRows; ++j) {
          const uint32_t mask = b + j < blockIdx.x ? 0xffffffffu : 0u;
          all.x += c[j].x, all.y += c[j].y, all.z += c[j].z, all.w += c[j].w;
          below.x += c[j].x & mask, below.y += c[j].y & mask, below.z += c[j].z & mask, below.w += c[j].w & mask;
        }
      }
      atomicAdd(&total[4 * quad], all.x), atomicAdd(&total[4 * quad + 1], all.y);
      atomicAdd(&total[4 * quad + 2], all.z), atomicAdd(&total[4 * quad + 3], all.w);
      atomicAdd(&before[4 * quad], below.x), atomicAdd(&before[4 * quad + 1], below.y);
      atomicAdd(&before[4 * quad + 2], below.z), atomicAdd(&before[4 * quad + 3], below.w);
    }
  }
  sort_steps(chosen, first, part, pairs, experts, ahead, [&](uint64_t, uint32_t e, bool there) {
    if (there) atomicAdd(&mine[e], 1u);
  });
  __syncthreads();
  if (groups == 1) {
    for (uint32_t e = threadIdx.x; e < bins; e += kSortThreads) {
      uint32_t sum = 0;
#pragma unroll
      for (uint32_t w = 0; w < kSortWaves; ++w) sum += next[w * bins + e];
      total[e] = sum;
    }
    __syncthreads();
  }
  // exclusive scan of the totals, consecutive experts to a thread
  constexpr uint32_t kPer = (kMostExperts + 4 + kSortThreads - 1) / kSortThreads;
  uint32_t own[kPer], sum = 0;
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    const uint32_t e = threadIdx.x * kPer + j;
    own[j] = e < bins ? total[e] : 0u;
    sum += own[j];
  }
  const uint32_t upto = wave_inclusive_scan_u32(sum);
  if (lane == kWave - 1) wave_total[wave] = upto;
  __syncthreads();
  uint32_t start = upto - sum;
#pragma unroll
  for (uint32_t w = 0; w < kSortWaves; ++w) start += w < wave ? wave_total[w] : 0u;
#pragma unroll
  for (uint32_t j = 0; j < kPer; ++j) {
    const uint32_t e = threadIdx.x * kPer + j;
    if (e < bins) before[e] += start;
    if (e <= experts && blockIdx.x == 0) indptr[e] = start;
    start += own[j];
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < bins; e += kSortThreads) {
    uint32_t c[kSortWaves], at = before[e];
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) c[w] = next[w * bins + e];
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) {
      next[w * bins + e] = at;
      at += c[w];
    }
  }
  __syncthreads();
  const uint32_t bits = 32u - __builtin_clz(experts);
  volatile uint32_t *const places = mine;
  sort_steps(chosen, first, part, pairs, experts, ahead, [&](uint64_t p, uint32_t e, bool there) {
    uint64_t same = __ballot(there);
    for (uint32_t b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1u);
      same &= (e >> b) & 1u ? set : ~set;
    }
    if (there) {
      const uint32_t rank = __popcll(same & ((1ull << lane) - 1ull));
      const uint32_t at = places[e] + rank;
      // (a wave's LDS instructions are carried out in order: all lanes have read before the first of a kind adds)
      __builtin_amdgcn_wave_barrier();
      if (rank == 0) places[e] = at + static_cast<uint32_t>(__popcll(same));
      __builtin_amdgcn_wave_barrier();
      const bool dropped = e == experts;
      order[at] = dropped ? kNone : static_cast<uint32_t>(p);
      position[p] = dropped ? kNone : at;
    }
  });
}

void sort(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  const uint32_t pairs = d.tokens * d.per_token;
  const SortShape s = sort_shape(pairs);
  const auto *chosen = static_cast<const uint32_t *>(buffers[0]);
  auto *counts = static_cast<uint32_t *>(buffers[4]);
  if (s.groups > 1) {
    hipLaunchKernelGGL(sort_count_kernel, dim3(s.groups), dim3(kSortThreads), 0, stream, chosen, counts, pairs, d.experts,
                       s.pairs);
    if (!check_launch(target)) return;
  }
  hipLaunchKernelGGL(sort_place_kernel, dim3(s.groups), dim3(kSortThreads), (kSortWaves + 2) * sort_bins(d.experts) * 4, stream,
                     chosen, counts, static_cast<uint32_t *>(buffers[1]), static_cast<uint32_t *>(buffers[2]),
                     static_cast<uint32_t *>(buffers[3]), pairs, d.experts, s.pairs, s.groups);
  check_launch(target);
}

// The value of lane i, the same for all lanes.
__device__ __forceinline__ uint32_t lane_value(uint32_t v, uint32_t i) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(i)));
}
__device__ __forceinline__ float lane_value(float v, uint32_t i) { return __uint_as_float(lane_value(__float_as_uint(v), i)); }

// ---- the rows' two ways ---------------------------------------------------------------------------------------------
// Bound by memory.  A wave takes a piece of 64 * 16 bytes of a token's row, reads it once and writes it k times (or the other
// way round): 16,385 tokens of 2,048 bfloat16 to 8 experts each 104 us, 5.8 TB/s.  Its lanes read the token's positions side
// by side and look up what the rows there say (a pair counts only where order and position answer each other, so that no
// arrays, however made, lead two tokens to one row or beyond the arrays).
struct Pair {
  uint32_t row;  // kNone: no row
  bool answered;
};
__device__ __forceinline__ Pair pair_of(const uint32_t *__restrict__ order, const uint32_t *__restrict__ position, uint32_t t,
                                        uint32_t i, uint32_t k, uint32_t pairs) {
  Pair r{kNone, false};
  if (i < k) {
    const uint32_t p = t * k + i, at = position[p];
    if (at < pairs) {
      r.row = at;
      r.answered = order[at] == p;
    }
  }
  return r;
}

// Rows that no pair leads to are zero: the lanes of a wave look at a row each of the eight that it takes.
constexpr uint32_t kZeroRows = 8;
template <typename T, bool WHOLE>
__device__ __forceinline__ void zero_rows(const uint32_t *__restrict__ order, const uint32_t *__restrict__ position,
                                          T *__restrict__ rows, uint32_t pairs, uint32_t width, uint32_t unit) {
  const uint32_t lane = threadIdx.x % kWave;
  const uint64_t row = static_cast<uint64_t>(unit) * kZeroRows + lane;
  bool empty = false;
  if (lane < kZeroRows && row < pairs) {
    const uint32_t p = order[row];
    empty = p >= pairs || position[p] != row;
  }
  uint64_t left = __ballot(empty);
  typename Piece<T>::type zero;
#pragma unroll
  for (uint32_t j = 0; j < Piece<T>::kElems; ++j) zero[j] = static_cast<T>(0.f);
  while (left != 0) {
    const uint32_t j = __builtin_ctzll(left);
    left &= left - 1;
    T *const to = rows + (static_cast<size_t>(unit) * kZeroRows + j) * width;
    for (uint32_t col = lane * Piece<T>::kElems; col < width; col += kWave * Piece<T>::kElems) store_piece<T, WHOLE>(to, col, width, zero);
  }
}

template <typename T, bool WHOLE, bool PAST>
__global__ __launch_bounds__(256) void dispatch_kernel(const T *__restrict__ tokens, const uint32_t *__restrict__ order,
                                                       const uint32_t *__restrict__ position, T *__restrict__ rows,
                                                       uint32_t n, uint32_t k, uint32_t width, uint32_t chunks,
                                                       uint64_t units, uint32_t zero_units) {
  const uint32_t lane = threadIdx.x % kWave, pairs = n * k;
  const uint64_t waves = static_cast<uint64_t>(gridDim.x) * (256 / kWave);
  for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * (256 / kWave) + threadIdx.x / kWave; u < units + zero_units; u += waves) {
    if (u >= units) {
      zero_rows<T, WHOLE>(order, position, rows, pairs, width, static_cast<uint32_t>(u - units));
      continue;
    }
    const uint32_t t = static_cast<uint32_t>(u / chunks), chunk = static_cast<uint32_t>(u % chunks);
    const uint32_t col = (chunk * kWave + lane) * Piece<T>::kElems;
    const Pair mine = pair_of(order, position, t, lane, k, pairs);
    typename Piece<T>::type v{};
    if (col < width) v = load_piece<T, WHOLE>(tokens + static_cast<size_t>(t) * width, col, width);
    const uint32_t row = mine.answered ? mine.row : kNone;
    for (uint32_t i = 0; i < k; ++i) {
      const uint32_t to = lane_value(row, i);
      if (to != kNone && col < width) store_piece<T, WHOLE, PAST>(rows + static_cast<size_t>(to) * width, col, width, v);
    }
  }
}

// out[t] = sum over i of [weights[t][i] *] rows[position[t][i]], in 32 bits in the order of i: the way back, and without
// weights the gradient of the way there.  Eight rows are requested before the first is added.  Bound by memory: 131,080 rows
// of 2,048 bfloat16, a twentieth dropped, 98 us, 5.9 TB/s, both ways (130 and 153 us while the rows went through the caches).
template <typename T, bool WEIGHTED>
__global__ __launch_bounds__(256) void combine_kernel(const T *__restrict__ rows, const float *__restrict__ weights,
                                                      const uint32_t *__restrict__ order, const uint32_t *__restrict__ position,
                                                      T *__restrict__ out, uint32_t n, uint32_t k, uint32_t width,
                                                      uint32_t chunks, uint64_t units) {
  constexpr uint32_t kElems = Piece<T>::kElems, kAhead = 8;
  const uint32_t lane = threadIdx.x % kWave, pairs = n * k;
  const uint64_t waves = static_cast<uint64_t>(gridDim.x) * (256 / kWave);
  for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * (256 / kWave) + threadIdx.x / kWave; u < units; u += waves) {
    const uint32_t t = static_cast<uint32_t>(u / chunks), chunk = static_cast<uint32_t>(u % chunks);
    const uint32_t col = (chunk * kWave + lane) * kElems;
    const Pair mine = pair_of(order, position, t, lane, k, pairs);
    const float w = WEIGHTED && lane < k ? weights[static_cast<size_t>(t) * k + lane] : 0.f;
    const uint64_t answered = __ballot(mine.answered);
    float sum[kElems] = {};
    for (uint32_t i0 = 0; i0 < k; i0 += kAhead) {
      typename Piece<T>::type v[kAhead];
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        if (i0 + j >= k) continue;
        const uint32_t at = lane_value(mine.row, i0 + j);
        if (at != kNone && col < width) v[j] = load_piece<T, false, true>(rows + static_cast<size_t>(at) * width, col, width);
      }
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        if (i0 + j >= k || !((answered >> (i0 + j)) & 1u)) continue;
        const float by = WEIGHTED ? lane_value(w, i0 + j) : 1.f;
#pragma unroll
        for (uint32_t c = 0; c < kElems; ++c) {
          const float x = static_cast<float>(v[j][c]);
          sum[c] = WEIGHTED ? fmaf(by, x, sum[c]) : sum[c] + x;
        }
      }
    }
    if (col < width) {
      typename Piece<T>::type r;
#pragma unroll
      for (uint32_t c = 0; c < kElems; ++c) r[c] = static_cast<T>(sum[c]);
      store_piece<T>(out + static_cast<size_t>(t) * width, col, width, r);
    }
  }
}

// d_rows[position[t][i]] = weights[t][i] * ct[t];  d_weights[t][i] = <ct[t], rows[position[t][i]]>: a workgroup to a
// token, four of its pairs at a time (eight hold 136 registers and leave three waves to a SIMD: 131,080 rows of 2,048
// bfloat16 250 us, four 232, with stores past the caches 203).
template <typename T, bool WHOLE, bool PAST>
__global__ __launch_bounds__(256) void combine_gradient_kernel(const T *__restrict__ rows, const float *__restrict__ weights,
                                                               const uint32_t *__restrict__ order,
                                                               const uint32_t *__restrict__ position, const T *__restrict__ ct,
                                                               T *__restrict__ d_rows, float *__restrict__ d_weights, uint32_t n,
                                                               uint32_t k, uint32_t width, uint32_t zero_groups) {
  constexpr uint32_t kElems = Piece<T>::kElems, kAtOnce = 4, kWaves = 256 / kWave;
  __shared__ float partial[kWaves][kAtOnce];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, pairs = n * k;
  const uint32_t workers = gridDim.x - zero_groups;
  if (blockIdx.x >= workers) {
    const uint32_t units = (pairs + kZeroRows - 1) / kZeroRows;
    for (uint32_t u = (blockIdx.x - workers) * kWaves + wave; u < units; u += zero_groups * kWaves)
      zero_rows<T, WHOLE>(order, position, d_rows, pairs, width, u);
    return;
  }
  for (uint32_t t = blockIdx.x; t < n; t += workers) {
    const Pair mine = pair_of(order, position, t, lane, k, pairs);
    const uint32_t row = mine.answered ? mine.row : kNone;
    const float w = lane < k ? weights[static_cast<size_t>(t) * k + lane] : 0.f;
    const T *const from = ct + static_cast<size_t>(t) * width;
    for (uint32_t i0 = 0; i0 < k; i0 += kAtOnce) {
      float dot[kAtOnce] = {};
      for (uint32_t base = 0; base < width; base += 256 * kElems) {
        const uint32_t col = base + threadIdx.x * kElems;
        const bool inside = col < width;  // (all lanes stay in the loop: each holds a pair that the others read)
        typename Piece<T>::type g{}, v[kAtOnce];
        if (inside) g = load_piece<T, WHOLE>(from, col, width);
        if (d_weights != nullptr) {
#pragma unroll
          for (uint32_t j = 0; j < kAtOnce; ++j) {
            v[j] = typename Piece<T>::type{};
            if (i0 + j >= k) continue;
            const uint32_t at = lane_value(row, i0 + j);
            if (at != kNone && inside) v[j] = load_piece<T, WHOLE, true>(rows + static_cast<size_t>(at) * width, col, width);
          }
        }
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
          if (i0 + j >= k) continue;
          const uint32_t at = lane_value(row, i0 + j);
          if (at == kNone) continue;
          if (d_rows != nullptr) {
            const float by = lane_value(w, i0 + j);
            typename Piece<T>::type r;
#pragma unroll
            for (uint32_t c = 0; c < kElems; ++c) r[c] = static_cast<T>(by * static_cast<float>(g[c]));
            if (inside) store_piece<T, WHOLE, PAST>(d_rows + static_cast<size_t>(at) * width, col, width, r);
          }
          if (d_weights != nullptr) {
#pragma unroll
            for (uint32_t c = 0; c < kElems; ++c) dot[j] = fmaf(static_cast<float>(g[c]), static_cast<float>(v[j][c]), dot[j]);
          }
        }
      }
      if (d_weights != nullptr) {
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
          const float sum = group_add<kWave>(dot[j]);
          if (lane == 0) partial[wave][j] = sum;
        }
        __syncthreads();
        if (threadIdx.x < kAtOnce && i0 + threadIdx.x < k) {
          float sum = 0.f;
#pragma unroll
          for (uint32_t v = 0; v < kWaves; ++v) sum += partial[v][threadIdx.x];
          d_weights[static_cast<size_t>(t) * k + i0 + threadIdx.x] = sum;
        }
        __syncthreads();
      }
    }
  }
}

// Rows of 64 MB and more are stored past the caches: 131,080 rows of 2,048 bfloat16 114 -> 104 us there, 250 -> 203 us back.
// Where lines of 128 bytes are shared by rows, which then meet in the last cache, only what that does not hold (of the gradients,
// d_rows and d_weights, past the caches and not: rows of 1,000 bfloat16, 180 MB 102 and 96 us, 400 MB 220 and 235; of 2,052 float32,
// 240 MB 120 and 103, 400 MB 201 and 212 us; d_rows alone there 73 and 54, of 516 float32, 800 MB, 267 and 386).
constexpr uint64_t kPastCaches = 64ull << 20, kPastCachesShared = 256ull << 20;

template <typename T>
uint32_t chunks_of(uint32_t width) { return div_up(width, kWave * Piece<T>::kElems); }

template <typename T>
void dispatch(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  const uint32_t pairs = d.tokens * d.per_token;
  if (pairs == 0 || d.width == 0) return;
  const uint32_t chunks = chunks_of<T>(d.width), zero_units = div_up(pairs, kZeroRows);
  const uint64_t units = static_cast<uint64_t>(d.tokens) * chunks;
  // (lines that two waves write in part must meet in the cache: rows of 1,000 elements took 37 instead of 28 us)
  const bool past = static_cast<uint64_t>(pairs) * d.width * sizeof(T) >= kPastCaches && d.width * sizeof(T) % 128 == 0 &&
                    reinterpret_cast<uintptr_t>(buffers[3]) % 128 == 0;
  const bool whole = d.width % Piece<T>::kElems == 0;
  const auto kernel = past ? &dispatch_kernel<T, true, true> : whole ? &dispatch_kernel<T, true, false> : &dispatch_kernel<T, false, false>;
  hipLaunchKernelGGL(kernel, dim3(capped((units + zero_units + 3) / 4)), dim3(256), 0, stream,
                     static_cast<const T *>(buffers[0]), static_cast<const uint32_t *>(buffers[1]),
                     static_cast<const uint32_t *>(buffers[2]), static_cast<T *>(buffers[3]), d.tokens, d.per_token,
                     d.width, chunks, units, zero_units);
  check_launch(target);
}

template <typename T, bool WEIGHTED>
void combine_rows(const char *target, hipStream_t stream, const bpl_expert_descriptor &d, const void *rows,
                  const void *weights, const void *order, const void *position, void *out) {
  if (d.tokens == 0 || d.width == 0) return;
  const uint32_t chunks = chunks_of<T>(d.width);
  const uint64_t units = static_cast<uint64_t>(d.tokens) * chunks;
  hipLaunchKernelGGL((combine_kernel<T, WEIGHTED>), dim3(capped((units + 3) / 4)), dim3(256), 0, stream,
                     static_cast<const T *>(rows), static_cast<const float *>(weights),
                     static_cast<const uint32_t *>(order), static_cast<const uint32_t *>(position),
                     static_cast<T *>(out), d.tokens, d.per_token, d.width, chunks, units);
  check_launch(target);
}

template <typename T>
void dispatch_gradient(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  combine_rows<T, false>(target, stream, d, buffers[0], nullptr, buffers[1], buffers[2], buffers[3]);
}

template <typename T>
void combine(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  combine_rows<T, true>(target, stream, d, buffers[0], buffers[1], buffers[2], buffers[3], buffers[4]);
}

template <typename T>
void combine_gradient(const char *target, hipStream_t stream, void **buffers, const char *opaque, size_t opaque_len) {
  bpl_expert_descriptor d;
  if (!unpack(target, opaque, opaque_len, &d) || !expert_limits(target, d)) return;
  const uint32_t pairs = d.tokens * d.per_token;
  T *const d_rows = d.flags & BPL_EXPERT_D_ROWS && d.width != 0 ? static_cast<T *>(buffers[5]) : nullptr;
  float *const d_weights = d.flags & BPL_EXPERT_D_WEIGHTS ? static_cast<float *>(buffers[6]) : nullptr;
  if (pairs == 0 || (d_rows == nullptr && d_weights == nullptr)) return;
  const uint32_t zero_groups = d_rows != nullptr ? capped(div_up(pairs, kZeroRows * 4)) : 0u;
  const bool whole = d.width % Piece<T>::kElems == 0;
  const bool lines = d.width * sizeof(T) % 128 == 0 && reinterpret_cast<uintptr_t>(buffers[5]) % 128 == 0;
  const bool past = static_cast<uint64_t>(pairs) * d.width * sizeof(T) >= (lines ? kPastCaches : kPastCachesShared);
  const auto kernel = !whole ? &combine_gradient_kernel<T, false, false>
                      : past ? &combine_gradient_kernel<T, true, true> : &combine_gradient_kernel<T, true, false>;
  hipLaunchKernelGGL(kernel, dim3(capped(d.tokens) + zero_groups), dim3(256), 0, stream,
                     static_cast<const T *>(buffers[0]), static_cast<const float *>(buffers[1]),
                     static_cast<const uint32_t *>(buffers[2]), static_cast<const uint32_t *>(buffers[3]),
                     static_cast<const T *>(buffers[4]), d_rows, d_weights, d.tokens, d.per_token, d.width, zero_groups);
  check_launch(target);
}

}  // namespace

extern "C" {

size_t bpl_expert_sort_scratch_bytes(uint32_t pairs, uint32_t experts) {
  const SortShape s = sort_shape(pairs);
  return s.groups > 1 ? static_cast<size_t>(s.groups) * sort_bins(experts) * sizeof(uint32_t) : 0;
}

BPL_EXPERT_DEFINE(expert_topk, topk)
BPL_EXPERT_DEFINE(expert_topk_gradient, topk_gradient)
BPL_TARGET(expert_sort) { sort("expert_sort", static_cast<hipStream_t>(stream), buffers, opaque, opaque_len); }
BPL_EXPERT_DEFINE(expert_dispatch, dispatch)
BPL_EXPERT_DEFINE(expert_dispatch_gradient, dispatch_gradient)
BPL_EXPERT_DEFINE(expert_combine, combine)
BPL_EXPERT_DEFINE(expert_combine_gradient, combine_gradient)

}  // extern "C"
