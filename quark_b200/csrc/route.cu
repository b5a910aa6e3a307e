// Routing of tokens to experts by scores: softmax or sigmoid of the logits, an optional bias that takes part in the choice only, the
// choice inside the best groups of experts, and the slot tables of the experts' products (rows sorted by expert, every expert's run
// padded to whole 128-row tiles).
//
//   s = softmax(l) | sigmoid(l)      c = s + bias      group score = the sum of a group's best one or two c
//   the kept groups, then the top k of c inside them (equal values: the lower index first)      w = s / sum of the chosen s * factor
//
// A choice compares numbers that may lie next to one another, so it is made on what the formula says and not on a rounding of it:
// where c grows with l alone (no bias, groups by their best one) on the logits themselves, else on c in 64 bits.  Weights are f32.
//
// A warp takes a token; its lanes hold P consecutive experts each.  The tables need, for every choice, how many earlier tokens chose
// the same expert: a block's tokens are a 64-bit mask per expert (rank = set bits below the token), and blocks are joined by the
// counts that each leaves in the workspace.  Up to 64 tokens one block does all in one launch.
#include "common.cuh"

namespace qb {

constexpr int kRouteMaxExperts = 512, kRouteMaxGroups = 32, kRouteMaxTopK = 32;
constexpr int kRouteTokens = 64;    // tokens of a block
constexpr int kRouteThreads = 512;  // one thread per expert in the scan
constexpr int kRouteTile = 128;     // row tile of the grouped product
constexpr size_t kRouteWsOffset = 64u << 10;  // the area in front belongs to the GEMM's counters

struct RouteArgs {
  const void* logits;
  const float* bias;
  int f32, sigmoid, M, E, top_k, groups, kept, top, renorm;
  float factor;
  int *experts, *slot_token, *tile_expert, *tile_rows, *token_slot;
  float *weights, *slot_weight;
  int n_tiles;
  int* counts;  // [block][E]
};

// Unsigned keys in the order of the values; 0 is kept for what cannot be chosen, NaN comes next.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);  // (-0 is 0)
  return v != v ? 1u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return v != v ? 1ull : (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = static_cast<uint32_t>(k >> 32), top = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t lo = __reduce_max_sync(0xffffffffu, hi == top ? static_cast<uint32_t>(k) : 0u);
  return static_cast<uint64_t>(top) << 32 | lo;
}
template <typename V>
__device__ __forceinline__ V lowest() {
  return sizeof(V) == 8 ? static_cast<V>(__longlong_as_double(0xfff0000000000000ll)) : static_cast<V>(__uint_as_float(0xff800000u));
}

// One token: lane j < top_k returns its j-th choice and weight.  V: what the choice compares (float: the logits; double: scores).
template <int P, typename V>
__device__ __forceinline__ void choose(const RouteArgs& a, int t, V* scratch, int& my_expert, float& my_weight) {
  const int lane = threadIdx.x & 31, e0 = lane * P;
  float l[P];
  const size_t at = static_cast<size_t>(t) * a.E + e0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    l[i] = __uint_as_float(0xff800000u);
    if (e0 + i < a.E) l[i] = a.f32 ? static_cast<const float*>(a.logits)[at + i] : bf16_bits_to_f32(static_cast<const uint16_t*>(a.logits)[at + i]);
  }
  // softmax: the largest logit (0 for a row that has none) and the sum
  float top = 0.f, total = 1.f;
  V c[P];
  if (!a.sigmoid) {
    top = l[0];
#pragma unroll
    for (int i = 1; i < P; ++i) top = fmaxf(top, l[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == __uint_as_float(0xff800000u)) top = 0.f;
  }
  if constexpr (sizeof(V) == 8) {
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] = 1.0 / (1.0 + exp(-static_cast<double>(l[i])));
    } else {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        c[i] = exp(static_cast<double>(l[i]) - static_cast<double>(top));
        sum += c[i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      total = static_cast<float>(sum);
      const double inv = sum == 0.0 ? 0.0 : 1.0 / sum;
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] *= inv;
    }
    if (a.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (e0 + i < a.E) c[i] += static_cast<double>(a.bias[e0 + i]);
    }
  } else {
    if (!a.sigmoid && !a.renorm) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) total += expf(l[i] - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = l[i];
  }
  unsigned kept = 0xffffffffu;  // groups
  const int size = a.E / a.groups;
  if (a.groups > 1) {
    V best = lowest<V>(), second = lowest<V>();
    auto take = [&](V v) {
      if (v > best) {
        second = best;
        best = v;
      } else if (v > second) {
        second = v;
      }
    };
    const int lanes = size / P;  // of a group
    if (size % P == 0 && (lanes & (lanes - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < P; ++i) take(c[i]);
      for (int o = 1; o < lanes; o <<= 1) {
        const V b = __shfl_xor_sync(0xffffffffu, best, o), s = __shfl_xor_sync(0xffffffffu, second, o);
        take(b);
        if (s > second) second = s;
      }
      best = __shfl_sync(0xffffffffu, best, lane * lanes & 31);
      second = __shfl_sync(0xffffffffu, second, lane * lanes & 31);
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (e0 + i < a.E) scratch[e0 + i] = c[i];
      __syncwarp();
      if (lane < a.groups)
        for (int i = 0; i < size; ++i) take(scratch[lane * size + i]);
      __syncwarp();
    }
    auto key = order_key(a.top == 2 ? best + second : best);
    if (lane >= a.groups) key = 0;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const auto other = __shfl_sync(0xffffffffu, key, g);
      rank += other > key || (other == key && g < lane);
    }
    kept = __ballot_sync(0xffffffffu, lane < a.groups && rank < a.kept);
  }
  decltype(order_key(V{})) key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = e0 + i;
    key[i] = e < a.E && (a.groups == 1 || (kept >> (e / size) & 1u)) ? order_key(c[i]) : 0;
  }
  my_expert = 0;
  float my_logit = 0.f;
  for (int j = 0; j < a.top_k; ++j) {
    auto k = key[0];
    int at_i = 0;
    float v = l[0];
#pragma unroll
    for (int i = 1; i < P; ++i)
      if (key[i] > k) {
        k = key[i];
        at_i = i;
        v = l[i];
      }
    const auto most = warp_max(k);
    const int who = __ffs(__ballot_sync(0xffffffffu, k == most)) - 1;
    const int e = __shfl_sync(0xffffffffu, e0 + at_i, who);
    v = __shfl_sync(0xffffffffu, v, who);
    if (lane == j) {
      my_expert = e;
      my_logit = v;
    }
    if (lane == who) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (i == at_i) key[i] = 0;
    }
  }
  float s = 0.f;
  if (lane < a.top_k) s = a.sigmoid ? 1.f / (1.f + expf(-my_logit)) : expf(my_logit - top);
  float by = total;
  if (a.renorm) {
    by = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) by += __shfl_xor_sync(0xffffffffu, by, o);
  }
  my_weight = by == 0.f ? 0.f : s / by * a.factor;
}

struct RouteShared {
  unsigned mask[kRouteMaxExperts][2];  // tokens of the block that chose the expert
  int total[kRouteMaxExperts], first[kRouteMaxExperts], before[kRouteMaxExperts];  // tokens of an expert, its first tile, tokens of earlier blocks
  int warp_sum[kRouteThreads / 32];
};

// The tables of the block's tokens, and the tiles blockIdx.x, blockIdx.x + gridDim.x, ... of all.  mask, total and before are in place.
__device__ __forceinline__ void write_tables(const RouteArgs& a, RouteShared& sh, int t0, int tokens) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tiles = tid < a.E ? (sh.total[tid] + kRouteTile - 1) / kRouteTile : 0;
  int inc = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) sh.warp_sum[warp] = inc;
  __syncthreads();
  for (int w = 0; w < warp; ++w) inc += sh.warp_sum[w];
  if (tid < a.E) sh.first[tid] = inc - tiles;
  __syncthreads();
  for (int i = tid; i < tokens * a.top_k; i += kRouteThreads) {
    const int tl = i / a.top_k, t = t0 + tl;
    const size_t at = static_cast<size_t>(t0) * a.top_k + i;
    const int e = a.experts[at];
    const unsigned lo = sh.mask[e][0], hi = sh.mask[e][1];
    const int rank = tl < 32 ? __popc(lo & ((1u << tl) - 1u)) : __popc(lo) + __popc(hi & ((1u << (tl - 32)) - 1u));
    const int slot = sh.first[e] * kRouteTile + sh.before[e] + rank;
    a.token_slot[at] = slot;
    a.slot_token[slot] = t;
    a.slot_weight[slot] = a.weights[at];
  }
  // four tiles at a time: their experts and rows, and the slots that hold no token
  for (int i = blockIdx.x * (kRouteThreads / kRouteTile) + tid / kRouteTile; i < a.n_tiles; i += gridDim.x * (kRouteThreads / kRouteTile)) {
    int lo = 0, hi = a.E;  // the first expert whose run ends behind tile i
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (sh.first[mid] + (sh.total[mid] + kRouteTile - 1) / kRouteTile > i) hi = mid;
      else lo = mid + 1;
    }
    const int rows = lo < a.E ? min(sh.total[lo] - (i - sh.first[lo]) * kRouteTile, kRouteTile) : 0;
    const int r = tid % kRouteTile;
    if (r == 0) {
      a.tile_expert[i] = lo < a.E ? lo : -1;
      a.tile_rows[i] = rows;
    }
    if (r >= rows) {
      a.slot_token[i * kRouteTile + r] = -1;
      a.slot_weight[i * kRouteTile + r] = 0.f;
    }
  }
}

template <int P, typename V>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs args) {
  __shared__ RouteShared sh;
  extern __shared__ double route_scratch[];  // [warp][E] of V where there are groups
  RouteArgs a = args;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  sh.mask[tid][0] = sh.mask[tid][1] = 0u;
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();
  a.logits = after_wait(a.logits);
  a.bias = after_wait(a.bias);
  const int t0 = blockIdx.x * kRouteTokens, tokens = min(a.M - t0, kRouteTokens);
  V* scratch = reinterpret_cast<V*>(route_scratch) + static_cast<size_t>(warp) * a.E;
  for (int tl = warp; tl < tokens; tl += kRouteThreads / 32) {
    int e;
    float w;
    choose<P, V>(a, t0 + tl, scratch, e, w);
    if (lane < a.top_k) {
      const size_t at = static_cast<size_t>(t0 + tl) * a.top_k + lane;
      a.experts[at] = e;
      a.weights[at] = w;
      if (a.n_tiles > 0) atomicOr(&sh.mask[e][tl >> 5], 1u << (tl & 31));  // (an or of different bits: the same whatever the order)
    }
  }
  if (a.n_tiles == 0) return;
  __syncthreads();
  const int n = tid < a.E ? __popc(sh.mask[tid][0]) + __popc(sh.mask[tid][1]) : 0;
  if (gridDim.x > 1) {
    if (tid < a.E) a.counts[static_cast<size_t>(blockIdx.x) * a.E + tid] = n;
    return;
  }
  sh.total[tid] = n;
  sh.before[tid] = 0;
  write_tables(a, sh, t0, tokens);
}

__global__ void __launch_bounds__(kRouteThreads) route_tables_kernel(const RouteArgs args) {
  __shared__ RouteShared sh;
  RouteArgs a = args;
  const int tid = threadIdx.x;
  sh.mask[tid][0] = sh.mask[tid][1] = 0u;
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();
  a.experts = after_wait(a.experts);
  a.weights = after_wait(a.weights);
  const int* counts = after_wait(a.counts);
  const int t0 = blockIdx.x * kRouteTokens, tokens = min(a.M - t0, kRouteTokens);
  for (int i = tid; i < tokens * a.top_k; i += kRouteThreads) {
    const int tl = i / a.top_k;
    atomicOr(&sh.mask[a.experts[static_cast<size_t>(t0) * a.top_k + i]][tl >> 5], 1u << (tl & 31));
  }
  int total = 0, before = 0;
  if (tid < a.E) {
#pragma unroll 8
    for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
      const int n = counts[static_cast<size_t>(b) * a.E + tid];
      total += n;
      if (b < static_cast<int>(blockIdx.x)) before += n;
    }
  }
  sh.total[tid] = total;
  sh.before[tid] = before;
  __syncthreads();
  write_tables(a, sh, t0, tokens);
}

template <typename V>
static int32_t launch_choose(const RouteArgs& a, int blocks, size_t smem, cudaStream_t st) {
  auto go = [&](auto kernel) -> int32_t {
    if (smem > 32768) QB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));  // (beside the static tables)
    return launch_dep("moe_route_scored", kernel, dim3(blocks), dim3(kRouteThreads), smem, st, a);
  };
  const int per_lane = (a.E + 31) / 32;
  if (per_lane <= 1) return go(route_choose_kernel<1, V>);
  if (per_lane <= 2) return go(route_choose_kernel<2, V>);
  if (per_lane <= 4) return go(route_choose_kernel<4, V>);
  if (per_lane <= 8) return go(route_choose_kernel<8, V>);
  return go(route_choose_kernel<16, V>);
}

static int32_t validate_route(const qb_route_params* p) {
  QB_REQUIRE(p != nullptr, QB_ERR_INVALID_ARG, "moe_route_scored: params are NULL");
  QB_REQUIRE(p->M > 0 && p->E > 0 && p->E <= kRouteMaxExperts, QB_ERR_INVALID_ARG, "moe_route_scored: %d tokens, %d experts (at most %d)", p->M, p->E, kRouteMaxExperts);
  QB_REQUIRE(p->top_k > 0 && p->top_k <= p->E && p->top_k <= kRouteMaxTopK, QB_ERR_INVALID_ARG, "moe_route_scored: top_k %d of %d experts (at most %d)", p->top_k, p->E,
             kRouteMaxTopK);
  QB_REQUIRE(static_cast<long long>(p->M) * p->E < (1ll << 40) && static_cast<long long>(p->M) * p->top_k < (1ll << 30), QB_ERR_INVALID_ARG, "moe_route_scored: %d tokens", p->M);
  QB_REQUIRE(p->logits_dtype == QB_BF16 || p->logits_dtype == QB_F32, QB_ERR_INVALID_ARG, "moe_route_scored: logits dtype %d", p->logits_dtype);
  QB_REQUIRE(p->scoring == 0 || p->scoring == 1, QB_ERR_INVALID_ARG, "moe_route_scored: scoring %d", p->scoring);
  QB_REQUIRE(p->n_groups >= 1 && p->n_groups <= kRouteMaxGroups && p->E % p->n_groups == 0, QB_ERR_INVALID_ARG, "moe_route_scored: %d groups of %d experts (at most %d)",
             p->n_groups, p->E, kRouteMaxGroups);
  QB_REQUIRE(p->topk_groups >= 1 && p->topk_groups <= p->n_groups && p->topk_groups * (p->E / p->n_groups) >= p->top_k, QB_ERR_INVALID_ARG,
             "moe_route_scored: %d of %d groups of %d experts hold no %d choices", p->topk_groups, p->n_groups, p->E / p->n_groups, p->top_k);
  QB_REQUIRE(p->group_top == 1 || (p->group_top == 2 && (p->n_groups == 1 || p->E / p->n_groups >= 2)), QB_ERR_INVALID_ARG, "moe_route_scored: group_top %d of groups of %d",
             p->group_top, p->E / p->n_groups);
  return QB_OK;
}

}  // namespace qb

using namespace qb;

extern "C" size_t qb_moe_scored_slots(int32_t M, int32_t E, int32_t top_k) {
  if (M <= 0 || E <= 0 || top_k <= 0 || top_k > E || static_cast<long long>(M) * top_k >= (1ll << 30)) return 0;
  // u experts with a token each fill u tiles, and every 128 tokens more at most one
  const long long n = static_cast<long long>(M) * top_k, u = n < E ? n : E;
  return static_cast<size_t>((u + (n - u) / kRouteTile) * kRouteTile);
}

extern "C" size_t qb_moe_route_scored_workspace_bytes(const qb_route_params* p) {
  if (validate_route(p) != QB_OK || p->M <= kRouteTokens) return 0;
  return kRouteWsOffset + static_cast<size_t>((p->M + kRouteTokens - 1) / kRouteTokens) * p->E * sizeof(int);
}

extern "C" int32_t qb_moe_route_scored(const void* logits, const float* bias, int32_t* experts, float* weights, int32_t* slot_token, float* slot_weight, int32_t* tile_expert,
                                       int32_t* tile_rows, int32_t* token_slot, const qb_route_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  int32_t rc = validate_route(p);
  if (rc != QB_OK) return rc;
  QB_REQUIRE(logits && experts && weights, QB_ERR_INVALID_ARG, "moe_route_scored: NULL pointer");
  const bool tables = slot_token != nullptr;
  QB_REQUIRE((slot_weight != nullptr) == tables && (tile_expert != nullptr) == tables && (tile_rows != nullptr) == tables && (token_slot != nullptr) == tables,
             QB_ERR_INVALID_ARG, "moe_route_scored: the slot tables come together");
  const uintptr_t all = reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(experts) | reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(slot_token) |
                        reinterpret_cast<uintptr_t>(slot_weight) | reinterpret_cast<uintptr_t>(tile_expert) | reinterpret_cast<uintptr_t>(tile_rows) |
                        reinterpret_cast<uintptr_t>(token_slot);
  QB_REQUIRE(aligned16(logits) && (all & 3u) == 0, QB_ERR_ALIGN, "moe_route_scored: logits must be 16-byte aligned");
  const int blocks = (p->M + kRouteTokens - 1) / kRouteTokens;
  if (tables && blocks > 1) {
    const size_t need = qb_moe_route_scored_workspace_bytes(p);
    QB_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned16(workspace), QB_ERR_WORKSPACE, "moe_route_scored: workspace of %zu bytes needed, %zu given", need,
               workspace_bytes);
  }
  RouteArgs a{};
  a.logits = logits; a.bias = bias; a.f32 = p->logits_dtype == QB_F32; a.sigmoid = p->scoring; a.M = p->M; a.E = p->E; a.top_k = p->top_k;
  a.groups = p->n_groups; a.kept = p->topk_groups; a.top = p->group_top; a.renorm = p->renormalize != 0; a.factor = p->factor;
  if (a.kept == a.groups) a.groups = 1;  // every group is kept
  a.experts = experts; a.weights = weights; a.slot_token = slot_token; a.slot_weight = slot_weight; a.tile_expert = tile_expert; a.tile_rows = tile_rows;
  a.token_slot = token_slot;
  a.n_tiles = tables ? static_cast<int>(qb_moe_scored_slots(p->M, p->E, p->top_k) / kRouteTile) : 0;
  a.counts = tables && blocks > 1 ? reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + kRouteWsOffset) : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = bias != nullptr || (a.groups > 1 && a.top == 2);
  const size_t smem = a.groups > 1 ? static_cast<size_t>(kRouteThreads / 32) * a.E * (wide ? 8 : 4) : 0;
  rc = wide ? launch_choose<double>(a, blocks, smem, st) : launch_choose<float>(a, blocks, smem, st);
  if (rc != QB_OK || !tables || blocks == 1) return rc;
  return launch_dep("moe_route_scored (tables)", route_tables_kernel, dim3(blocks), dim3(kRouteThreads), 0, st, a);
}
