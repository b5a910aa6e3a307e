// Routing of tokens to experts by scores: softmax or sigmoid of the logits, an optional bias that takes part in the choice only, the
// choice inside the best groups of experts, and the slot tables of the experts' products (rows sorted by expert, every expert's run
// padded to whole 128-row tiles).
//
//   s = softmax(l) | sigmoid(l)      c = s + bias      group score = the sum of a group's best one or two c
//   the kept groups, then the top k of c inside them (equal values: the lower index first)      w = s / sum of the chosen s * factor
//
// A choice compares numbers that may lie next to one another, so it is made on what the formula says and not on a rounding of it:
// where c grows with l alone (no bias, groups by their best one) on the logits themselves, else on c in 32 bits as long as what it
// compares lies apart by more than those are off, and in 64 bits for a token where it does not.  Weights are f32, in 64 bits where
// chosen scores leave it.
//
// The choice in 32 bits (select_fast) takes every number of experts without groups, and groups of whole lanes, a power of two of them, at P = 1, 2, 4,
// 8 or 16 experts to a lane (E / 32 rounded up to one of these).  Others (24 experts in 4 groups, 40, 72, 96, 160, 192, 320 or 384 in 8) go the slow way
// (select_exact) for every token, and where the choice is on c, all of it in 64 bits.  8192 tokens, 8 groups, sigmoid with a bias, us with tables: 256 experts
// 20.9, 512 32; 96 25, 160 37, 192 42, 320 76, 384 88 (one token: 256 6.2, 160 10.4, 384 17.6).  So do choices of 32 of more experts on c, since the 33rd has no
// lane to be compared in, and of 31 where two candidates are close (256 experts without groups and tables: top_k 30 18.7, 31 28.5, 32 59.5).
//
// A warp takes a token; its lanes hold P consecutive experts each.  The tables need, for every choice, how many earlier tokens chose
// the same expert: a block's tokens are a 64-bit mask per expert (rank = set bits below the token), and blocks are joined by the
// counts (a byte each) that they leave in the workspace.  A few tokens are one block's, which does all in one launch.
//
// What bounds it: a token of 256 experts in 8 groups is about 1100 instructions, so 8192 tokens take 13 us of issue slots (6.5 us 2048); among 512 or more
// there is likely one with a comparison that needs the 64 bits, 1.5 us that nothing hides (3.7 with all of its scores in 64 bits instead of two to a lane:
// 512 tokens 12.3 us with their tables instead of 9.6, 8192 24.9 instead of 20.9).  The tables add 3.7 - 8 us, a chain of trips to L2.  Every block adds up
// the counts of all, which past 10,000 tokens grows with their square (65536 tokens: 70 of 163 us, 2^18 0.9 of 1.2 ms, 2^20 12 of 14).
#include <atomic>

#include "common.cuh"

namespace qb {

constexpr int kRouteMaxExperts = 512, kRouteMaxGroups = 32, kRouteMaxTopK = 32;
constexpr int kRouteTokens = 64, kRouteFewTokens = 4;  // most and fewest tokens of a block
constexpr int kRouteThreads = 1024;
// Tokens of a call with tables.  Every block reads the counts of all, 64 tokens each: 14 ms at 2^20 tokens of 256 experts, some seconds here, and
// the threads of all blocks, which slots are numbered by, stay far inside 32 bits.
constexpr int kRouteMaxTableTokens = 1 << 24;
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
  int tokens;       // of a block
  uint8_t* counts;  // [block][E rounded up to 4]
  int vec, vec_bias;  // rows of logits, and the bias, are whole 16-byte vectors
  int size;     // experts of a group
  int regular;  // no groups, or groups of whole lanes, a power of two of them
  int lanes;    // of a group then
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

__device__ __forceinline__ float logit_at(const RouteArgs& a, const uint8_t* row, int e) {
  return a.f32 ? reinterpret_cast<const float*>(row)[e] : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[e]);
}

// What the formula compares, in 64 bits.
struct Exact {
  const RouteArgs& a;
  const uint8_t* row;
  float top;  // softmax: the largest logit
  // softmax: 1 / the sum over the row, 0 for a row without one (the whole warp)
  __device__ __forceinline__ double scale() const {
    double sum = 0.0;
    if (!a.sigmoid) {
#pragma unroll 2
      for (int e = threadIdx.x & 31; e < a.E; e += 32) sum += exp(static_cast<double>(logit_at(a, row, e)) - static_cast<double>(top));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    return sum == 0.0 ? 0.0 : 1.0 / sum;
  }
  __device__ __forceinline__ double value(int e, double by) const {
    const double x = static_cast<double>(logit_at(a, row, e));
    const double s = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - static_cast<double>(top)) * by;
    return a.bias != nullptr ? s + static_cast<double>(a.bias[e]) : s;
  }
};

// The choice of one token among the values c of its lanes' experts: lane j < top_k receives the j-th expert.  Exact, and the slow way:
// up to 3000 instructions a token.
template <int P, typename V>
__device__ __noinline__ int select_exact(const RouteArgs& a, const V (&c)[P], V* scratch) {
  const int lane = threadIdx.x & 31, e0 = lane * P;
  unsigned kept = 0xffffffffu;  // groups
  const int size = a.size;
  if (a.groups > 1) {
    V best = lowest<V>(), second = lowest<V>();
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (e0 + i < a.E) scratch[e0 + i] = c[i];
    __syncwarp();
    if (lane < a.groups)
      for (int i = 0; i < size; ++i) {
        const V v = scratch[lane * size + i];
        if (v > best) {
          second = best;
          best = v;
        } else if (v > second) {
          second = v;
        }
      }
    __syncwarp();
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
  int mine = 0;
  for (int j = 0; j < a.top_k; ++j) {
    auto k = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < P; ++i)
      if (key[i] > k) {
        k = key[i];
        at = i;
      }
    const auto most = warp_max(k);
    const int who = __ffs(__ballot_sync(0xffffffffu, k == most)) - 1;
    const int e = __shfl_sync(0xffffffffu, e0 + at, who);
    if (lane == j) mine = e;
    if (lane == who) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (i == at) key[i] = 0;
    }
  }
  return mine;
}

// The same on values in 32 bits: a lane's experts become keys whose low bits hold their place in the lane, sorted once, and a round takes
// the largest head.  kMargin: the values are off by less than kOff of max(1, their size) each, and a key lies below its value by up to kLow
// units of its last place, kCut of its size.  (In units of 2^-24, a score being at most 1: an exponential 4; for softmax the P + 5
// roundings of the sum, 13 with 8 experts to a lane, 21 with 16, and a quotient and a product 2; for the sigmoid a sum and a quotient 5; the
// bias 1: 20 and 28, of the 24 and 32 that kOff is.)  Without, the values are exact but for the low bits.  What the whole warp learns:
// kFound, kOrder (with kMargin: the choice is among the first top_k + 1, which lanes 0 .. top_k hold, but some of them lie within
// 2 kOff + kCut of one another), or kOpen (too close for that, or equal with low bits lost: select_exact has to choose).
enum Selected { kFound, kOrder, kOpen };
template <int P, bool kMargin>
__device__ __forceinline__ Selected select_fast(const RouteArgs& a, const float (&c)[P], bool lossless, const Exact& exact, int& mine) {
  constexpr uint32_t kLow = P > 8 ? 15u : 7u;
  constexpr float kOff = P > 8 ? 0x1p-19f : 0x1.8p-20f, kCut = static_cast<float>(kLow) * 0x1p-23f, kApart = P > 8 ? 0x1.8p-18f : 0x1p-18f;
  static_assert(2.f * kOff + kCut < kApart, "see above");
  const int lane = threadIdx.x & 31, e0 = lane * P;
  uint32_t key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    uint32_t k = order_key(c[i]);
    if (c[i] != c[i]) k = kLow + 1;
    key[i] = e0 + i < a.E ? (k & ~kLow) | (kLow - i) : 0u;
  }
  auto value = [](uint32_t k) {
    k &= ~kLow;
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
  };
  auto apart = [](float hi, float lo) { return hi - lo > kApart * fmaxf(1.f, fmaxf(fabsf(hi), fabsf(lo))); };
#pragma unroll
  for (int size = 2; size <= P; size *= 2)  // descending, by a bitonic network
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2)
#pragma unroll
      for (int i = 0; i < P; ++i)
        if ((i & d) == 0) {
          const bool down = (i & size) == 0 || size == P;
          const uint32_t hi = max(key[i], key[i + d]), lo = min(key[i], key[i + d]);
          key[i] = down ? hi : lo;
          key[i + d] = down ? lo : hi;
        }
  bool fine = true;
  if (a.groups > 1) {
    const int lanes = a.lanes;
    float best = value(key[0]), second = P > 1 ? value(key[P > 1 ? 1 : 0]) : __uint_as_float(0xff800000u);
    for (int o = 1; o < lanes; o <<= 1) {
      const float b = __shfl_xor_sync(0xffffffffu, best, o), s = __shfl_xor_sync(0xffffffffu, second, o);
      second = fmaxf(fminf(best, b), fmaxf(second, s));
      best = fmaxf(best, b);
    }
    const float score = a.top == 2 ? best + second : best;  // of this lane's group
    uint32_t open = lane * P < a.E ? order_key(score) : 0u;
    bool mine_kept = false;
    uint32_t last = 0u;
    for (int j = 0; j < a.kept; ++j) {  // (kept < groups)
      last = __reduce_max_sync(0xffffffffu, open);
      const int who = __ffs(__ballot_sync(0xffffffffu, open == last)) - 1;
      if ((lane ^ who) < lanes) {  // the same group
        mine_kept = true;
        open = 0u;
      }
    }
    if (kMargin) {
      // A sum is off by what its terms are, which may be far larger than it: the lowest that any kept group's may be, against the highest
      // of any other's.  (Minus infinity is exact, and as a bound NaN, the lowest key.)
      const float size = a.top == 2 ? 2.f * fmaxf(fabsf(best), fabsf(second)) : fabsf(best), off = 2.f * kOff * fmaxf(1.f, size);
      const uint32_t lo = mine_kept ? order_key(score - off) : 0xffffffffu;
      const uint32_t hi = mine_kept || lane * P >= a.E ? 0u : order_key(score + (off + kCut * size));
      fine = __reduce_min_sync(0xffffffffu, lo) > __reduce_max_sync(0xffffffffu, hi);
      if (!fine && __all_sync(0xffffffffu, P <= 2 || lane * P >= a.E || apart(value(key[P > 2 ? 1 : 0]), value(key[P > 2 ? 2 : 0])))) {
        // Which two are a lane's best is plain: their sums in 64 bits, two scores to a lane instead of all.
        const double by = exact.scale(), none = lowest<double>();
        double hi2[2] = {none, none};
#pragma unroll
        for (int i = 0; i < (P > 1 ? 2 : 1); ++i)
          if (lane * P < a.E) {
            const double v = exact.value(e0 + static_cast<int>(kLow - (key[i] & kLow)), by);
            if (v == v) hi2[i] = v;
          }
        double most = fmax(hi2[0], hi2[1]), next = fmin(hi2[0], hi2[1]);
        for (int o = 1; o < lanes; o <<= 1) {
          const double b = __shfl_xor_sync(0xffffffffu, most, o), s = __shfl_xor_sync(0xffffffffu, next, o);
          next = fmax(fmin(most, b), fmax(next, s));
          most = fmax(most, b);
        }
        uint64_t left = lane * P < a.E ? order_key(a.top == 2 ? most + next : most) : 0ull;
        mine_kept = false;
        for (int j = 0; j < a.kept; ++j) {
          const uint64_t first = warp_max(left);
          const int who = __ffs(__ballot_sync(0xffffffffu, left == first)) - 1;
          if ((lane ^ who) < lanes) {
            mine_kept = true;
            left = 0ull;
          }
        }
        fine = true;
      }
    } else {
      fine = lossless || last != __reduce_max_sync(0xffffffffu, open);
    }
    if (!mine_kept) {
#pragma unroll
      for (int i = 0; i < P; ++i) key[i] = 0u;
    }
  }
  const int left = a.groups == 1 ? a.E : a.kept * a.size;
  // top_k choices and the next one or two, as far as there are lanes and experts for them; lane j keeps the j-th and its key
  const int rounds = min(min(a.top_k + (kMargin ? 2 : 1), left), 32);
  mine = 0;
  uint32_t got = 0u;
  for (int j = 0; j < rounds; ++j) {
    // (with kMargin, whichever of two equal values comes first: they are too close to count)
    const uint32_t head = kMargin ? key[0] : key[0] & ~kLow, most = __reduce_max_sync(0xffffffffu, head);
    const int who = __ffs(__ballot_sync(0xffffffffu, head == most)) - 1;
    const int e = kMargin ? who * P + static_cast<int>(kLow - (most & kLow)) : __shfl_sync(0xffffffffu, e0 + static_cast<int>(kLow - (key[0] & kLow)), who);
    if (lane == j) {
      mine = e;
      got = most;
    }
    if (lane == who) {
#pragma unroll
      for (int i = 0; i + 1 < P; ++i) key[i] = key[i + 1];
      key[P - 1] = 0u;
    }
  }
  const int k = a.top_k;
  const uint32_t next = __shfl_down_sync(0xffffffffu, got, 1), second = __shfl_down_sync(0xffffffffu, got, 2);
  if (!kMargin) {
    const bool same = __any_sync(0xffffffffu, lane < k && lane + 1 < rounds && got == next);
    if (!lossless && (same || (left > k && rounds <= k))) fine = false;
    return fine ? kFound : kOpen;
  }
  const bool close = __any_sync(0xffffffffu, lane < k && lane + 1 < rounds && !apart(value(got), value(next)));
  // the last choice against the one behind the next: else that might be among the top k
  const bool far = !__any_sync(0xffffffffu, lane == k - 1 && lane + 2 < rounds && !apart(value(got), value(second)));
  if (left > k && rounds <= k) return kOpen;  // the 32nd choice has no lane to be compared with
  if (!close) return fine ? kFound : kOpen;
  return fine && far && rounds > k && (rounds == k + 2 || left == k + 1) ? kOrder : kOpen;
}

// P consecutive values of a row as f32; `fill` past E.
template <int P>
__device__ __forceinline__ void load_row(const void* row, bool f32, bool vec, int e0, int E, float fill, float (&v)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) v[i] = fill;
  if constexpr (P >= 4) {
    if (vec) {  // rows are whole 16-byte vectors
      if (f32) {
#pragma unroll
        for (int i = 0; i < P; i += 4)
          if (e0 + i < E) {
            const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + e0 + i);
            v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
          }
        return;
      }
      if constexpr (P >= 8) {
#pragma unroll
        for (int i = 0; i < P; i += 8)
          if (e0 + i < E) {
            const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + e0 + i);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              v[i + 2 * q] = bf16lo(w[q]);
              v[i + 2 * q + 1] = bf16hi(w[q]);
            }
          }
        return;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (e0 + i < E) v[i] = f32 ? static_cast<const float*>(row)[e0 + i] : bf16_bits_to_f32(static_cast<const uint16_t*>(row)[e0 + i]);
}

// One token: lane j < top_k returns its j-th choice and weight.  kScores: the choice is on c, else on the logits.
template <int P, bool kScores>
__device__ __forceinline__ void choose(const RouteArgs& a, int t, double* scratch, int& my_expert, float& my_weight) {
  const int lane = threadIdx.x & 31, e0 = lane * P;
  const float none = __uint_as_float(0xff800000u);
  const uint8_t* row = static_cast<const uint8_t*>(a.logits) + static_cast<size_t>(t) * a.E * (a.f32 ? 4 : 2);
  float l[P];
  load_row<P>(row, a.f32 != 0, a.vec != 0, e0, a.E, none, l);
  // softmax: the largest logit (0 for a row that has none) and the sum
  float top = 0.f, total = 1.f;
  if (!a.sigmoid) {
    top = l[0];
#pragma unroll
    for (int i = 1; i < P; ++i) top = fmaxf(top, l[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == none) top = 0.f;
    bool lost = false;  // NaN or infinity among the logits: the formula's scores are NaN, all of the row's
#pragma unroll
    for (int i = 0; i < P; ++i) lost |= !(l[i] < __uint_as_float(0x7f800000u));
    if (__any_sync(0xffffffffu, lost)) top = __uint_as_float(0x7fffffffu);
    if (kScores || !a.renorm) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) total += expf(l[i] - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
  }
  const Exact exact{a, row, top};
  if (!kScores) {
    if (!a.regular || select_fast<P, false>(a, l, a.f32 == 0, exact, my_expert) != kFound) my_expert = select_exact<P, float>(a, l, reinterpret_cast<float*>(scratch));
  } else {
    Selected found = kOpen;
    if (a.regular) {
      float c[P];
      const float by = total == 0.f ? 0.f : 1.f / total;
      if (a.bias != nullptr) load_row<P>(a.bias, true, a.vec_bias != 0, e0, a.E, 0.f, c);
      else {
#pragma unroll
        for (int i = 0; i < P; ++i) c[i] = 0.f;
      }
      // (|e^x| (2 + 1.16 |x|) 2^-24, what __expf may be off, is largest at small x: 2^-22)
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] += a.sigmoid ? __fdividef(1.f, 1.f + __expf(-l[i])) : __expf(l[i] - top) * by;
      found = select_fast<P, true>(a, c, false, exact, my_expert);
    }
    if (found != kFound) {
      const double by = exact.scale();
      if (found == kOrder) {  // the candidates in 64 bits, each by the lane that holds it
        const int n = a.top_k + 1;
        uint64_t key = 0;
        if (lane < n) key = order_key(exact.value(my_expert, by));
        int rank = 0, sorted = 0;
        for (int i = 0; i < n; ++i) {
          const uint64_t k = __shfl_sync(0xffffffffu, key, i);
          const int e = __shfl_sync(0xffffffffu, my_expert, i);
          rank += k > key || (k == key && e < my_expert);
        }
        for (int i = 0; i < n; ++i) {
          const int e = __shfl_sync(0xffffffffu, my_expert, i);
          if (__shfl_sync(0xffffffffu, rank, i) == lane) sorted = e;
        }
        my_expert = sorted;
      } else {
        double d[P];
#pragma unroll 1  // (the logits again from memory: indexed by a loop they would lie in local memory from the start, 8192 tokens 25.3 us instead of 24.2)
        for (int i = 0; i < P; ++i) d[i] = e0 + i < a.E ? exact.value(e0 + i, by) : 0.0;
        my_expert = select_exact<P, double>(a, d, scratch);
      }
    }
  }
  float s = 0.f, x = 0.f;
  if (lane < a.top_k) {
    x = logit_at(a, row, my_expert);
    if (a.sigmoid) {
      s = 1.f / (1.f + expf(-x));
    } else {  // with what the difference was rounded by: far below the row's largest that is more than the rest
      const float d = x - top, back = d - x, lost = (x - (d - back)) - (top + back);
      s = expf(d);
      if (s > 0.f) s = fmaf(s, lost, s);
    }
  }
  float by = total;
  if (a.renorm) {
    by = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) by += __shfl_xor_sync(0xffffffffu, by, o);
    // The bias chose experts whose scores leave 32 bits (a subnormal one has lost bits, a sum this small may be of such); their ratios do not.
    const bool tiny = lane < a.top_k && s < 1.17549435e-38f && x > __uint_as_float(0xff800000u);
    if (by < 1e-25f || __any_sync(0xffffffffu, tiny)) {
      const double t = static_cast<double>(top);
      const double wide = lane < a.top_k ? (a.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : exp(static_cast<double>(x) - t)) : 0.0;
      double all = wide;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      my_weight = all == 0.0 ? 0.f : static_cast<float>(wide / all) * a.factor;
      return;
    }
  }
  my_weight = by == 0.f ? 0.f : s / by * a.factor;
}

struct RouteShared {
  unsigned mask[kRouteMaxExperts][2];  // tokens of the block that chose the expert
  int total[kRouteMaxExperts], first[kRouteMaxExperts], before[kRouteMaxExperts];  // tokens of an expert, its first tile, tokens of earlier blocks
  int warp_sum[kRouteThreads / 32];
};

// The tables of the block's tokens, and its share of the rest.  mask, total and before are in place.
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
  int up_to = sh.warp_sum[lane];  // of this many warps and the ones before
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, up_to, o);
    if (lane >= o) up_to += x;
  }
  const int used = __shfl_sync(0xffffffffu, up_to, 31), earlier = __shfl_sync(0xffffffffu, up_to, max(warp - 1, 0));
  if (tid < a.E) sh.first[tid] = inc - tiles + (warp > 0 ? earlier : 0);
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
  // a warp per expert: the tiles of its run, and the slots behind its last token
  for (int e = blockIdx.x * (kRouteThreads / 32) + warp; e < a.E; e += gridDim.x * (kRouteThreads / 32)) {
    const int n = sh.total[e], f = sh.first[e], tl = (n + kRouteTile - 1) / kRouteTile;
    for (int i = lane; i < tl; i += 32) {
      a.tile_expert[f + i] = e;
      a.tile_rows[f + i] = min(n - i * kRouteTile, kRouteTile);
    }
    for (int i = n + lane; i < tl * kRouteTile; i += 32) {
      a.slot_token[f * kRouteTile + i] = -1;
      a.slot_weight[f * kRouteTile + i] = 0.f;
    }
  }
  // the tiles that no run reaches
  for (int i = used * kRouteTile + blockIdx.x * kRouteThreads + tid; i < a.n_tiles * kRouteTile; i += gridDim.x * kRouteThreads) {
    a.slot_token[i] = -1;
    a.slot_weight[i] = 0.f;
    if (i % kRouteTile == 0) {
      a.tile_expert[i / kRouteTile] = -1;
      a.tile_rows[i / kRouteTile] = 0;
    }
  }
}

__device__ __forceinline__ void clear_shared(RouteShared& sh) {
  for (int e = threadIdx.x; e < kRouteMaxExperts; e += blockDim.x) sh.mask[e][0] = sh.mask[e][1] = sh.total[e] = sh.before[e] = 0;
  __syncthreads();
}

template <int P, bool kScores>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs args) {
  __shared__ RouteShared sh;
  extern __shared__ double route_scratch[];  // [warp][E] of select_exact (of doubles, whatever it holds), where there are groups
  RouteArgs a = args;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  clear_shared(sh);
  grid_dep_wait();
  grid_dep_launch();
  a.logits = after_wait(a.logits);
  a.bias = after_wait(a.bias);
  const int t0 = blockIdx.x * a.tokens, tokens = min(a.M - t0, a.tokens);
  double* scratch = route_scratch + static_cast<size_t>(warp) * a.E;
  for (int tl = warp; tl < tokens; tl += blockDim.x / 32) {
    int e;
    float w;
    choose<P, kScores>(a, t0 + tl, scratch, e, w);
    if (lane < a.top_k) {
      const size_t at = static_cast<size_t>(t0 + tl) * a.top_k + lane;
      a.experts[at] = e;
      a.weights[at] = w;
      if (a.n_tiles > 0) atomicOr(&sh.mask[e][tl >> 5], 1u << (tl & 31));  // (an or of different bits: the same whatever the order)
    }
  }
  if (a.n_tiles == 0) return;
  __syncthreads();
  for (int e = tid; e < a.E; e += blockDim.x) {
    const int n = __popc(sh.mask[e][0]) + __popc(sh.mask[e][1]);
    if (gridDim.x > 1) a.counts[static_cast<size_t>(blockIdx.x) * ((a.E + 3) & ~3) + e] = static_cast<uint8_t>(n);
    sh.total[e] = n;
  }
  if (gridDim.x == 1) write_tables(a, sh, t0, tokens);
}

__global__ void __launch_bounds__(kRouteThreads) route_tables_kernel(const RouteArgs args) {
  __shared__ RouteShared sh;
  RouteArgs a = args;
  const int tid = threadIdx.x;
  clear_shared(sh);
  grid_dep_wait();
  grid_dep_launch();
  a.experts = after_wait(a.experts);
  a.weights = after_wait(a.weights);
  const int t0 = blockIdx.x * a.tokens, tokens = min(a.M - t0, a.tokens);
  for (int i = tid; i < tokens * a.top_k; i += kRouteThreads) {
    const int tl = i / a.top_k;
    atomicOr(&sh.mask[a.experts[static_cast<size_t>(t0) * a.top_k + i]][tl >> 5], 1u << (tl & 31));
  }
  // every block adds up the counts of all: four experts to a thread, the blocks shared by the threads
  const int words = (a.E + 3) / 4, word = tid % words, slices = kRouteThreads / words;
  const uint32_t* counts = reinterpret_cast<const uint32_t*>(after_wait(a.counts)) + word;
  if (tid / words < slices) {
    const int blocks = gridDim.x, self = blockIdx.x;
    for (int b0 = tid / words; b0 < blocks; b0 += 512 * slices) {  // (512 counts of up to 64 fit 16 bits)
      uint32_t total[2] = {0u, 0u}, before[2] = {0u, 0u};          // experts 0 and 2, 1 and 3
#pragma unroll 8
      for (int b = b0; b < min(blocks, b0 + 512 * slices); b += slices) {
        const uint32_t n = counts[static_cast<size_t>(b) * words], lo = n & 0x00ff00ffu, hi = n >> 8 & 0x00ff00ffu;
        total[0] += lo;
        total[1] += hi;
        if (b < self) {
          before[0] += lo;
          before[1] += hi;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (word * 4 + i < a.E) {  // (integer sums: the same whatever the order)
          atomicAdd(&sh.total[word * 4 + i], static_cast<int>(total[i & 1] >> (8 * (i & 2)) & 0xffffu));
          atomicAdd(&sh.before[word * 4 + i], static_cast<int>(before[i & 1] >> (8 * (i & 2)) & 0xffffu));
        }
    }
  }
  __syncthreads();
  write_tables(a, sh, t0, tokens);
}

template <int P, bool kScores>
static int32_t launch_choose(RouteArgs a, int blocks, cudaStream_t st) {
  a.size = a.E / a.groups;
  a.lanes = a.size / P;
  a.regular = a.groups == 1 || (a.size % P == 0 && (a.lanes & (a.lanes - 1)) == 0);
  static std::atomic<unsigned long long> configured{0};  // one bit per device
  int dev = 0;
  QB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || (configured.load(std::memory_order_relaxed) >> dev & 1) == 0) {
    QB_CUDA_OK(cudaFuncSetAttribute(route_choose_kernel<P, kScores>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRouteThreads / 32 * P * 32 * 8));
    if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int threads = blocks == 1 ? kRouteThreads : min(32 * a.tokens, kRouteThreads);  // (one block writes the tables as well)
  return launch_dep("moe_route_scored", route_choose_kernel<P, kScores>, dim3(blocks), dim3(threads), a.groups > 1 ? static_cast<size_t>(threads / 32) * a.E * sizeof(double) : 0, st, a);
}

template <bool kScores>
static int32_t launch_choose(const RouteArgs& a, int blocks, cudaStream_t st) {
  const int per_lane = (a.E + 31) / 32;
  if (per_lane <= 1) return launch_choose<1, kScores>(a, blocks, st);
  if (per_lane <= 2) return launch_choose<2, kScores>(a, blocks, st);
  if (per_lane <= 4) return launch_choose<4, kScores>(a, blocks, st);
  if (per_lane <= 8) return launch_choose<8, kScores>(a, blocks, st);
  return launch_choose<16, kScores>(a, blocks, st);
}

// Tokens of a block, a warp to each up to 32.  Few, so that few warps share an SM's issue slots (64 tokens of 256 experts,
// tables included, in one block: 19 us, in blocks of 4: 7.6), and as few blocks as that leaves, since every block of the tables
// adds up the counts of all and waits for the others' lines (512 tokens: 2 us more
// with 4 to a block than with 8).
static int block_tokens(int M) {
  int n = kRouteFewTokens;
  while (n < 16 && (M + n - 1) / n > 64) n *= 2;
  while (n < kRouteTokens && (M + n - 1) / n > 128) n *= 2;
  return n;
}
static int route_blocks(int M) { return (M + block_tokens(M) - 1) / block_tokens(M); }

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
  if (validate_route(p) != QB_OK || route_blocks(p->M) == 1) return 0;
  return kRouteWsOffset + static_cast<size_t>(route_blocks(p->M)) * ((p->E + 3) & ~3);
}

extern "C" int32_t qb_moe_route_scored(const void* logits, const float* bias, int32_t* experts, float* weights, int32_t* slot_token, float* slot_weight, int32_t* tile_expert,
                                       int32_t* tile_rows, int32_t* token_slot, const qb_route_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  int32_t rc = validate_route(p);
  if (rc != QB_OK) return rc;
  QB_REQUIRE(logits && experts && weights, QB_ERR_INVALID_ARG, "moe_route_scored: NULL pointer");
  const bool tables = slot_token != nullptr;
  QB_REQUIRE((slot_weight != nullptr) == tables && (tile_expert != nullptr) == tables && (tile_rows != nullptr) == tables && (token_slot != nullptr) == tables,
             QB_ERR_INVALID_ARG, "moe_route_scored: the slot tables come together");
  QB_REQUIRE(!tables || p->M <= kRouteMaxTableTokens, QB_ERR_UNSUPPORTED, "moe_route_scored: slot tables of at most %d tokens (got %d)", kRouteMaxTableTokens, p->M);
  const uintptr_t all = reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(experts) | reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(slot_token) |
                        reinterpret_cast<uintptr_t>(slot_weight) | reinterpret_cast<uintptr_t>(tile_expert) | reinterpret_cast<uintptr_t>(tile_rows) |
                        reinterpret_cast<uintptr_t>(token_slot);
  QB_REQUIRE(aligned16(logits) && (all & 3u) == 0, QB_ERR_ALIGN, "moe_route_scored: logits must be 16-byte aligned");
  const int blocks = route_blocks(p->M);
  if (tables && blocks > 1) {
    const size_t need = qb_moe_route_scored_workspace_bytes(p);
    QB_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned16(workspace), QB_ERR_WORKSPACE, "moe_route_scored: workspace of %zu bytes needed, %zu given", need,
               workspace_bytes);
  }
  RouteArgs a{};
  a.logits = logits; a.bias = bias; a.f32 = p->logits_dtype == QB_F32; a.sigmoid = p->scoring; a.M = p->M; a.E = p->E; a.top_k = p->top_k;
  a.groups = p->n_groups; a.kept = p->topk_groups; a.top = p->group_top; a.renorm = p->renormalize != 0; a.factor = p->factor;
  if (a.kept == a.groups) a.groups = 1;  // every group is kept
  a.vec = a.E % (a.f32 ? 4 : 8) == 0;
  a.vec_bias = aligned16(bias) && a.E % 4 == 0;
  a.experts = experts; a.weights = weights; a.slot_token = slot_token; a.slot_weight = slot_weight; a.tile_expert = tile_expert; a.tile_rows = tile_rows;
  a.token_slot = token_slot;
  a.tokens = block_tokens(p->M);
  a.n_tiles = tables ? static_cast<int>(qb_moe_scored_slots(p->M, p->E, p->top_k) / kRouteTile) : 0;
  a.counts = tables && blocks > 1 ? static_cast<uint8_t*>(workspace) + kRouteWsOffset : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool scores = bias != nullptr || (a.groups > 1 && a.top == 2);  // (else the choice is the logits')
  rc = scores ? launch_choose<true>(a, blocks, st) : launch_choose<false>(a, blocks, st);
  if (rc != QB_OK || !tables || blocks == 1) return rc;
  return launch_dep("moe_route_scored (tables)", route_tables_kernel, dim3(blocks), dim3(kRouteThreads), 0, st, a);
}
