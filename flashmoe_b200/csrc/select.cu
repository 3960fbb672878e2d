// Routing from logits: scores, choice, weights, and the order of the (token, choice) pairs by expert.
//
// Choosing is one warp per token with the row of scores in registers; ordering is a stable counting
// sort of the pairs by expert, by one cluster of CTAs whose histograms meet in distributed shared
// memory, so neither step needs scratch memory or atomics whose order could show.
//
// Which experts are chosen hangs on comparisons, and fp32 scores carry an error: where two of the
// scores that a decision hangs on are closer than twice that error, the token's row is decided again
// in 64 bits.  Without a bias the scores are never compared at all: softmax and sigmoid keep the
// order of the logits, so the logits, which are exact, are (inside a group too).
//
// Measured: 8192 tokens of 128 experts 14.3 us, 2048 of 256 experts in 8 groups 12.6 us, one token 4.2 us.  Reading the
// logits takes 0.8 us of the first; the rest is instructions (59 % of issue slots) and, in the ordering, a chain of
// steps that wait for one another.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "fp8.cuh"

namespace fmoe {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 32;
constexpr unsigned kAll = 0xffffffffu;

struct SelectParams {
  const void* logits;
  const float* bias;
  int32_t* ids;
  float* weights;
  int32_t* counts;
  int32_t* offsets;
  int32_t* positions;
  TokenSlot* table;     // of an MoE context, or null
  Route* routes;
  int capacity, round_ec;
  int S, E, k, dtype, score, groups, top_groups, group_max, renormalize;
  float scale;
};

// ---- choosing ---------------------------------------------------------------------------------------

// A masked expert (-infinity or NaN) orders below every other; +infinity is the largest finite number.
__device__ __forceinline__ float sane(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }

__device__ __forceinline__ float logit_at(const SelectParams& p, size_t i) {
  float x;
  if (p.dtype == FMOE_DT_FP32) x = fp8::fetched(static_cast<const float*>(p.logits) + i);
  else if (p.dtype == FMOE_DT_BF16) x = __bfloat162float(fp8::fetched(static_cast<const __nv_bfloat16*>(p.logits) + i));
  else x = __half2float(fp8::fetched(static_cast<const __half*>(p.logits) + i));
  return sane(x);
}

// A lane's logits of a row, lane + 32 i, all on their way together (the type is chosen around the loop, not in it: a
// branch around each load made them wait for one another, 4000 cycles for eight).  -infinity behind the last.
template <int V>
__device__ __forceinline__ void load_row(const SelectParams& p, size_t row, int lane, float (&v)[V]) {
  auto load = [&](const auto* from) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = lane + 32 * i < p.E ? fp8::to_float(fp8::fetched(from + row + lane + 32 * i)) : -INFINITY;
  };
  if (p.dtype == FMOE_DT_FP32) load(static_cast<const float*>(p.logits));
  else if (p.dtype == FMOE_DT_BF16) load(static_cast<const __nv_bfloat16*>(p.logits));
  else load(static_cast<const __half*>(p.logits));
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = sane(v[i]);
}

// An unsigned number that orders like the value (+0 and -0 alike); 0 is left for "nothing".
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template <typename F>
__device__ __forceinline__ F exp_of(F x) {
  if constexpr (sizeof(F) == 8) return exp(x); else return expf(x);
}
// exp(l - largest) or sigmoid(l); 0 for a masked logit.  In fp32 sigmoid is taken from exp(-|l|), which cannot
// overflow, without a branch on the sign.
template <typename F>
__device__ __forceinline__ F raw_score(F l, F largest, int score) {
  F s;
  if (score == FMOE_SCORE_SOFTMAX) {
    s = exp_of<F>(l - largest);
  } else if constexpr (sizeof(F) == 8) {
    s = 1.0 / (1.0 + exp(-l));
  } else {
    const float e = expf(-fabsf(l));
    s = __fdividef(l >= 0.0f ? 1.0f : e, 1.0f + e);
  }
  return l == -INFINITY ? F(0) : s;
}

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_max(F v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    const F o = __shfl_xor_sync(kAll, v, d);
    v = o > v ? o : v;
  }
  return v;
}

// A group's score from its experts' values in shared memory (each group's run one place longer than it has to be, so
// that the groups fall on different banks): teams of lanes, one a group, walk the values and keep the two
// largest.  Lane g < groups leaves with group g's score.
template <typename F>
__device__ __forceinline__ F group_score(const F* row, int E, int groups, bool largest_only, int lane) {
  int team = 32;
  while (team * groups > 32) team >>= 1;
  const int g = lane / team, sub = lane - g * team, size = E / groups;
  F a = -INFINITY, b = -INFINITY;   // the largest two
  if (g < groups) {
    for (int j = sub; j < size; j += team) {
      const F v = row[g * (size + 1) + j];
      if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
    }
  }
  for (int d = 1; d < team; d <<= 1) {
    const F oa = __shfl_xor_sync(kAll, a, d), ob = __shfl_xor_sync(kAll, b, d);
    if (oa > a) { b = a > ob ? a : ob; a = oa; } else { b = oa > b ? oa : b; }
  }
  const F s = largest_only || b == -INFINITY ? a : a + b;   // (masked experts add nothing)
  return __shfl_sync(kAll, s, (lane * team) & 31);
}

// Which groups stay, as bits; `gap` is how far the worst that stays lies above the best that goes.
template <typename F>
__device__ __forceinline__ uint32_t kept_groups(F mine, int groups, int top_groups, int lane, F& worst_kept, F& best_gone) {
  int before = 0;
  for (int g = 0; g < groups; ++g) {
    const F o = __shfl_sync(kAll, mine, g);
    before += o > mine || (o == mine && g < lane);
  }
  const bool stays = lane < groups && before < top_groups;
  worst_kept = -warp_max<F>(stays ? -mine : F(-INFINITY));
  best_gone = warp_max<F>(lane < groups && !stays ? mine : F(-INFINITY));
  return __ballot_sync(kAll, stays);
}

// The group of expert e: (e + 1/2) / size lies at least 1/2048 from a whole number, fp32 is exact to far less.
__device__ __forceinline__ int group_of(int e, float groups_per_expert) {
  return static_cast<int>((static_cast<float>(e) + 0.5f) * groups_per_expert);
}
// Bits i of the experts lane + 32 i that exist and whose group stays.
template <int V>
__device__ __forceinline__ uint32_t alive_bits(int E, int groups, uint32_t kept, int lane) {
  uint32_t alive = 0;
  if (groups == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane + 32 * i < E) alive |= 1u << i;
    return alive;
  }
  const float per = static_cast<float>(groups) / static_cast<float>(E);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 32 * i;
    if (e < E && (kept >> group_of(e, per) & 1)) alive |= 1u << i;
  }
  return alive;
}

// What is compared, in 64 bits.
template <int V>
__device__ __forceinline__ void exact_scores(const SelectParams& p, size_t row, int lane, double (&c)[V]) {
  double top = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 32 * i;
    c[i] = e < p.E ? static_cast<double>(logit_at(p, row + e)) : static_cast<double>(-INFINITY);
    top = c[i] > top ? c[i] : top;
  }
  top = warp_max<double>(top);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const bool masked = c[i] == -INFINITY;
    c[i] = raw_score<double>(c[i], top, p.score);
    sum += c[i];
    if (masked) c[i] = -INFINITY;
  }
  sum = warp_sum<double>(sum);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 32 * i;
    if (p.score == FMOE_SCORE_SOFTMAX && sum > 0.0) c[i] /= sum;
    if (p.bias != nullptr && e < p.E) c[i] += static_cast<double>(sane(fp8::fetched(p.bias + e)));
  }
}

// The groups that stay, decided in 64 bits.
template <int V>
__device__ __noinline__ uint32_t exact_groups(const SelectParams& p, size_t row, int lane, double* shared_row) {
  double c[V];
  exact_scores<V>(p, row, lane, c);
  const float per = static_cast<float>(p.groups) / static_cast<float>(p.E);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane + 32 * i < p.E) shared_row[lane + 32 * i + group_of(lane + 32 * i, per)] = c[i];
  __syncwarp();
  double worst, best;
  return kept_groups<double>(group_score<double>(shared_row, p.E, p.groups, p.group_max, lane), p.groups, p.top_groups, lane,
                             worst, best);
}

// The choice among the experts of the groups that stay, decided in 64 bits; lane j < k leaves with the j-th.
template <int V>
__device__ __noinline__ int choose_exactly(const SelectParams& p, size_t row, int lane, uint32_t kept) {
  double c[V];
  exact_scores<V>(p, row, lane, c);
  uint32_t alive = alive_bits<V>(p.E, p.groups, kept, lane);
  int mine = 0;
  for (int r = 0; r < p.k; ++r) {
    double best = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if ((alive >> i & 1) && (at == 0x7fffffff || c[i] > best)) { best = c[i]; at = lane + 32 * i; }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
      const double o = __shfl_xor_sync(kAll, best, d);
      const int oa = __shfl_xor_sync(kAll, at, d);
      if (oa != 0x7fffffff && (at == 0x7fffffff || o > best || (o == best && oa < at))) { best = o; at = oa; }
    }
    if (lane == (at & 31)) alive &= ~(1u << (at >> 5));
    if (lane == r) mine = at;
  }
  return mine;
}

// One token by one warp: ids and weights.  shared_row: row_doubles(E, groups) doubles, used with groups only.
template <int V>
__device__ __forceinline__ void select_token(const SelectParams& p, int token, int lane, double* shared_row) {
  const size_t row = static_cast<size_t>(token) * p.E;
  const bool softmax = p.score == FMOE_SCORE_SOFTMAX, by_score = p.bias != nullptr || p.groups > 1;
  float v[V], bias[V];
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = lane + 32 * i < p.E ? fp8::fetched(p.bias + lane + 32 * i) : 0.0f;
  }
  load_row<V>(p, row, lane, v);
  float top = -INFINITY;
  if (softmax && (by_score || !p.renormalize)) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, v[i]);
    top = warp_max<float>(top);
  }
  float sum = 1.0f;
  float c[V];   // what is compared
  if (by_score || (softmax && !p.renormalize)) {
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = raw_score<float>(v[i], top, p.score);
      part += c[i];
    }
    if (softmax) sum = warp_sum<float>(part);
  }
  // How far a computed score may be from the true one.  Sigmoid: an exp of 1 ulp below 1 (2^-24), the sum (2^-24) and a
  // quotient of 2 ulp, of a value below 1: 3/2 2^-22.  Softmax: also the rounding of l - max (at most 2^-25 of the
  // largest score: x exp(-x) < 1/2) and a sum of up to 37 additions in a row, all relative to the score, which is at
  // most exp(0) / sum.
  const float error = softmax ? 0x1p-18f / (sum > 0.0f ? sum : 1.0f) : 0x1.8p-22f;
  uint32_t kept = kAll;
  if (by_score) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (softmax && sum > 0.0f) c[i] = __fdividef(c[i], sum);
      if (v[i] == -INFINITY) c[i] = -INFINITY;
      if (p.bias != nullptr) c[i] += sane(bias[i]);
    }
    if (p.groups > 1) {
      float* shared = reinterpret_cast<float*>(shared_row);
      const float per = static_cast<float>(p.groups) / static_cast<float>(p.E);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane + 32 * i < p.E) shared[lane + 32 * i + group_of(lane + 32 * i, per)] = c[i];
      __syncwarp();
      float worst, best;
      kept = kept_groups<float>(group_score<float>(shared, p.E, p.groups, p.group_max, lane), p.groups, p.top_groups, lane,
                                worst, best);
      // a group's sum: two scores, each rounded when its bias was added, and a rounding of its own, none of them over
      // 2^-24 of twice the largest |c|
      float size = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) size = fmaxf(size, c[i] == -INFINITY ? 0.0f : fabsf(c[i]));
      if (worst - best <= 4.0f * error + 0x1p-21f * warp_max<float>(size)) kept = exact_groups<V>(p, row, lane, shared_row);
    }
  }
  const bool by_logit = p.bias == nullptr;
  if (by_logit) {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = v[i];
  }
  const uint32_t alive = alive_bits<V>(p.E, p.groups, kept, lane);
  // this lane's candidates, best first (equal ones in index order); 0: none left
  uint32_t keys[V];
  int at[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    keys[i] = alive >> i & 1 ? order_key(c[i]) : 0;
    at[i] = lane + 32 * i;
  }
  constexpr bool kSorted = V <= 8;   // sorting 16 takes 120 exchanges, more than looking for the best nine times
  if constexpr (kSorted) {
    // odd-even transposition: neighbours only, so equal keys keep their order
#pragma unroll
    for (int pass = 0; pass < V; ++pass)
#pragma unroll
      for (int i = pass & 1; i + 1 < V; i += 2) {
        const bool swap = keys[i + 1] > keys[i];
        const uint32_t hi = swap ? keys[i + 1] : keys[i], lo = swap ? keys[i] : keys[i + 1];
        const int first = swap ? at[i + 1] : at[i], then = swap ? at[i] : at[i + 1];
        keys[i] = hi; keys[i + 1] = lo;
        at[i] = first; at[i + 1] = then;
      }
  }
  uint32_t head = keys[0];
  int head_at = at[0];
  auto find_head = [&] {
    head = keys[0];
    head_at = lane;
#pragma unroll
    for (int i = 1; i < V; ++i)
      if (keys[i] > head) { head = keys[i]; head_at = lane + 32 * i; }
  };
  if constexpr (!kSorted) find_head();
  // Lane r gets the r-th candidate.  By score there is at least one more than k, and more as long as the last two
  // are too close to tell apart (up to the warp's 32).
  int mine = 0, found = 0;
  uint32_t mine_key = 0;
  float last = 0.0f;
  bool close = false, unsure = false;   // some are too close; more than a warp can hold
  for (;; ++found) {
    if (by_logit && found == p.k) break;
    const uint32_t key = __reduce_max_sync(kAll, head);
    if (key == 0) break;                         // every expert is taken
    const int e = __reduce_min_sync(kAll, head == key ? head_at : 0x7fffffff);
    if (!by_logit) {
      const float now = key_value(key);
      const bool near = found > 0 && last - now <= 2.0f * error + 0x1p-23f * fmaxf(fabsf(last), fabsf(now));
      if (found >= p.k && !near) break;          // the chosen ones are known, and no later one is near
      close |= near;
      last = now;
      if (found == 32) { unsure = true; break; }
    }
    if (lane == found) {
      mine = e;
      mine_key = key;
    }
    const bool took = lane == (e & 31);
    if constexpr (kSorted) {
#pragma unroll
      for (int i = 0; i + 1 < V; ++i) {
        keys[i] = took ? keys[i + 1] : keys[i];
        at[i] = took ? at[i + 1] : at[i];
      }
      keys[V - 1] = took ? 0 : keys[V - 1];
      head = keys[0];
      head_at = at[0];
    } else if (took) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i == e >> 5) keys[i] = 0;
      find_head();
    }
  }
  if (unsure) {                                  // (the same for the whole warp, as everything that follows)
    mine = choose_exactly<V>(p, row, lane, kept);
  } else if (close) {
    // the candidates' scores again, in 64 bits, one a lane; each candidate's place is the number that come before it
    double sum64 = 1.0;
    if (softmax) {
      double part = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (v[i] != -INFINITY) part += exp(static_cast<double>(v[i]) - static_cast<double>(top));
      sum64 = warp_sum<double>(part);
    }
    double exact = -INFINITY;
    if (lane < found) {
      const double l = static_cast<double>(logit_at(p, row + mine));
      if (l != -INFINITY) {
        exact = raw_score<double>(l, static_cast<double>(top), p.score);
        if (softmax) exact /= sum64;
        exact += static_cast<double>(sane(fp8::fetched(p.bias + mine)));
      }
    }
    int place = 0;
    for (int j = 0; j < found; ++j) {
      const double o = __shfl_sync(kAll, exact, j);
      const int e = __shfl_sync(kAll, mine, j);
      place += o > exact || (o == exact && e < mine);
    }
    if (lane >= found) place = 32;
    int sorted = 0;
    for (int j = 0; j < found; ++j) {
      const int to = __shfl_sync(kAll, place, j), e = __shfl_sync(kAll, mine, j);
      if (to == lane) sorted = e;
    }
    mine = sorted;
  }
  float l = -INFINITY;
  if (lane < p.k) l = by_logit ? key_value(mine_key) : logit_at(p, row + mine);
  // (shares among the chosen do not depend on the largest of all, which may be far above theirs)
  float s = raw_score<float>(l, p.renormalize ? (by_logit ? __shfl_sync(kAll, l, 0) : warp_max<float>(l)) : top, p.score);
  if (softmax && !p.renormalize && sum > 0.0f) s = s / sum;
  if (p.renormalize) {
    const float total = warp_sum<float>(s);
    s = total > 0.0f ? s / total : 0.0f;
  }
  if (lane < p.k) {
    p.ids[static_cast<size_t>(token) * p.k + lane] = mine;
    p.weights[static_cast<size_t>(token) * p.k + lane] = s * p.scale;
  }
}

__host__ __device__ __forceinline__ size_t row_doubles(int E, int groups) { return groups > 1 ? E + groups : 0; }

template <int V>
__global__ void __launch_bounds__(256) select_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  fp8::wait_for_primary();
  fp8::launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x * 8 + warp;
  if (token < p.S) select_token<V>(p, token, lane, reinterpret_cast<double*>(s_raw) + warp * row_doubles(p.E, p.groups));
}

// ---- ordering ---------------------------------------------------------------------------------------

constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32;
constexpr int kAhead = 8;   // pairs a lane loads before it uses the first

// What is known of pair i: its expert e, its slot there, and the first row of the expert.
__device__ __forceinline__ void place_pair(const SelectParams& p, long long i, int e, int slot, int first_row) {
  if (p.positions != nullptr) p.positions[i] = first_row + slot;
  if (p.table != nullptr) {
    const float w = p.weights[i];
    if (slot < p.capacity)
      p.table[static_cast<size_t>(e) * p.round_ec + slot] = TokenSlot{static_cast<uint32_t>(i / p.k), w};
    p.routes[i] = Route{e, slot, w, 0};
  }
}

// The lanes whose id is this lane's, by one ballot for each of the ids' bits (match.any takes about 1000 cycles for 32
// ids that differ).  id < 0: none.
__device__ __forceinline__ unsigned lanes_alike(int id, int bits) {
  const unsigned here = __ballot_sync(kAll, id >= 0);
  unsigned same = id >= 0 ? here : 0;
#pragma unroll
  for (int b = 0; b < 10; ++b) {
    if (b < bits) {
      const bool one = id >> b & 1;
      const unsigned ones = __ballot_sync(kAll, one);
      same &= one ? ones : ~ones;
    }
  }
  return same;
}

// Stable counting sort of the pairs by expert: the CTAs of one cluster (or one CTA) take consecutive runs of pairs,
// their warps consecutive runs of those.  Pass one counts, pass two hands out places in the same order; in between
// the CTAs' counts meet in distributed shared memory.  (A token's experts differ, so pairs in order are tokens in
// order within an expert.)  What it costs is its chain of steps, so each step has its loads in flight together.
// One CTA per expert that scans all pairs for itself needs no steps but reads the pairs once per expert: 65536 pairs
// of 128 experts took 18 us.
template <int kCtas>
__device__ __forceinline__ void order_pairs(const SelectParams& p, int* hist, bool behind) {
  __shared__ int s_sum[kOrderWarps];
  const int E = p.E, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = kCtas > 1 ? blockIdx.x : 0;     // (the grid is one cluster)
  // hist [warps][E]: counts, then places already handed out
  int* total = hist + kOrderWarps * E;            // [E]: this CTA's pairs
  int* start = total + E;                         // [E]: the expert's first row
  int* base = start + E;                          // [E]: its pairs in the CTAs before this one
  for (int i = threadIdx.x; i < kOrderWarps * E; i += kOrderThreads) hist[i] = 0;
  __syncthreads();
  if (behind) {                                   // the ids are another grid's
    fp8::wait_for_primary();
    fp8::launch_dependents();
  }
  const long long pairs = static_cast<long long>(p.S) * p.k;
  constexpr long long kWorkers = static_cast<long long>(kCtas) * kOrderWarps;
  const long long share = ((pairs + kWorkers - 1) / kWorkers + 31) & ~31ll;
  const long long first = min(pairs, (static_cast<long long>(cta) * kOrderWarps + warp) * share);
  const int n = static_cast<int>(min(pairs, first + share) - first);
  const int32_t* ids = p.ids + first;
  int* mine = hist + warp * E;
  int ahead[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) ahead[j] = i0 + 32 * j + lane < n ? ids[i0 + 32 * j + lane] : -1;
  };
  for (int i0 = 0; i0 < n; i0 += 32 * kAhead) {
    load(i0);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (ahead[j] >= 0) atomicAdd(mine + ahead[j], 1);
  }
  __syncthreads();
  const int e = threadIdx.x;                      // (at most kOrderThreads experts)
  if (e < E) {
    int sum = 0;
#pragma unroll
    for (int w0 = 0; w0 < kOrderWarps; w0 += 16) {
      int c[16];
#pragma unroll
      for (int w = 0; w < 16; ++w) c[w] = hist[(w0 + w) * E + e];
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        hist[(w0 + w) * E + e] = sum;
        sum += c[w];
      }
    }
    total[e] = sum;
  }
  int all = 0, lower = 0;                         // expert e's pairs: of all CTAs, of the CTAs before this one
  if constexpr (kCtas > 1) {
    ptx::cluster_sync_all();
    if (e < E) {
      int c[kCtas];
#pragma unroll
      for (int q = 0; q < kCtas; ++q)
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c[q]) : "r"(ptx::map_to_cta(total + e, q)) : "memory");
#pragma unroll
      for (int q = 0; q < kCtas; ++q) {
        lower += q < cta ? c[q] : 0;
        all += c[q];
      }
    }
  } else if (e < E) {
    all = total[e];
  }
  // exclusive sum over the experts
  int sum = all;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(kAll, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) s_sum[warp] = sum;
  __syncthreads();
  int before = lane < warp ? s_sum[lane] : 0;
  before = __reduce_add_sync(kAll, before);
  if (e < E) {
    const int row = before + sum - all;
    start[e] = row;
    base[e] = lower;
    if (cta == 0) {
      p.counts[e] = all;
      if (p.offsets != nullptr) {
        p.offsets[e] = row;
        if (e == E - 1) p.offsets[E] = row + all;
      }
    }
  }
  __syncthreads();
  const bool once = n <= 32 * kAhead;             // the ids are still in registers
  const int id_bits = 32 - __clz(E - 1);          // (E = 1: no bits)
  const bool placed = p.positions != nullptr || p.table != nullptr;
  for (int i0 = 0; placed && i0 < n; i0 += 32 * kAhead) {
    if (!once) load(i0);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + 32 * j >= n) break;
      const int id = ahead[j];
      const unsigned same = lanes_alike(id, id_bits);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int slot = id >= 0 ? base[id] + mine[id] + rank : 0;
      __syncwarp();
      if (id >= 0 && rank == 0) mine[id] += __popc(same);
      __syncwarp();
      if (id >= 0) place_pair(p, first + i0 + 32 * j + lane, id, slot, start[id]);
    }
  }
  if constexpr (kCtas > 1) ptx::cluster_sync_all();   // no CTA leaves while another reads its totals
}

template <int kCtas>
__global__ void __launch_bounds__(kOrderThreads) order_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  order_pairs<kCtas>(p, reinterpret_cast<int*>(s_raw), true);
}

// Few tokens: one CTA chooses and orders.
template <int V>
__global__ void __launch_bounds__(kOrderThreads) select_few_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  fp8::wait_for_primary();
  fp8::launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int token = warp; token < p.S; token += kOrderWarps)
    select_token<V>(p, token, lane, reinterpret_cast<double*>(s_raw) + warp * row_doubles(p.E, p.groups));
  __syncthreads();
  order_pairs<1>(p, reinterpret_cast<int*>(s_raw), false);
}

template <typename Kernel>
cudaError_t launch(Kernel kernel, const SelectParams& p, int grid, int threads, size_t smem, int cluster, cudaStream_t stream) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return fp8::launch_behind(kernel, dim3(grid), threads, smem, cluster, stream, p);
}

// Up to this many tokens one CTA does it all, in two rounds of its 32 warps, for want of a second launch (one token: 10.3
// us by two launches, 6.2 by one).
constexpr int kFewTokens = 64;

template <int V>
cudaError_t launch_select(const SelectParams& p, cudaStream_t stream) {
  const size_t group_row = row_doubles(p.E, p.groups) * sizeof(double);
  const size_t order = static_cast<size_t>(kOrderWarps + 3) * p.E * sizeof(int);
  if constexpr (V <= 8) {   // (the registers of 32 warps)
    if (p.S <= kFewTokens) {
      const size_t rows = kOrderWarps * group_row;
      return launch(select_few_kernel<V>, p, 1, kOrderThreads, rows > order ? rows : order, 1, stream);
    }
  }
  if (p.S > 0) {
    const cudaError_t e = launch(select_kernel<V>, p, (p.S + 7) / 8, 256, 8 * group_row, 1, stream);
    if (e != cudaSuccess) return e;
  }
  // (both kernels, 65536 pairs of 128 experts: 18.5 us by 8 CTAs, 16.4 by 16; 16384 pairs of 256 experts: 15.1 and 14.4)
  const long long pairs = static_cast<long long>(p.S) * p.k;
  if (pairs <= kOrderThreads) return launch(order_kernel<1>, p, 1, kOrderThreads, order, 1, stream);
  const cudaError_t e = cudaFuncSetAttribute(order_kernel<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  return launch(order_kernel<16>, p, 16, kOrderThreads, order, 16, stream);
}

int check(const fmoe_select_args* a) {
  if (a == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "arguments are null");
  if (a->num_tokens < 0) return set_error(FMOE_ERR_INVALID_ARG, "num_tokens must not be negative");
  if (a->num_experts < 1 || a->num_experts > kMaxExperts)
    return set_error(FMOE_ERR_INVALID_ARG, "num_experts must be between 1 and " + std::to_string(kMaxExperts));
  if (a->num_groups < 1 || a->num_groups > kMaxGroups || a->num_experts % a->num_groups != 0)
    return set_error(FMOE_ERR_INVALID_ARG, "num_groups must divide num_experts and be at most " + std::to_string(kMaxGroups));
  if (a->top_groups < 1 || a->top_groups > a->num_groups)
    return set_error(FMOE_ERR_INVALID_ARG, "top_groups must be between 1 and num_groups");
  if (a->top_k < 1 || a->top_k > kMaxTopK || a->top_k > a->top_groups * (a->num_experts / a->num_groups))
    return set_error(FMOE_ERR_INVALID_ARG, "top_k must not exceed the experts of top_groups groups (or 32)");
  if (a->score != FMOE_SCORE_SOFTMAX && a->score != FMOE_SCORE_SIGMOID)
    return set_error(FMOE_ERR_INVALID_ARG, "unknown score");
  if (a->group_score != FMOE_GROUP_TOP2 && a->group_score != FMOE_GROUP_MAX)
    return set_error(FMOE_ERR_INVALID_ARG, "unknown group_score");
  if (a->data_type != FMOE_DT_BF16 && a->data_type != FMOE_DT_FP16 && a->data_type != FMOE_DT_FP32)
    return set_error(FMOE_ERR_UNSUPPORTED, "logits are BF16, FP16 or FP32");
  if (a->device_id < 0 || a->device_id >= fp8::kMaxDevices) return set_error(FMOE_ERR_INVALID_ARG, "device_id out of range");
  if (static_cast<long long>(a->num_tokens) * a->top_k > 0x7fffffffll)
    return set_error(FMOE_ERR_UNSUPPORTED, "num_tokens * top_k must fit 32 bits");
  if (a->expert_counts == nullptr || (a->num_tokens > 0 && (a->logits == nullptr || a->ids == nullptr || a->weights == nullptr)))
    return set_error(FMOE_ERR_INVALID_ARG, "logits, ids, weights and expert_counts are required");
  if (fp8::misaligned(a->logits, fp8::element_bytes(a->data_type)) || fp8::misaligned(a->bias, 4) || fp8::misaligned(a->ids, 4) ||
      fp8::misaligned(a->weights, 4) || fp8::misaligned(a->expert_counts, 4) || fp8::misaligned(a->offsets, 4) ||
      fp8::misaligned(a->positions, 4))
    return set_error(FMOE_ERR_INVALID_ARG, "every array must be aligned to its type");
  return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

extern "C" int fmoe_router_select(fmoe_ctx* moe, const fmoe_select_args* a, void* stream) {
  using namespace fmoe;
  int rc = check(a);
  if (rc != FMOE_OK) return rc;
  SelectParams p{};
  if (moe != nullptr) {
    rc = routing_targets(moe, a->num_tokens, a->num_experts, a->top_k, a->device_id, &p.table, &p.routes, &p.capacity, &p.round_ec);
    if (rc != FMOE_OK) return rc;
  }
  p.logits = a->logits; p.bias = a->bias; p.ids = a->ids; p.weights = a->weights;
  p.counts = a->expert_counts; p.offsets = a->offsets; p.positions = a->positions;
  p.S = a->num_tokens; p.E = a->num_experts; p.k = a->top_k; p.dtype = a->data_type; p.score = a->score;
  p.groups = a->top_groups == a->num_groups ? 1 : a->num_groups;   // every group stays: as if there were none
  p.top_groups = p.groups == 1 ? 1 : a->top_groups;
  p.group_max = a->group_score == FMOE_GROUP_MAX;
  p.renormalize = a->renormalize != 0; p.scale = a->scale;
  fp8::OnDevice on(a->device_id);
  if (on.err != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(on.err));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (p.E <= 32) e = launch_select<1>(p, st);
  else if (p.E <= 64) e = launch_select<2>(p, st);
  else if (p.E <= 128) e = launch_select<4>(p, st);
  else if (p.E <= 256) e = launch_select<8>(p, st);
  else if (p.E <= 512) e = launch_select<16>(p, st);
  else e = launch_select<32>(p, st);
  if (e != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("select launch: ") + cudaGetErrorString(e));
  return FMOE_OK;
}
