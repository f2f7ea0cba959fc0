// Routing of tokens to experts: scores, balance bias, groups, the top_k choice and its weights (the router
// step in front of the fused-experts call, hi2/moe.py:53-121).
//
// One warp per token, expert 32 i + lane in element i of a lane.  A choice is one maximum over the lanes
// (redux.sync on order-preserving integer keys) and one minimum over the indices of those that hold it, so
// equal keys go to the lowest index.  Without a bias the keys are the logits themselves (both scores
// grow with the logit); with one, or with groups, scores are formed in fp64, since two biased scores that
// agree to the last fp32 bits must still be told apart the way their exact values are.
//
// What bounds it: with groups the integer pipe (64 % busy in a capture before the keys were compared as fp64, 1343 instructions
// per token): 16384 tokens of 128 experts in 8 groups take 24.6 us a call, 23.1 replayed (a call 28.9 with 64-bit integer keys and a division per expert).
// A single token takes 2.5 us, one launch.
#include <type_traits>

#include "common.cuh"

namespace hi2 {
namespace {

constexpr int ROUTE_WARPS = 4;
constexpr uint32_t ALL = 0xffffffffu;

struct RouteParams {
  const void* logits;
  const float* bias;
  int64_t tokens, ld;
  int64_t* index;
  float* weight;
  float scale;
  int dtype, experts, top_k, sigmoid, groups, top_groups, renormalise;
  int team_log;              // lanes that read through a group: as many as the groups leave, a power of two
  uint32_t per, per_inverse; // experts of a group; e / per = e * per_inverse >> 20 for e < 1024 (per * per_inverse < 2^20 + per)
};

// Order-preserving integers; 0 is below every number and marks a closed expert.  -0 counts as 0.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}
// Keys in fp64 are compared as they are, on a pipe that has the time, and become integers for the lanes' maximum only;
// -inf marks a closed expert there.
constexpr double CLOSED = -INFINITY;
__device__ __forceinline__ uint64_t order_of(double key) { return key > CLOSED ? key_of(key) : 0; }
__device__ __forceinline__ uint32_t order_of(uint32_t key) { return key; }
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(ALL, v); }
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(ALL, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(ALL, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}

// Whether a key is left; if so the lowest index of the largest of the lanes' keys (PER each), which is cleared.
template <int PER, typename KEY>
__device__ __forceinline__ bool take_best(KEY (&key)[PER], int lane, uint32_t& at) {
  KEY best = key[0];
  int mine = 0;
#pragma unroll
  for (int i = 1; i < PER; ++i)
    if (key[i] > best) best = key[i], mine = i;
  const auto order = order_of(best), top = warp_max(order);
  at = __reduce_min_sync(ALL, order == top ? (uint32_t)(mine * 32 + lane) : ALL);
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (at == (uint32_t)(i * 32 + lane)) key[i] = std::is_same<KEY, double>::value ? (KEY)CLOSED : (KEY)0;
  return top != 0;
}

// The top_k best keys: lane r ends up with the r-th choice's index (-1: none) and score.
template <int PER, typename KEY, typename SCORE>
__device__ __forceinline__ void choose(KEY (&key)[PER], const SCORE* score, int top_k, int lane, int& index, SCORE& chosen, SCORE& sum) {
  index = -1, chosen = 0, sum = 0;
  for (int r = 0; r < top_k; ++r) {
    uint32_t at;
    if (!take_best(key, lane, at)) return;  // no open expert is left
    const SCORE s = score[at];
    sum += s;
    if (lane == r) index = (int)at, chosen = s;
  }
}

template <int PER, bool EXACT_KEYS>
__global__ void __launch_bounds__(ROUTE_WARPS * 32)
route_kernel(const RouteParams p) {
  typedef typename std::conditional<EXACT_KEYS, double, float>::type SCORE;
  __shared__ union {  // a token's scores; before them, where experts form groups, its keys
    SCORE scores[PER * 32];
    double keys[EXACT_KEYS ? PER * 32 : 1];
  } shared[ROUTE_WARPS];
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  float logit[PER];
  uint32_t open = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    float v = -INFINITY;
    if (e < p.experts) {
      const int64_t at = token * p.ld + e;
      v = p.dtype == HI2_F32 ? static_cast<const float*>(p.logits)[at]
          : p.dtype == HI2_F16 ? __half2float(static_cast<const __half*>(p.logits)[at])
                               : __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[at]);
    }
    bool usable = v > -INFINITY;
    if (p.bias != nullptr && e < p.experts) usable = usable && p.bias[e] > -INFINITY;
    open |= (usable ? 1u : 0u) << i;
    logit[i] = fminf(v, 3.402823466e38f);  // +inf counts as the largest number
  }
  SCORE score[PER];
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) score[i] = (SCORE)1 / ((SCORE)1 + exp(-(SCORE)logit[i]));
  } else {
    float top = -3.402823466e38f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (open >> i & 1) top = fmaxf(top, logit[i]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, d));
    SCORE sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      score[i] = open >> i & 1 ? exp((SCORE)logit[i] - (SCORE)top) : (SCORE)0;
      sum += score[i];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(ALL, sum, d);
    if (sum > 0)
#pragma unroll
      for (int i = 0; i < PER; ++i) score[i] /= sum;
  }
  SCORE* const of = shared[threadIdx.x >> 5].scores;
  int index;
  SCORE chosen, sum;
  if (EXACT_KEYS) {
    double key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 + lane;
      const double b = p.bias != nullptr && e < p.experts ? (double)p.bias[e] : 0.0;
      key[i] = open >> i & 1 ? (double)score[i] + b : CLOSED;
    }
    if (p.groups > 1) {
      // Several lanes read through a group each, and find its two best keys together.
      double* const all = shared[threadIdx.x >> 5].keys;
#pragma unroll
      for (int i = 0; i < PER; ++i) all[i * 32 + lane] = key[i];
      __syncwarp();
      const int team = 1 << p.team_log, per = (int)p.per, mine = lane >> p.team_log;
      double first = CLOSED, second = CLOSED;
      if (mine < p.groups)
        for (int e = mine * per + (lane & (team - 1)); e < (mine + 1) * per; e += team) {
          const double k = all[e];
          if (k > first) second = first, first = k;
          else if (k > second) second = k;
        }
      for (int d = team >> 1; d > 0; d >>= 1) {
        const double f = __shfl_xor_sync(ALL, first, d), s = __shfl_xor_sync(ALL, second, d);
        const double low = first < f ? first : f, high = second > s ? second : s;
        first = first < f ? f : first;
        second = low > high ? low : high;
      }
      double total = second > CLOSED ? first + second : first;
      total = __shfl_sync(ALL, total, (lane << p.team_log) & 31);  // lane q: the key of group q
      if (lane >= p.groups) total = CLOSED;
      uint32_t kept = 0;
      double of_group[1] = {total};
      for (int r = 0; r < p.top_groups; ++r) {
        uint32_t q;
        if (take_best(of_group, lane, q)) kept |= 1u << q;
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = i * 32 + lane;
        if (!(kept >> ((uint32_t)e * p.per_inverse >> 20 & 31) & 1)) key[i] = CLOSED;  // (those behind the last are closed already)
      }
    }
    if (p.bias == nullptr) {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = key[i] > CLOSED ? (double)logit[i] : CLOSED;
    }
    __syncwarp();  // the keys have been read
#pragma unroll
    for (int i = 0; i < PER; ++i) of[i * 32 + lane] = score[i];
    __syncwarp();
    choose(key, of, p.top_k, lane, index, chosen, sum);
  } else {
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) of[i * 32 + lane] = score[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = open >> i & 1 ? key_of(logit[i]) : 0;
    choose(key, of, p.top_k, lane, index, chosen, sum);
  }
  if (lane < p.top_k) {
    if (p.renormalise) chosen /= sum > (SCORE)1e-20f ? sum : (SCORE)1e-20f;
    p.index[token * p.top_k + lane] = index;
    p.weight[token * p.top_k + lane] = (float)(chosen * (SCORE)p.scale);
  }
}

template <int PER>
void launch(const RouteParams& p, bool exact, unsigned grid, cudaStream_t s) {
  if (exact) route_kernel<PER, true><<<grid, ROUTE_WARPS * 32, 0, s>>>(p);
  else route_kernel<PER, false><<<grid, ROUTE_WARPS * 32, 0, s>>>(p);
}

}  // namespace
}  // namespace hi2

extern "C" int hi2_route(const void* logits, int dtype, int64_t tokens, int experts, int64_t ld, int top_k, int sigmoid,
                         const float* bias, int groups, int top_groups, int renormalise, float scale, int64_t* index,
                         float* weight, void* stream) {
  using namespace hi2;
  HI2_REQUIRE(dtype == HI2_F32 || dtype == HI2_F16 || dtype == HI2_BF16, "route: logits must be fp32, fp16 or bf16");
  HI2_REQUIRE(experts >= 1 && experts <= 1024, "route: 1 to 1024 experts");
  HI2_REQUIRE(top_k >= 1 && top_k <= 32 && top_k <= experts, "route: top_k must be 1 to min(experts, 32)");
  HI2_REQUIRE(groups >= 1 && groups <= 32 && experts % groups == 0, "route: up to 32 groups of equal size");
  HI2_REQUIRE(top_groups >= 1 && top_groups <= groups, "route: top_groups must be 1 to groups");
  HI2_REQUIRE(tokens >= 0 && tokens < (int64_t)1 << 31, "route: too many tokens");
  if (tokens == 0) return HI2_OK;
  HI2_REQUIRE(logits && index && weight, "route: null pointer");
  int team_log = 5;
  while (groups << team_log > 32) --team_log;
  const uint32_t per = (uint32_t)(experts / groups);
  const RouteParams p{logits, bias, tokens, ld, index, weight, scale, dtype, experts, top_k, sigmoid, groups, top_groups, renormalise,
                      team_log, per, ((1u << 20) + per - 1) / per};
  const bool exact = bias != nullptr || groups > 1;
  const unsigned grid = (unsigned)ceil_div(tokens, (int64_t)ROUTE_WARPS);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (experts <= 32) launch<1>(p, exact, grid, s);
  else if (experts <= 64) launch<2>(p, exact, grid, s);
  else if (experts <= 128) launch<4>(p, exact, grid, s);
  else if (experts <= 256) launch<8>(p, exact, grid, s);
  else if (experts <= 512) launch<16>(p, exact, grid, s);
  else launch<32>(p, exact, grid, s);
  return check_launch("route");
}
