// Choosing experts: scores, a balance bias, expert groups, top-k, weights, and
// the gradient of the weights (cvmm_router_select, cvmm_router_select_backward).
//
//   s = softmax(z) or 1 / (1 + exp(-z))                    z: a token's logits
//   c = s + b        (no bias: the order of z, which s grows with)
//   group value = max c, or the sum of the two largest c, of its experts
//   sel = the k largest c within the top_groups best groups, descending,
//         ties to the lowest index; z = -inf ranks below every other expert
//   w_j = scale * s_j / max(sum_i s_i, 1e-20)              (or scale * s_j)
//
// An order must not depend on how exp rounds, so it is that of c in 64 bits.
// Computing every c in 64 bits would cost more than all the rest; instead the
// order is taken from 32-bit values whose error is bounded, every pair of
// neighbours in it is checked against that bound, and only a token with a pair
// nearer than the bound (about one in a thousand) is decided again in 64 bits.
#include "common.cuh"
#include "launch.h"

namespace cvmm {
namespace router {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;    // lane j of a warp holds the j-th chosen expert
constexpr int kMaxGroups = 32;  // lane g of a warp holds (or shares) group g
constexpr int kWarps = 4;
constexpr int kBadSelTag = 30;  // status-word site: a chosen id outside [0, n_experts)

// How far the difference of two 32-bit values may be from the exact one. expf
// is within 2 ulp (2.4e-7 relative). Softmax, in units of the largest score
// 1 / sum: the argument's half ulp gives x e^-x 6e-8 <= 2.2e-8, expf 2.4e-7 and
// the division 6e-8 for each of the two; the sum's error scales the whole
// difference, which is at most one unit: NPER additions in a lane and 5 across
// at 6e-8 and its terms' 2.4e-7. Sigmoid: s (1 - s) 2.4e-7 + 1.2e-7 s for each.
// c = s + b adds half an ulp of each c.
template <int NPER>
__device__ __forceinline__ float pair_error(bool softmax, float smax) {
  return softmax ? smax * (1e-6f + 6e-8f * (NPER + 5)) : 6e-7f;
}
constexpr float kAddErr = 6e-8f;   // relative, of c
constexpr float kTinyErr = 1e-38f; // scores below the normal range

enum Scoring : int { kSoftmax = CVMM_SCORE_SOFTMAX, kSigmoid = CVMM_SCORE_SIGMOID };

struct Args {
  const void* logits;
  int dtype;
  int64_t ld, T;
  int E, k, scoring;
  const void* bias;  // [E] or null
  int bias_dtype;
  int G, top_groups, top2;
  uint32_t size_inv;  // ceil(2^22 / experts of a group)
  int renorm;
  float scale;
  int64_t* sel;
  float* weights;
};

// Orders floats as unsigned integers: NaN above everything, -inf at 0x007fffff,
// so that 0 is free for "not a candidate". -0 and +0 get one key.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The same order for doubles (64-bit keys), for the rare second decision.
__device__ __forceinline__ unsigned long long key_of(double v) {
  if (v != v) return ~0ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// 1 / (1 + exp(-z)) without overflow: exp of -|z| only.
__device__ __forceinline__ float sigmoid(float z) {
  const float e = expf(-fabsf(z));
  return (z < 0.f ? e : 1.f) / (1.f + e);
}

// The value of a key: the inverse of key_of up to the sign of zero and NaN bits.
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// Largest over the warp in one integer reduction; NaN only if every value is (as fmaxf).
__device__ __forceinline__ float warp_max(float v) {
  return value_of(__reduce_max_sync(0xffffffffu, v != v ? 0u : key_of(v)));
}

// Two largest values of a group, in key order, and their keys.
template <typename R>
struct Top2 {
  R a = -(R)INFINITY, b = -(R)INFINITY;
  __device__ __forceinline__ void add(R v) {
    // NaN (above everything) compares false both ways: `!(v <= a)` takes it.
    if (!(v <= a) && a == a) { b = a; a = v; }
    else if (!(v <= b) && b == b) b = v;
  }
};

// The top_groups best of p.G groups of `size` consecutive values v[e], as bits:
// 32 / (G rounded up to a power of two) lanes share a group. worst and other:
// the lowest chosen and the highest other group value (NaN if all are chosen).
template <typename R>
__device__ __forceinline__ uint32_t best_groups(const Args& p, const R* v, int size, R& worst, R& other) {
  const int lane = threadIdx.x & 31, lanes = 32 >> (32 - __clz(p.G - 1));
  const int g = lane / lanes;
  Top2<R> top;
  if (g < p.G)
    for (int m = lane % lanes; m < size; m += lanes) top.add(v[g * size + m]);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    const R oa = __shfl_xor_sync(0xffffffffu, top.a, o), ob = __shfl_xor_sync(0xffffffffu, top.b, o);
    top.add(oa);
    top.add(ob);
  }
  // A masked (-inf) second counts as nothing.
  const R gv = p.top2 && top.b != -(R)INFINITY ? top.a + top.b : top.a;
  const auto mine = g < p.G ? key_of(gv) : 0;
  int rank = 0;
  uint32_t chosen = 0;
  for (int o = 0; o < p.G; ++o) {
    const auto k = __shfl_sync(0xffffffffu, mine, o * lanes);
    rank += k > mine || (k == mine && o < g);
  }
  const uint32_t in = __ballot_sync(0xffffffffu, g < p.G && rank < p.top_groups);
  for (int o = 0; o < p.G; ++o) chosen |= ((in >> (o * lanes)) & 1u) << o;
  // Ranks are a permutation: exactly one group has each.
  const uint32_t lo = __ballot_sync(0xffffffffu, g < p.G && rank == p.top_groups - 1);
  const uint32_t hi = __ballot_sync(0xffffffffu, g < p.G && rank == p.top_groups);
  worst = __shfl_sync(0xffffffffu, gv, __ffs(lo) - 1);
  other = hi ? __shfl_sync(0xffffffffu, gv, __ffs(hi) - 1) : (R)NAN;
  return chosen;
}

// e / size for e < 1024: with m = ceil(2^22 / size), e m / 2^22 is at most 2^-12
// above e / size, less than the 1 / size to the next whole number.
__device__ __forceinline__ int group_of(const Args& p, int e) { return (int)((uint32_t)e * p.size_inv >> 22); }

__device__ __forceinline__ float logit(const Args& p, int64_t t, int e) {
  return load_as_float(p.logits, p.dtype, t * p.ld + e);
}

// Decides token t again with 64-bit scores, kept in the warp's shared memory v
// (E doubles). Lane j < k returns the j-th expert.
__device__ __noinline__ int decide_in_64(const Args& p, int64_t t, double* v) {
  const int lane = threadIdx.x & 31;
  const bool softmax = p.scoring == kSoftmax;
  double mx = 0.0, sum = 1.0;
  if (softmax) {
    float m = -INFINITY;
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, logit(p, t, e));
    mx = warp_max(m);
    if (mx == -(double)INFINITY) mx = 0.0;
    sum = 0.0;
  }
  for (int e = lane; e < p.E; e += 32) {
    const double z = logit(p, t, e);
    v[e] = softmax ? exp(z - mx) : 1.0 / (1.0 + exp(-z));
    if (softmax) sum += v[e];
  }
  if (softmax) {
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum == 0.0) sum = 1.0;
  }
  for (int e = lane; e < p.E; e += 32) {
    const double c = v[e] / sum + (p.bias ? (double)load_as_float(p.bias, p.bias_dtype, e) : 0.0);
    v[e] = logit(p, t, e) == -INFINITY ? -(double)INFINITY : c;
  }
  __syncwarp();
  uint32_t groups = 0xffffffffu;
  if (p.G > 1) {
    double worst, other;
    groups = best_groups(p, v, p.E / p.G, worst, other);
  }
  uint32_t out = 0;  // bit q: expert lane + 32 q is taken or in no chosen group
  for (int q = 0; lane + 32 * q < p.E; ++q)
    if (p.G > 1 && !((groups >> group_of(p, lane + 32 * q)) & 1u)) out |= 1u << q;
  int chosen = 0;
  for (int j = 0; j < p.k; ++j) {
    unsigned long long best = 0;
    int be = 0x7fffffff;
    for (int q = 0; lane + 32 * q < p.E; ++q) {
      if ((out >> q) & 1u) continue;
      const int e = lane + 32 * q;
      const unsigned long long key = key_of(p.bias ? v[e] : (double)logit(p, t, e));
      if (key > best) { best = key; be = e; }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int oe = __shfl_xor_sync(0xffffffffu, be, o);
      if (ov > best || (ov == best && oe < be)) { best = ov; be = oe; }
    }
    if ((be & 31) == lane) out |= 1u << (be >> 5);
    if (lane == j) chosen = be;
  }
  return chosen;
}

// The row of logits of token t in registers: lane l holds experts l + 32 q.
template <int NPER>
__device__ __forceinline__ void load_row(float (&z)[NPER], const void* logits, int dtype, int64_t at, int E) {
  const int lane = threadIdx.x & 31;
  if (dtype == F32) {
#pragma unroll
    for (int q = 0; q < NPER; ++q)
      z[q] = lane + 32 * q < E ? static_cast<const float*>(logits)[at + lane + 32 * q] : -INFINITY;
    return;
  }
  uint16_t h[NPER];
#pragma unroll
  for (int q = 0; q < NPER; ++q)
    h[q] = lane + 32 * q < E ? static_cast<const uint16_t*>(logits)[at + lane + 32 * q] : 0;
#pragma unroll
  for (int q = 0; q < NPER; ++q) z[q] = lane + 32 * q < E ? bits_to_float(h[q], dtype) : -INFINITY;
}

// One warp a token; lane l holds experts l, l + 32, ... (NPER of them) and
// keeps the largest of its keys. A round of the top-k is the largest key over
// the warp, then the lowest index that has it, each one warp-wide integer
// reduction; only the lane that gave the expert looks for its next largest.
// BIAS and GROUPS leave out what a call without them does not do.
template <int NPER, bool BIAS, bool GROUPS>
__global__ void __launch_bounds__(kWarps * 32) select_kernel(const __grid_constant__ Args p) {
  pdl_enter();
  extern __shared__ double sh[];  // per warp E doubles (BIAS or GROUPS only)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x * (int64_t)kWarps + warp;
  if (t >= p.T) return;
  const int E = p.E;
  const bool softmax = p.scoring == kSoftmax;
  float z[NPER], b[NPER];
  load_row(z, p.logits, p.dtype, t * p.ld, E);
  if (BIAS) {
#pragma unroll
    for (int q = 0; q < NPER; ++q) b[q] = lane + 32 * q < E ? load_as_float(p.bias, p.bias_dtype, lane + 32 * q) : 0.f;
  }
  float mx = 0.f, sum = 1.f;
  float s[NPER];
  if (softmax) {
    mx = z[0];
#pragma unroll
    for (int q = 1; q < NPER; ++q) mx = fmaxf(mx, z[q]);
    mx = warp_max(mx);
    if (mx == -INFINITY || mx != mx) mx = 0.f;  // every expert masked: all scores are 0
    sum = 0.f;
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      s[q] = expf(z[q] - mx);
      sum += lane + 32 * q < E ? s[q] : 0.f;
    }
    sum = warp_sum(sum);
    if (sum == 0.f) sum = 1.f;
  }
  const float smax = softmax ? 1.f / sum : 1.f;  // no score is above this
  const float err = pair_error<NPER>(softmax, smax);
  if (BIAS || (GROUPS && p.top2)) {
#pragma unroll
    for (int q = 0; q < NPER; ++q) s[q] = softmax ? s[q] / sum : sigmoid(z[q]);
  }
  uint32_t key[NPER];
#pragma unroll
  for (int q = 0; q < NPER; ++q)
    key[q] = lane + 32 * q < E ? key_of(BIAS && z[q] != -INFINITY ? s[q] + b[q] : z[q]) : 0u;
  bool again = false;
  if (GROUPS) {
    float* v = reinterpret_cast<float*>(sh + warp * E);
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      const int e = lane + 32 * q;
      if (e < E) v[e] = BIAS ? (z[q] == -INFINITY ? z[q] : s[q] + b[q]) : p.top2 && z[q] != -INFINITY ? s[q] : z[q];
    }
    __syncwarp();
    float worst, other;
    const uint32_t groups = best_groups(p, v, E / p.G, worst, other);
    __syncwarp();
    // The worst chosen and the best other group must differ by more than the error of both.
    if (BIAS || p.top2)
      again = other > -INFINITY &&
              worst - other <= 2.f * err + 4.f * kAddErr * (fabsf(worst) + fabsf(other)) + kTinyErr;
#pragma unroll
    for (int q = 0; q < NPER; ++q)
      if (!((groups >> group_of(p, lane + 32 * q)) & 1u)) key[q] = 0u;
  }
  uint32_t best = 0;
  int bq = 0;
  auto local_best = [&]() {
    best = key[0];
    bq = 0;
#pragma unroll
    for (int q = 1; q < NPER; ++q)
      if (key[q] > best) {
        best = key[q];
        bq = q;
      }
  };
  local_best();
  int chosen = 0, last = 0;
  float pc = 0.f;  // the value of the expert before
  const int n_cand = GROUPS ? p.top_groups * (E / p.G) : E;
  // With a bias one more expert is looked at, to see that it is clearly lower than the k-th.
  int rounds = BIAS ? min(p.k + 1, n_cand) : p.k;
  for (int j = 0; j < rounds && !again; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const int be = (int)__reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(lane + 32 * bq) : 0xffffffffu);
    if (BIAS) {
      // Neighbours nearer than their errors are decided again, unless they
      // have equal logits and biases and so are equal in any number of bits.
      const float c = value_of(top);
      if (j > 0 && c > -INFINITY && pc - c <= err + kAddErr * (fabsf(pc) + fabsf(c)) + kTinyErr) {
        again = logit(p, t, be) != logit(p, t, last) ||
                load_as_float(p.bias, p.bias_dtype, be) != load_as_float(p.bias, p.bias_dtype, last);
        if (j >= p.k) rounds = min(rounds + 1, n_cand);  // one equal to the k-th: look at the next, too
      }
      pc = c;
      last = be;
    }
    if (lane == (be & 31)) {
#pragma unroll
      for (int q = 0; q < NPER; ++q)
        if (q == bq) key[q] = 0u;
      local_best();
    }
    if (lane == j) chosen = be;
  }
  if ((BIAS || GROUPS) && again) chosen = decide_in_64(p, t, sh + warp * E);
  float score = 0.f;
  if (lane < p.k) {
    const float zc = logit(p, t, chosen);
    score = softmax ? expf(zc - mx) / sum : sigmoid(zc);
  }
  const float tot = warp_sum(score);
  if (lane < p.k) {
    const float held = tot < 1e-20f ? 1e-20f : tot;
    p.sel[t * p.k + lane] = chosen;
    p.weights[t * p.k + lane] = p.scale * (p.renorm ? score / held : score);
  }
}

// d w / d z. With S = max(sum s_j, 1e-20) and g the weights' gradient:
//   gs_j = scale (g_j - sum_i g_i s_i / S) / S   (no sum term where S is held; scale g_j without renormalising)
//   softmax: gz_e = s_e (gs_e - sum_j s_j gs_j)      sigmoid: gz_e = gs_e s_e (1 - s_e)
// with gs_e = 0 off the chosen experts. One warp a token writes the row once
// and then the chosen entries over it.
template <int NPER>
__global__ void __launch_bounds__(kWarps * 32)
select_backward_kernel(const void* __restrict__ logits, int dtype, int64_t ld, const int64_t* __restrict__ sel,
                       const float* __restrict__ grad_w, int64_t T, int E, int k, int scoring, int renorm, float scale,
                       void* __restrict__ grad_logits) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x * (int64_t)kWarps + (threadIdx.x >> 5);
  if (t >= T) return;
  const bool softmax = scoring == kSoftmax;
  int64_t e = -1;
  float g = 0.f;
  if (lane < k) {
    e = sel[t * k + lane];
    g = scale * grad_w[t * k + lane];
    if (e < 0 || e >= E) {
      report(CVMM_DEV_BAD_INDEX, kBadSelTag, (long long)e);
      e = -1;
    }
  }
  float s[NPER];
  float mx = 0.f, inv = 1.f;
  if (softmax) {
    load_row(s, logits, dtype, t * ld, E);
    mx = s[0];
#pragma unroll
    for (int q = 1; q < NPER; ++q) mx = fmaxf(mx, s[q]);
    mx = warp_max(mx);
    if (mx == -INFINITY || mx != mx) mx = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      s[q] = expf(s[q] - mx);
      sum += lane + 32 * q < E ? s[q] : 0.f;
    }
    sum = warp_sum(sum);
    inv = sum == 0.f ? 1.f : 1.f / sum;
  }
  float sj = 0.f, rest = 0.f;  // rest: 1 - s, from the other side
  if (e >= 0) {
    const float z = load_as_float(logits, dtype, t * ld + e);
    sj = softmax ? expf(z - mx) * inv : sigmoid(z);
    rest = sigmoid(-z);
  } else {
    g = 0.f;
  }
  if (renorm) {
    const float tot = warp_sum(sj), gs = warp_sum(g * sj);
    const float held = tot < 1e-20f ? 1e-20f : tot;
    g = (g - (tot < 1e-20f ? 0.f : gs / held)) / held;
  }
  const float dot = softmax ? warp_sum(e >= 0 ? sj * g : 0.f) : 0.f;
#pragma unroll
  for (int q = 0; q < NPER; ++q) {
    const int c = lane + 32 * q;
    if (c < E) store_from_float(grad_logits, dtype, t * E + c, softmax ? -s[q] * inv * dot : 0.f);
  }
  __syncwarp();
  if (e >= 0)
    store_from_float(grad_logits, dtype, t * E + e, softmax ? sj * (g - dot) : g * sj * rest);
}

template <typename F>
static int with_nper(int64_t E, F f) {
  if (E <= 32) return f(std::integral_constant<int, 1>());
  if (E <= 64) return f(std::integral_constant<int, 2>());
  if (E <= 128) return f(std::integral_constant<int, 4>());
  if (E <= 256) return f(std::integral_constant<int, 8>());
  if (E <= 512) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}

}  // namespace router
}  // namespace cvmm

extern "C" int cvmm_router_select(const void* logits, int logits_dtype, int64_t logits_ld, int64_t n_tokens,
                                  int64_t n_experts, int64_t top_k, int scoring, const void* bias, int bias_dtype,
                                  int64_t n_groups, int64_t top_groups, int group_score, int renormalize, float scale,
                                  int64_t* sel, float* weights, cvmm_stream_t stream) {
  using namespace cvmm;
  if (!is_float_dtype(logits_dtype) || (bias && !is_float_dtype(bias_dtype)))
    return fail(CVMM_ERR_UNSUPPORTED_DTYPE, "cvmm_router_select: unsupported dtype");
  if (scoring != CVMM_SCORE_SOFTMAX && scoring != CVMM_SCORE_SIGMOID)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select: scoring must be softmax or sigmoid");
  if (group_score != CVMM_GROUP_MAX && group_score != CVMM_GROUP_TOP2)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select: group_score must be max or top2");
  if (n_tokens < 0 || n_experts <= 0 || n_experts > router::kMaxExperts || logits_ld < n_experts)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select: needs 1 <= n_experts <= 1024 and logits_ld >= n_experts");
  if (n_groups < 1 || n_groups > router::kMaxGroups || n_experts % n_groups != 0 || top_groups < 1 ||
      top_groups > n_groups)
    return fail(CVMM_ERR_INVALID_ARG,
                "cvmm_router_select: needs 1 <= top_groups <= n_groups <= 32 and n_experts a multiple of n_groups");
  if (top_k < 1 || top_k > router::kMaxTopK || top_k > n_experts / n_groups * top_groups)
    return fail(CVMM_ERR_INVALID_ARG,
                "cvmm_router_select: needs 1 <= top_k <= min(32, the experts of top_groups groups)");
  if (n_tokens == 0) return CVMM_OK;
  if (n_tokens > (int64_t)INT32_MAX) return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select: more than 2^31 tokens");
  if (!logits || !sel || !weights) return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select: null pointer");
  router::Args p = {};
  p.logits = logits; p.dtype = logits_dtype; p.ld = logits_ld; p.T = n_tokens;
  p.E = (int)n_experts; p.k = (int)top_k; p.scoring = scoring;
  p.bias = bias; p.bias_dtype = bias_dtype;
  p.G = (int)n_groups; p.top_groups = (int)top_groups; p.top2 = group_score == CVMM_GROUP_TOP2;
  const int64_t size = n_experts / n_groups;
  p.size_inv = (uint32_t)((((int64_t)1 << 22) + size - 1) / size);
  p.renorm = renormalize; p.scale = scale; p.sel = sel; p.weights = weights;
  const unsigned grid = (unsigned)((n_tokens + router::kWarps - 1) / router::kWarps);
  const size_t smem = bias || n_groups > 1 ? (size_t)router::kWarps * n_experts * sizeof(double) : 0;
  return router::with_nper(n_experts, [&](auto nper) {
    constexpr int n = decltype(nper)::value;
    const auto kernel = n_groups > 1 ? (bias ? router::select_kernel<n, true, true> : router::select_kernel<n, false, true>)
                                     : (bias ? router::select_kernel<n, true, false> : router::select_kernel<n, false, false>);
    launch(kernel, grid, router::kWarps * 32, smem, reinterpret_cast<cudaStream_t>(stream), p);
    return check_launch("cvmm_router_select");
  });
}

extern "C" int cvmm_router_select_backward(const void* logits, int logits_dtype, int64_t logits_ld, const int64_t* sel,
                                           const float* grad_weights, int64_t n_tokens, int64_t n_experts,
                                           int64_t top_k, int scoring, int renormalize, float scale,
                                           void* grad_logits, cvmm_stream_t stream) {
  using namespace cvmm;
  if (!is_float_dtype(logits_dtype))
    return fail(CVMM_ERR_UNSUPPORTED_DTYPE, "cvmm_router_select_backward: unsupported dtype");
  if (scoring != CVMM_SCORE_SOFTMAX && scoring != CVMM_SCORE_SIGMOID)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select_backward: scoring must be softmax or sigmoid");
  if (n_tokens < 0 || n_experts <= 0 || n_experts > router::kMaxExperts || logits_ld < n_experts || top_k < 1 ||
      top_k > router::kMaxTopK || top_k > n_experts || n_tokens > (int64_t)INT32_MAX)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select_backward: bad sizes");
  if (n_tokens == 0) return CVMM_OK;
  if (!logits || !sel || !grad_weights || !grad_logits)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_router_select_backward: null pointer");
  const unsigned grid = (unsigned)((n_tokens + router::kWarps - 1) / router::kWarps);
  return router::with_nper(n_experts, [&](auto nper) {
    launch(router::select_backward_kernel<decltype(nper)::value>, grid, router::kWarps * 32, 0,
           reinterpret_cast<cudaStream_t>(stream), logits, logits_dtype, logits_ld, sel, grad_weights, n_tokens,
           (int)n_experts, (int)top_k, scoring, renormalize, scale, grad_logits);
    return check_launch("cvmm_router_select_backward");
  });
}
