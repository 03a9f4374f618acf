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
__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 1 / (1 + exp(-z)) without overflow: exp of -|z| only.
__device__ __forceinline__ float sigmoid(float z) {
  const float e = expf(-fabsf(z));
  return (z < 0.f ? e : 1.f) / (1.f + e);
}

// Two largest values of a group, in key order.
template <typename R>
struct Top2 {
  R a, b;
  __device__ __forceinline__ void add(R v) {
    if (key_of(v) > key_of(a)) { b = a; a = v; }
    else if (key_of(v) > key_of(b)) b = v;
  }
};
// Group value from its two largest: a masked (-inf) second counts as nothing.
template <typename R>
__device__ __forceinline__ R group_value(const Top2<R>& t, int top2) {
  return top2 && t.b != -(R)INFINITY ? t.a + t.b : t.a;
}

// Decides one token again with 64-bit scores; z: its logits in shared memory.
// Lane j < k returns the j-th expert. Candidates are marked by bit q of `out`
// (expert lane + 32 q already taken or outside the chosen groups).
__device__ __noinline__ int decide_in_64(const Args& p, const float* z) {
  const int lane = threadIdx.x & 31;
  const bool softmax = p.scoring == kSoftmax;
  double mx = 0.0, sum = 1.0;
  if (softmax) {
    float m = -INFINITY;
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, z[e]);
    mx = warp_max(m);
    if (mx == -(double)INFINITY) mx = 0.0;
    sum = 0.0;
    for (int e = lane; e < p.E; e += 32) sum += exp((double)z[e] - mx);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum == 0.0) sum = 1.0;
  }
  auto by = [&](int e) -> double {
    const double s = softmax ? exp((double)z[e] - mx) / sum : 1.0 / (1.0 + exp(-(double)z[e]));
    const double c = p.bias ? s + (double)load_as_float(p.bias, p.bias_dtype, e) : s;
    return z[e] == -INFINITY ? -(double)INFINITY : c;
  };
  auto order = [&](int e) -> double { return p.bias ? by(e) : (double)z[e]; };
  uint32_t groups = 0xffffffffu;
  const int size = p.E / p.G;
  if (p.G > 1) {
    unsigned long long mine = 0;
    if (lane < p.G) {
      Top2<double> t = {-(double)INFINITY, -(double)INFINITY};
      for (int m = 0; m < size; ++m) t.add(p.top2 ? by(lane * size + m) : order(lane * size + m));
      mine = key_of(group_value(t, p.top2));
    }
    int rank = 0;
    for (int g = 0; g < p.G; ++g) {
      const unsigned long long o = __shfl_sync(0xffffffffu, mine, g);
      rank += o > mine || (o == mine && g < lane);
    }
    groups = __ballot_sync(0xffffffffu, lane < p.G && rank < p.top_groups);
  }
  uint32_t out = 0;
  for (int q = 0; lane + 32 * q < p.E; ++q)
    if (p.G > 1 && !((groups >> ((lane + 32 * q) / size)) & 1u)) out |= 1u << q;
  int chosen = 0;
  for (int j = 0; j < p.k; ++j) {
    unsigned long long best = 0;
    int be = 0x7fffffff;
    for (int q = 0; lane + 32 * q < p.E; ++q) {
      if ((out >> q) & 1u) continue;
      const unsigned long long v = key_of(order(lane + 32 * q));
      if (v > best) { best = v; be = lane + 32 * q; }
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

// One warp a token; lane l holds experts l, l + 32, ... (NPER of them).
// Per round of the top-k: the largest key over the warp, then the lowest index
// that has it, each one warp-wide integer reduction.
template <int NPER>
__global__ void __launch_bounds__(kWarps * 32) select_kernel(const __grid_constant__ Args p) {
  pdl_enter();
  extern __shared__ float sh[];  // per warp: logits [E], group operand [E] (with a bias or groups only)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x * (int64_t)kWarps + warp;
  if (t >= p.T) return;
  const int E = p.E;
  const bool softmax = p.scoring == kSoftmax;
  float z[NPER], s[NPER];
  float mx = -INFINITY;
#pragma unroll
  for (int q = 0; q < NPER; ++q) {
    const int e = lane + 32 * q;
    z[q] = e < E ? load_as_float(p.logits, p.dtype, t * p.ld + e) : -INFINITY;
    mx = fmaxf(mx, z[q]);
  }
  float smax = 1.f;  // no score is above this
  if (softmax) {
    mx = warp_max(mx);
    if (mx == -INFINITY) mx = 0.f;  // every expert masked: all scores are 0
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      s[q] = expf(z[q] - mx);
      sum += lane + 32 * q < E ? s[q] : 0.f;
    }
    sum = warp_sum(sum);
    if (sum == 0.f) sum = 1.f;
#pragma unroll
    for (int q = 0; q < NPER; ++q) s[q] /= sum;
    smax = 1.f / sum;
  } else {
#pragma unroll
    for (int q = 0; q < NPER; ++q) s[q] = sigmoid(z[q]);
  }
  float c[NPER], b[NPER];
#pragma unroll
  for (int q = 0; q < NPER; ++q) {
    const int e = lane + 32 * q;
    b[q] = p.bias && e < E ? load_as_float(p.bias, p.bias_dtype, e) : 0.f;
    c[q] = p.bias && z[q] != -INFINITY ? s[q] + b[q] : z[q];
  }
  const float err = pair_error<NPER>(softmax, smax);
  float* shz = sh + warp * 2 * E;
  float* shv = shz + E;
  const bool again_possible = p.bias || p.G > 1;
  if (again_possible) {
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      const int e = lane + 32 * q;
      if (e < E) {
        shz[e] = z[q];
        shv[e] = p.bias || !p.top2 ? c[q] : (z[q] == -INFINITY ? -INFINITY : s[q]);
      }
    }
    __syncwarp();
  }
  bool again = false;
  uint32_t groups = 0xffffffffu;
  const int size = E / p.G;
  if (p.G > 1) {
    // 32 / (G rounded up to a power of two) lanes share a group.
    const int lanes = 32 >> (32 - __clz(p.G - 1));
    const int g = lane / lanes;
    Top2<float> top = {-INFINITY, -INFINITY};
    if (g < p.G)
      for (int m = lane % lanes; m < size; m += lanes) top.add(shv[g * size + m]);
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      const float oa = __shfl_xor_sync(0xffffffffu, top.a, o), ob = __shfl_xor_sync(0xffffffffu, top.b, o);
      top.add(oa);
      top.add(ob);
    }
    const float gv = group_value(top, p.top2);
    const uint32_t mine = g < p.G ? key_of(gv) : 0u;
    int rank = 0;
    for (int o = 0; o < p.G; ++o) {
      const uint32_t v = __shfl_sync(0xffffffffu, mine, o * lanes);
      rank += v > mine || (v == mine && o < g);
    }
    const bool in = g < p.G && rank < p.top_groups;
    const uint32_t ballot = __ballot_sync(0xffffffffu, in);
    groups = 0;
    for (int o = 0; o < p.G; ++o) groups |= ((ballot >> (o * lanes)) & 1u) << o;
    if (p.top_groups < p.G && (p.bias || p.top2)) {
      // The worst chosen and the best other group must differ by more than the error of both.
      const uint32_t lo = __reduce_min_sync(0xffffffffu, in ? mine : 0xffffffffu);
      const uint32_t hi = __reduce_max_sync(0xffffffffu, g < p.G && !in ? mine : 0u);
      const float worst = __shfl_sync(0xffffffffu, gv, __ffs(__ballot_sync(0xffffffffu, in && mine == lo)) - 1);
      const float other = __shfl_sync(0xffffffffu, gv,
                                      __ffs(__ballot_sync(0xffffffffu, g < p.G && !in && mine == hi)) - 1);
      again = worst - other <= 2.f * err + 4.f * kAddErr * (fabsf(worst) + fabsf(other)) + kTinyErr;
    }
  }
  uint32_t key[NPER];
#pragma unroll
  for (int q = 0; q < NPER; ++q) {
    const int e = lane + 32 * q;
    key[q] = e < E && (p.G == 1 || ((groups >> (e / size)) & 1u)) ? key_of(c[q]) : 0u;
  }
  int chosen = 0;
  float score = 0.f;
  float pc = 0.f, pz = 0.f, pb = 0.f;  // the expert before: c, z, b
  const int n_cand = p.G == 1 ? E : p.top_groups * size;
  for (int j = 0; j < n_cand; ++j) {
    if (again || (j >= p.k && !p.bias)) break;
    uint32_t best = 0;
    int be = 0x7fffffff;
#pragma unroll
    for (int q = 0; q < NPER; ++q)
      if (key[q] > best) {
        best = key[q];
        be = lane + 32 * q;
      }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    be = (int)__reduce_min_sync(0xffffffffu, best == top ? (uint32_t)be : 0xffffffffu);
    float bs = 0.f, bc = 0.f, bz = 0.f, bb = 0.f;
#pragma unroll
    for (int q = 0; q < NPER; ++q)
      if (lane + 32 * q == be) {
        key[q] = 0;
        bs = s[q];
        bc = c[q];
        bz = z[q];
        bb = b[q];
      }
    bs = __shfl_sync(0xffffffffu, bs, be & 31);
    if (p.bias) {
      // Neighbours nearer than their errors are decided again, unless they are
      // the same expert twice over (equal logit and bias: equal in any number
      // of bits). Past the k-th the check runs on until one is clearly lower.
      bc = __shfl_sync(0xffffffffu, bc, be & 31);
      bz = __shfl_sync(0xffffffffu, bz, be & 31);
      bb = __shfl_sync(0xffffffffu, bb, be & 31);
      const bool same = bz == pz && bb == pb;
      if (j > 0 && !same && pc - bc <= err + kAddErr * (fabsf(pc) + fabsf(bc)) + kTinyErr) again = true;
      if (j >= p.k && !same) break;
      pc = bc;
      pz = bz;
      pb = bb;
    }
    if (lane == j) {
      chosen = be;
      score = bs;
    }
  }
  if (again) {
    chosen = decide_in_64(p, shz);
    if (lane < p.k) {
      const float zc = shz[chosen];
      score = softmax ? expf(zc - mx) * smax : sigmoid(zc);
    }
  }
  if (lane >= p.k) score = 0.f;
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
  float s[NPER];
  float mx = 0.f, inv = 1.f;
  if (softmax) {
    mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      const int e = lane + 32 * q;
      s[q] = e < E ? load_as_float(logits, dtype, t * ld + e) : -INFINITY;
      mx = fmaxf(mx, s[q]);
    }
    mx = warp_max(mx);
    if (mx == -INFINITY) mx = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < NPER; ++q) {
      s[q] = expf(s[q] - mx);
      sum += lane + 32 * q < E ? s[q] : 0.f;
    }
    sum = warp_sum(sum);
    inv = sum == 0.f ? 1.f : 1.f / sum;
  }
  int64_t e = -1;
  float g = 0.f, sj = 0.f, rest = 0.f;  // rest: 1 - s, from the other side
  if (lane < k) {
    e = sel[t * k + lane];
    if (e < 0 || e >= E) {
      report(CVMM_DEV_BAD_INDEX, kBadSelTag, (long long)e);
      e = -1;
    } else {
      const float z = load_as_float(logits, dtype, t * ld + e);
      sj = softmax ? expf(z - mx) * inv : sigmoid(z);
      rest = sigmoid(-z);
      g = scale * grad_w[t * k + lane];
    }
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
  p.renorm = renormalize; p.scale = scale; p.sel = sel; p.weights = weights;
  const unsigned grid = (unsigned)((n_tokens + router::kWarps - 1) / router::kWarps);
  const size_t smem = bias || n_groups > 1 ? (size_t)router::kWarps * 2 * n_experts * sizeof(float) : 0;
  return router::with_nper(n_experts, [&](auto nper) {
    launch(router::select_kernel<decltype(nper)::value>, grid, router::kWarps * 32, smem,
           reinterpret_cast<cudaStream_t>(stream), p);
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
