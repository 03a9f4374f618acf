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
// nearer than the bound is decided again in 64 bits. How many that are depends
// on the inputs (64 experts top 4 and 128 experts top 8, logits of deviation
// 1.5): 0.01 to 0.1 % with a bias of deviation 0.05. A zero bias leaves equal
// logits equal, and a tie between the k-th and the next expert always goes there:
// 3.4 and 7.3 % with bf16 logits, 1 % with fp16. The bound of a sigmoid is
// absolute, so with a zero bias scores near 0 or 1 go there, too: 95 % at logits
// around -14, 29 % around +6. 32768 tokens x 128 experts, bf16 softmax: 20.3 us
// without a bias, 29.4 with one, 45.1 with a zero one.
#include "common.cuh"
#include "launch.h"

namespace cvmm {
namespace router {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;
constexpr int kMaxGroups = 32;  // a bit each
constexpr int kWarps = 4;
constexpr int kBadSelTag = 30;  // status-word site: a chosen id outside [0, n_experts)

// How far the difference of two 32-bit values may be from the exact one.
// Softmax, in units of the largest score 1 / sum: expf's 2 ulp of 1.2e-7, the
// argument's half ulp, x e^-x 6e-8 <= 2.2e-8, and the product with the rounded
// 1 / sum, 1.8e-7, for each of the two; the sum's error scales the whole
// difference, which is at most one unit: EPL additions in a lane and 5 across at
// 6e-8 and its terms' 2.4e-7. Sigmoid takes __expf(-x), within 2 + 1.17 x ulp,
// and (2 + 1.17 x) e^-x <= 2.4: each s (1 - s) times that, 9e-8, half an ulp of
// 1 + e and 2 ulp of the division, 3e-7. c = s + b adds half an ulp of each c.
template <int EPL>
__device__ __forceinline__ float pair_error(bool softmax, float smax) {
  return softmax ? smax * (1.2e-6f + 6e-8f * (EPL + 5)) : 9e-7f;
}
constexpr float kAddErr = 6e-8f;   // relative, of c
constexpr float kTinyErr = 1e-37f; // scores below the normal range, which __expf gives as 0 (1.2e-38 each)

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
  int vec;            // runs of EPL logits (and biases) are whole and 16-byte aligned: 1 logits, 2 biases
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

// 1 / (1 + exp(-z)) without overflow: exp of -|z| only. FAST where an error in
// s of 3e-7 will do, else relative.
template <bool FAST = false>
__device__ __forceinline__ float sigmoid(float z) {
  const float e = FAST ? __expf(-fabsf(z)) : expf(-fabsf(z));
  return __fdividef(z < 0.f ? e : 1.f, 1.f + e);  // 2 ulp for divisors from 1 to 2
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

// Decides token t again with 64-bit scores; v: E doubles of the warp's shared
// memory. Lane j < k returns the j-th expert. Few tokens come here, but a launch
// ends with the last of them: loads go four at a time, the order is kept as
// integer keys, and a round is three warp reductions (its high and low halves,
// then the lowest index): 53 -> 47 us with 20 of 32768 tokens here.
__device__ __noinline__ int decide_in_64(const Args& p, int64_t t, double* v) {
  constexpr int kAtOnce = 4;
  const int lane = threadIdx.x & 31, E = p.E;
  const bool softmax = p.scoring == kSoftmax;
  auto each = [&](auto f) {  // f(e, z_e)
    for (int e0 = lane; e0 < E; e0 += 32 * kAtOnce) {
      float z[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) z[u] = e0 + 32 * u < E ? logit(p, t, e0 + 32 * u) : -INFINITY;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (e0 + 32 * u < E) f(e0 + 32 * u, z[u]);
    }
  };
  double mx = 0.0, sum = 1.0;
  if (softmax) {
    float m = -INFINITY;
    each([&](int, float z) { m = fmaxf(m, z); });
    mx = warp_max(m);
    if (mx == -(double)INFINITY) mx = 0.0;
    sum = 0.0;
    each([&](int e, float z) {
      const double x = exp((double)z - mx);
      v[e] = x;
      sum += x;
    });
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum == 0.0) sum = 1.0;
  }
  each([&](int e, float z) {
    const double s = softmax ? v[e] / sum : 1.0 / (1.0 + exp(-(double)z));
    const double c = p.bias ? s + (double)load_as_float(p.bias, p.bias_dtype, e) : s;
    v[e] = z == -INFINITY ? -(double)INFINITY : c;
  });
  __syncwarp();
  uint32_t groups = 0xffffffffu;
  if (p.G > 1) {
    double worst, other;
    groups = best_groups(p, v, E / p.G, worst, other);
    __syncwarp();
  }
  unsigned long long* key = reinterpret_cast<unsigned long long*>(v);
  each([&](int e, float z) {
    const bool in = p.G == 1 || ((groups >> group_of(p, e)) & 1u);
    key[e] = in ? key_of(p.bias ? v[e] : (double)z) : 0ull;
  });
  int chosen = 0;
  for (int j = 0; j < p.k; ++j) {  // a lane reads and writes its own keys only
    unsigned long long best = 0;
    int be = 0x7fffffff;
#pragma unroll 4
    for (int e = lane; e < E; e += 32)
      if (key[e] > best) {
        best = key[e];
        be = e;
      }
    const uint32_t hi = (uint32_t)(best >> 32), top = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = hi == top ? (uint32_t)best : 0u, low = __reduce_max_sync(0xffffffffu, lo);
    be = (int)__reduce_min_sync(0xffffffffu, hi == top && lo == low ? (uint32_t)be : 0xffffffffu);
    if ((be & 31) == lane) key[be] = 0ull;
    if (lane == j) chosen = be;
  }
  return chosen;
}

// Values e0 .. e0 + N - 1 of a row of E (those past it are `pad`), N consecutive
// to a lane. vec: the run is whole and 16-byte aligned.
template <int N>
__device__ __forceinline__ void load_run(float (&v)[N], const void* row, int dtype, int64_t at, int e0, int E, bool vec,
                                         float pad) {
  static_assert(N % 8 == 0, "16-byte loads of 16-bit values");
  if (vec && e0 < E) {
    if (dtype == F32) {
      const float4* from = reinterpret_cast<const float4*>(static_cast<const float*>(row) + at + e0);
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const float4 f = from[i];
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      }
    } else {
      const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + at + e0);
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        const uint4 f = from[i];
        const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] = bits_to_float((uint16_t)(w[j] & 0xffffu), dtype);
          v[8 * i + 2 * j + 1] = bits_to_float((uint16_t)(w[j] >> 16), dtype);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < N; ++q) v[q] = e0 + q < E ? load_as_float(row, dtype, at + e0 + q) : pad;
}

// Sums and maxima over the LPT lanes of a token.
template <int LPT>
__device__ __forceinline__ float token_sum(float v) {
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LPT>
__device__ __forceinline__ float token_max(float v) {  // NaN only if every value is
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Shared memory of a warp of `tokens` tokens, in bytes: keys or 64-bit values,
// group keys, k + 1 choices and their keys, later scores.
__host__ __device__ constexpr size_t values_bytes(int tokens, int E) {
  return tokens == 1 ? (size_t)E * 8 : ((size_t)tokens * E * 4 + 7) / 8 * 8;
}
__host__ __device__ constexpr size_t warp_bytes(int tokens, int E, int k, bool values) {
  return (values ? values_bytes(tokens, E) + (size_t)tokens * kMaxGroups * 4 : 0) + (size_t)tokens * (k + 1) * 8;
}

// LPT lanes a token, 32 / LPT tokens a warp; a lane holds EPL consecutive
// experts, so rows come in 16-byte loads and the lowest lane of equals has the
// lowest index. Every lane keeps the largest of its keys; a round of the top-k
// is a maximum over the token's lanes, a ballot for the lane that has it, and
// that lane's search for its next largest. Bound by instructions: with one
// token a warp (two reductions a round, lane l holding l + 32 q) 32768 tokens x
// 128 experts in 8 groups took 1280 instructions a token and 54 us.
// BIAS and GROUPS leave out what a call without them does not do.
template <int LPT, int EPL, bool BIAS, bool GROUPS>
__global__ void __launch_bounds__(kWarps * 32) select_kernel(const __grid_constant__ Args p) {
  pdl_enter();
  constexpr int TPW = 32 / LPT;
  extern __shared__ double sh[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane % LPT, tok = lane / LPT, e0 = sub * EPL;
  const int64_t t0 = (blockIdx.x * (int64_t)kWarps + warp) * TPW;
  if (t0 >= p.T) return;
  const bool live = t0 + tok < p.T;
  const int64_t t = live ? t0 + tok : p.T - 1;  // spare lanes repeat the last token
  const int E = p.E;
  const bool softmax = p.scoring == kSoftmax;
  char* mine = reinterpret_cast<char*>(sh) + warp * warp_bytes(TPW, E, p.k, BIAS || GROUPS);
  uint32_t* v = reinterpret_cast<uint32_t*>(mine) + tok * E;                                     // BIAS or GROUPS only
  uint32_t* gkey = reinterpret_cast<uint32_t*>(mine + values_bytes(TPW, E)) + tok * kMaxGroups;  // too
  int* sel = reinterpret_cast<int*>(mine + (BIAS || GROUPS ? values_bytes(TPW, E) + TPW * kMaxGroups * 4 : 0));
  uint32_t* ckey = reinterpret_cast<uint32_t*>(sel + TPW * (p.k + 1));
  sel += tok * (p.k + 1);
  ckey += tok * (p.k + 1);
  float z[EPL], b[EPL], s[EPL];
  load_run(z, p.logits, p.dtype, t * p.ld, e0, E, p.vec & 1, -INFINITY);
  if (BIAS) load_run(b, p.bias, p.bias_dtype, 0, e0, E, p.vec & 2, 0.f);
  float mx = 0.f, inv = 1.f;
  if (softmax) {
    mx = z[0];
#pragma unroll
    for (int q = 1; q < EPL; ++q) mx = fmaxf(mx, z[q]);
    mx = token_max<LPT>(mx);
    if (mx == -INFINITY || mx != mx) mx = 0.f;  // every expert masked: all scores are 0
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
      s[q] = expf(z[q] - mx);  // the sum is the weights' and the gradient's, too
      sum += e0 + q < E ? s[q] : 0.f;
    }
    sum = token_sum<LPT>(sum);
    inv = sum == 0.f ? 1.f : 1.f / sum;
  }
  const float err = pair_error<EPL>(softmax, inv);  // no softmax score is above 1 / sum
  if (BIAS || (GROUPS && p.top2)) {
#pragma unroll
    for (int q = 0; q < EPL; ++q) s[q] = softmax ? s[q] * inv : sigmoid<true>(z[q]);
  }
  uint32_t key[EPL];
#pragma unroll
  for (int q = 0; q < EPL; ++q) {
    key[q] = e0 + q < E ? key_of(BIAS && z[q] != -INFINITY ? s[q] + b[q] : z[q]) : 0u;
    if (GROUPS && e0 + q < E) v[e0 + q] = !BIAS && p.top2 && z[q] != -INFINITY ? key_of(s[q]) : key[q];
  }
  bool again = false;
  if (GROUPS) {
    const int size = E / p.G;
    __syncwarp();
    // A lane a group; it starts at another place of its group than its
    // neighbours, which else would meet in one bank.
    for (int g = sub; g < p.G; g += LPT) {
      uint32_t first = 0, second = 0;  // the two largest keys
      int m = g < size ? g : g % size;
      for (int i = 0; i < size; ++i) {
        const uint32_t k = v[g * size + m];
        second = max(second, min(first, k));
        first = max(first, k);
        if (++m == size) m = 0;
      }
      // A masked second (key_of(-inf), or none) counts as nothing.
      if (p.top2 && second > key_of(-INFINITY)) first = key_of(value_of(first) + value_of(second));
      gkey[g] = first;
    }
    __syncwarp();
    uint32_t chosen = 0, worst = 0, other = 0;  // groups as bits; two keys
    for (int g = sub; g < p.G; g += LPT) {
      const uint32_t k = gkey[g];
      int rank = 0;
      for (int o = 0; o < p.G; ++o) rank += gkey[o] > k || (gkey[o] == k && o < g);
      if (rank < p.top_groups) chosen |= 1u << g;
      if (rank == p.top_groups - 1) worst = k;
      if (rank == p.top_groups) other = k;
    }
    // Ranks are a permutation: one lane has each value, the others 0.
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) {
      chosen |= __shfl_xor_sync(0xffffffffu, chosen, o);
      worst |= __shfl_xor_sync(0xffffffffu, worst, o);
      other |= __shfl_xor_sync(0xffffffffu, other, o);
    }
    // The worst chosen and the best other group must differ by more than the
    // error of both. With a bias a value is a sum of up to two c, which may be
    // large with a small sum: half an ulp of each c (at most 1 + max |b|) and of
    // each sum (at most twice that), for two groups.
    const float lo = value_of(worst), hi = value_of(other);
    if ((BIAS || p.top2) && p.top_groups < p.G) {
      float size_c = fabsf(lo) + fabsf(hi);
      if (BIAS) {
        size_c = 0.f;
#pragma unroll
        for (int q = 0; q < EPL; ++q)
          if (fabsf(b[q]) < INFINITY) size_c = fmaxf(size_c, fabsf(b[q]));
        size_c = 2.f * (1.f + token_max<LPT>(size_c));
      }
      again = hi > -INFINITY && lo - hi <= 2.f * err + 4.f * kAddErr * size_c + kTinyErr;
    }
#pragma unroll
    for (int q = 0; q < EPL; ++q)
      if (!((chosen >> (group_of(p, min(e0 + q, E - 1)) & 31)) & 1u)) key[q] = 0u;
  }
  uint32_t best;
  int bq;
  auto local_best = [&]() {
    best = key[0];
    bq = 0;
#pragma unroll
    for (int q = 1; q < EPL; ++q)
      if (key[q] > best) {
        best = key[q];
        bq = q;
      }
  };
  local_best();
  // With a bias one more expert is looked at, to see that it is clearly lower than the k-th.
  const int rounds = BIAS ? min(p.k + 1, GROUPS ? p.top_groups * (E / p.G) : E) : p.k;
  for (int j = 0; j < rounds; ++j) {
    uint32_t top = best;
#pragma unroll
    for (int o = LPT / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t at = __ballot_sync(0xffffffffu, best == top) >> (tok * LPT);
    const int from = __ffs(LPT == 32 ? at : at & ((1u << (LPT & 31)) - 1u)) - 1;
    if (sub == from) {
      sel[j] = e0 + bq;
      if (BIAS) ckey[j] = top;
#pragma unroll
      for (int q = 0; q < EPL; ++q)
        if (q == bq) key[q] = 0u;
      local_best();
    }
  }
  __syncwarp();
  if (BIAS) {
    // Neighbours nearer than their errors are decided again, unless they have
    // equal logits and biases and so are equal in any number of bits (past the
    // k-th another equal one may follow: again).
    for (int j = sub; j + 1 < rounds; j += LPT) {
      const float c = value_of(ckey[j]), d = value_of(ckey[j + 1]);
      if (d > -INFINITY && c - d <= err + kAddErr * (fabsf(c) + fabsf(d)) + kTinyErr)
        again |= j + 1 == p.k || logit(p, t, sel[j]) != logit(p, t, sel[j + 1]) ||
                 load_as_float(p.bias, p.bias_dtype, sel[j]) != load_as_float(p.bias, p.bias_dtype, sel[j + 1]);
    }
    const uint32_t any = __ballot_sync(0xffffffffu, again) >> (tok * LPT);
    again = (LPT == 32 ? any : any & ((1u << (LPT & 31)) - 1u)) != 0;
  }
  __syncwarp();
  if (BIAS || GROUPS) {
    // Tokens to decide again, one after the other, by the whole warp.
    uint32_t todo = __ballot_sync(0xffffffffu, again && live && sub == 0);
    while (todo) {
      const int from = __ffs(todo) - 1;
      todo &= todo - 1;
      const int chosen = decide_in_64(p, t0 + from / LPT, reinterpret_cast<double*>(mine));
      int* to = reinterpret_cast<int*>(mine + values_bytes(TPW, E) + TPW * kMaxGroups * 4) + from / LPT * (p.k + 1);
      if (lane < p.k) to[lane] = chosen;
      __syncwarp();
    }
  }
  float* score = reinterpret_cast<float*>(ckey);
  float tot = 0.f;
  for (int j = sub; j < p.k; j += LPT) {
    const float zc = logit(p, t, sel[j]);
    const float sc = softmax ? expf(zc - mx) * inv : sigmoid(zc);
    score[j] = sc;
    tot += sc;
  }
  tot = token_sum<LPT>(tot);
  const float held = tot < 1e-20f ? 1e-20f : tot;
  if (!live) return;
  for (int j = sub; j < p.k; j += LPT) {
    p.sel[t * p.k + j] = sel[j];
    p.weights[t * p.k + j] = p.scale * (p.renorm ? score[j] / held : score[j]);
  }
}

// d w / d z. With S = max(sum s_j, 1e-20) and g the weights' gradient:
//   gs_j = scale (g_j - sum_i g_i s_i / S) / S   (no sum term where S is held; scale g_j without renormalising)
//   softmax: gz_e = s_e (gs_e - sum_j s_j gs_j)      sigmoid: gz_e = gs_e s_e (1 - s_e)
// with gs_e = 0 off the chosen experts. Lanes hold experts as select_kernel's
// do, write the row once and then the chosen entries over it.
template <int LPT, int EPL>
__global__ void __launch_bounds__(kWarps * 32)
select_backward_kernel(const void* __restrict__ logits, int dtype, int64_t ld, const int64_t* __restrict__ sel,
                       const float* __restrict__ grad_w, int64_t T, int E, int k, int scoring, int renorm, float scale,
                       bool vec, bool out_vec, void* __restrict__ grad_logits) {
  static_assert(EPL % 8 == 0, "rows are stored 8 values at a time");
  pdl_enter();
  constexpr int TPW = 32 / LPT;
  const int lane = threadIdx.x & 31, sub = lane % LPT, e0 = sub * EPL;
  const int64_t t0 = (blockIdx.x * (int64_t)kWarps + (threadIdx.x >> 5)) * TPW;
  if (t0 >= T) return;
  const bool live = t0 + lane / LPT < T;
  const int64_t t = live ? t0 + lane / LPT : T - 1;
  const bool softmax = scoring == kSoftmax;
  float s[EPL];
  float mx = 0.f, inv = 1.f;
  if (softmax) {
    load_run(s, logits, dtype, t * ld, e0, E, vec, -INFINITY);
    mx = s[0];
#pragma unroll
    for (int q = 1; q < EPL; ++q) mx = fmaxf(mx, s[q]);
    mx = token_max<LPT>(mx);
    if (mx == -INFINITY || mx != mx) mx = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
      s[q] = expf(s[q] - mx);
      sum += e0 + q < E ? s[q] : 0.f;
    }
    sum = token_sum<LPT>(sum);
    inv = sum == 0.f ? 1.f : 1.f / sum;
  }
  // Score of the j-th chosen expert; -1 for an id that names none.
  auto chosen = [&](int j, float& sj, float& rest, float& g) -> int {
    const int64_t e = sel[t * k + j];
    if (e < 0 || e >= E) {
      report(CVMM_DEV_BAD_INDEX, kBadSelTag, (long long)e);
      return -1;
    }
    const float z = load_as_float(logits, dtype, t * ld + e);
    sj = softmax ? expf(z - mx) * inv : sigmoid(z);
    rest = sigmoid(-z);  // 1 - s, from the other side
    g = scale * grad_w[t * k + j];
    return (int)e;
  };
  float tot = 0.f, gs = 0.f, sj, rest, g;
  for (int j = sub; j < k; j += LPT)
    if (chosen(j, sj, rest, g) >= 0) {
      tot += sj;
      gs += g * sj;
    }
  tot = token_sum<LPT>(tot);
  gs = token_sum<LPT>(gs);
  // gs_j = (g_j - mean) / held, so sum_j s_j gs_j = (gs - mean tot) / held
  const float held = renorm ? (tot < 1e-20f ? 1e-20f : tot) : 1.f;
  const float mean = renorm && !(tot < 1e-20f) ? gs / held : 0.f;
  const float dot = softmax ? (gs - mean * tot) / held : 0.f;
  if (live) {
    float out[EPL];
#pragma unroll
    for (int q = 0; q < EPL; ++q) out[q] = softmax ? -s[q] * inv * dot : 0.f;
    const int64_t at = t * E + e0;
    if (out_vec && e0 < E) {
#pragma unroll
      for (int i = 0; i < EPL; i += 8) {
        float (&o)[8] = *reinterpret_cast<float (*)[8]>(out + i);
        store8(static_cast<char*>(grad_logits) + (at + i) * dtype_bytes(dtype), dtype, o);
      }
    } else {
#pragma unroll
      for (int q = 0; q < EPL; ++q)
        if (e0 + q < E) store_from_float(grad_logits, dtype, at + q, out[q]);
    }
  }
  __syncwarp();
  if (!live) return;
  for (int j = sub; j < k; j += LPT) {
    const int e = chosen(j, sj, rest, g);
    if (e < 0) continue;
    g = (g - mean) / held;
    store_from_float(grad_logits, dtype, t * E + e, softmax ? sj * (g - dot) : g * sj * rest);
  }
}

// The lanes a token takes: 8 experts each up to 256, then 32 lanes of 16 or 32.
template <int L, int P>
struct Split {
  static constexpr int lpt = L, epl = P;
};
template <typename F>
static int with_split(int64_t E, F f) {
  if (E <= 8) return f(Split<1, 8>());
  if (E <= 16) return f(Split<2, 8>());
  if (E <= 32) return f(Split<4, 8>());
  if (E <= 64) return f(Split<8, 8>());
  if (E <= 128) return f(Split<16, 8>());
  if (E <= 256) return f(Split<32, 8>());
  if (E <= 512) return f(Split<32, 16>());
  return f(Split<32, 32>());
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
  return router::with_split(n_experts, [&](auto split) {
    constexpr int lpt = decltype(split)::lpt, epl = decltype(split)::epl, tokens = 32 / lpt;
    const auto aligned = [&](const void* q, int dtype, int64_t ld) {
      return n_experts % epl == 0 && al16(q) && ld * (int64_t)dtype_size(dtype) % 16 == 0;
    };
    p.vec = (aligned(logits, logits_dtype, logits_ld) ? 1 : 0) | (bias && aligned(bias, bias_dtype, 0) ? 2 : 0);
    const auto kernel = n_groups > 1 ? (bias ? router::select_kernel<lpt, epl, true, true> : router::select_kernel<lpt, epl, false, true>)
                                     : (bias ? router::select_kernel<lpt, epl, true, false> : router::select_kernel<lpt, epl, false, false>);
    const unsigned grid = (unsigned)((n_tokens + router::kWarps * tokens - 1) / (router::kWarps * tokens));
    launch(kernel, grid, router::kWarps * 32,
           router::kWarps * router::warp_bytes(tokens, p.E, p.k, bias || n_groups > 1),
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
  return router::with_split(n_experts, [&](auto split) {
    constexpr int lpt = decltype(split)::lpt, epl = decltype(split)::epl, per = router::kWarps * (32 / lpt);
    const int64_t size = (int64_t)dtype_size(logits_dtype);
    const bool vec = n_experts % epl == 0 && al16(logits) && logits_ld * size % 16 == 0;
    const bool out_vec = n_experts % epl == 0 && al16(grad_logits) && n_experts * size % 16 == 0;
    launch(router::select_backward_kernel<lpt, epl>, (unsigned)((n_tokens + per - 1) / per), router::kWarps * 32, 0,
           reinterpret_cast<cudaStream_t>(stream), logits, logits_dtype, logits_ld, sel, grad_weights, n_tokens,
           (int)n_experts, (int)top_k, scoring, renormalize, scale, vec, out_vec, grad_logits);
    return check_launch("cvmm_router_select_backward");
  });
}
