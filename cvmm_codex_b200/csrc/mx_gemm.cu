// Expert product of 4-bit rows with 4-bit expert weights (cvmm_mx_forward).
//
//   y[r] = Q(x[r / per_row]) . W[sel[r]]^T;  out[r] = y[r], or with weights
//   out[t] = sum_j w[t, j] y[t top_k + j]
//
// Three or four launches:
//   prepare  quantises the rows of x once, in their own order (4 bits a value,
//            so that all route copies of a row are reads of the same bytes), and
//            lists the routes of every expert and the 128-route tiles they make;
//   fill     (many routes only) writes the lists that prepare counted;
//   gemm     gathers a tile's rows with TMA and multiplies them with the
//            expert's weight tiles on the tensor cores, scales and all;
//   combine  (weights only) sums the route outputs.
// The order of the routes within an expert's list is left to atomics: a row's
// output does not depend on where in a tile it stands.
#include "launch.h"
#include "mx.cuh"
#include "ptx.cuh"

namespace cvmm {
namespace mx {

constexpr int kTile = 128;           // routes of a tile (MMA M)
constexpr int64_t kMaxExperts = 4096;
constexpr int kPlanThreads = 256;
constexpr int64_t kPlanChunk = 4096;  // routes one block counts or lists
constexpr int kBadIdTag = 31;         // status-word site: an expert id outside [0, n_experts)
enum : int { kTagEmpty = 40, kTagFull = 41, kTagAccFull = 42, kTagAccEmpty = 43, kTagDrain = 44 };

struct Product {
  // x
  const void* x;
  int x_dtype;
  int64_t x_rows, x_ld;
  bool x_vec;
  int per_row;  // routes that share a row
  uint8_t* xd;  // [x_rows][row_bytes]
  uint8_t* xs;  // [x_rows][cells] of 4 scale bytes, cells a multiple of 4
  int64_t cells;
  // routing
  const void* sel;
  int sel_dtype;
  int64_t R;
  int E;
  int* header;   // [0] tiles, [1] blocks that have counted
  int* cursor;   // [E] counts, then the next free place of every expert's list
  int4* tiles;   // (expert, first place in list, routes, -)
  int32_t* list; // routes by expert
  // weights and output
  const uint8_t* kd;
  const uint8_t* ks;
  int64_t K, N;
  uint16_t* y;  // route outputs, 16-bit
  int out_dtype;
  bool y_vec;
};

__device__ __forceinline__ int64_t expert_of(const Product& p, int64_t r) {
  return p.sel_dtype == CVMM_I64 ? static_cast<const int64_t*>(p.sel)[r]
                                 : (int64_t) static_cast<const int32_t*>(p.sel)[r];
}

// A route whose id names no expert: reported, and its output is zero.
__device__ __noinline__ void bad_route(const Product& p, int64_t r, int64_t e) {
  report(CVMM_DEV_BAD_INDEX, kBadIdTag, (long long)e);
  for (int64_t n = 0; n < p.N; ++n) p.y[r * p.N + n] = 0;
}

// From counts[E] in shared memory: counts[e] becomes the start of expert e's
// list, tstart[e] its first tile; writes the tile table and the tile count.
__device__ void plan_tiles(const Product& p, int* counts, int* tstart, int* scratch) {
  const int t = threadIdx.x, per = (p.E + kPlanThreads - 1) / kPlanThreads;
  const int e0 = min(t * per, p.E), e1 = min(e0 + per, p.E);
  int routes = 0, tiles = 0;
  for (int e = e0; e < e1; ++e) {
    routes += counts[e];
    tiles += (counts[e] + kTile - 1) / kTile;
  }
  int place = block_exclusive_scan(routes, scratch);
  int tile = block_exclusive_scan(tiles, scratch);
  if (t == kPlanThreads - 1) {
    tstart[p.E] = tile + tiles;
    scratch[33] = place + routes;
  }
  for (int e = e0; e < e1; ++e) {
    const int c = counts[e];
    counts[e] = place;
    tstart[e] = tile;
    place += c;
    tile += (c + kTile - 1) / kTile;
  }
  __syncthreads();
  const int total = tstart[p.E];
  for (int i = t; i < total; i += kPlanThreads) {
    int lo = 0, hi = p.E - 1;  // last expert with tstart <= i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tstart[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const int at = counts[lo] + (i - tstart[lo]) * kTile;
    const int end = lo + 1 < p.E ? counts[lo + 1] : scratch[33];
    p.tiles[i] = make_int4(lo, at, min(kTile, end - at), 0);
  }
  if (t == 0) p.header[0] = total;
  __syncthreads();
}

// Block 0 .. plan_blocks - 1 count (and, alone, list) routes; the others
// quantise x: 16 lanes take 128 values of a row as quantize_k_kernel does, but
// scale cells stay in row order, which is how a gathered tile reads them.
__global__ void __launch_bounds__(kPlanThreads) prepare_kernel(const Product p, int plan_blocks) {
  pdl_enter();
  extern __shared__ int sh[];  // counts[E], tstart[E + 1], 34 ints of scratch
  const int t = threadIdx.x;
  if ((int)blockIdx.x < plan_blocks) {
    int* counts = sh;
    int* tstart = sh + p.E;
    int* scratch = tstart + p.E + 1;
    for (int e = t; e < p.E; e += kPlanThreads) counts[e] = 0;
    __syncthreads();
    const int64_t r0 = blockIdx.x * kPlanChunk, r1 = imin64(r0 + kPlanChunk, p.R);
    for (int64_t r = r0 + t; r < r1; r += kPlanThreads) {
      const int64_t e = expert_of(p, r);
      if (e >= 0 && e < p.E) atomicAdd(&counts[e], 1);
    }
    __syncthreads();
    if (plan_blocks == 1) {
      plan_tiles(p, counts, tstart, scratch);
      for (int64_t r = r0 + t; r < r1; r += kPlanThreads) {
        const int64_t e = expert_of(p, r);
        if (e >= 0 && e < p.E) p.list[atomicAdd(&counts[e], 1)] = (int32_t)r;
        else bad_route(p, r, e);
      }
      return;
    }
    for (int e = t; e < p.E; e += kPlanThreads)
      if (counts[e]) atomicAdd(&p.cursor[e], counts[e]);
    __threadfence();
    __syncthreads();
    if (t == 0) scratch[32] = atomicAdd(&p.header[1], 1);
    __syncthreads();
    if (scratch[32] != plan_blocks - 1) return;
    __threadfence();
    for (int e = t; e < p.E; e += kPlanThreads) counts[e] = __ldcg(&p.cursor[e]);
    __syncthreads();
    plan_tiles(p, counts, tstart, scratch);
    for (int e = t; e < p.E; e += kPlanThreads) p.cursor[e] = counts[e];
    return;
  }
  const int64_t rb = row_bytes(p.K), items = p.x_rows * p.cells;
  const int sub = t & 15;
  const int64_t stride = (int64_t)(gridDim.x - plan_blocks) * (kPlanThreads / 16);
  const int64_t rounds = (items + stride - 1) / stride;
  for (int64_t i = 0; i < rounds; ++i) {
    const int64_t it = (int64_t)(blockIdx.x - plan_blocks) * (kPlanThreads / 16) + (t >> 4) + i * stride;
    const bool live = it < items;
    const int64_t r = live ? it / p.cells : 0, c = live ? it - r * p.cells : 0;
    const int64_t k0 = c * 128 + sub * 8;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    if (live && k0 < p.K) {
      const int64_t at = r * p.x_ld + k0;
      if (p.x_vec && k0 + 8 <= p.K) {
        load8(static_cast<const char*>(p.x) + at * dtype_bytes(p.x_dtype), p.x_dtype, f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k0 + j < p.K) f[j] = load_as_float(p.x, p.x_dtype, at + j);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, magnitude(f[j]));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const bool in = live && c * 128 + (sub & 12) * 8 < p.K;
    const uint32_t byte = in ? scale_byte(m) : 0u;
    if (in) *reinterpret_cast<uint32_t*>(p.xd + r * rb + k0 / 2) = pack8(f, inverse_scale(byte));
    uint32_t cell = byte << (8 * ((sub >> 2) & 3));
    cell |= __shfl_xor_sync(0xffffffffu, cell, 4);
    cell |= __shfl_xor_sync(0xffffffffu, cell, 8);
    if (live && sub == 0) *reinterpret_cast<uint32_t*>(p.xs + it * 4) = cell;
  }
}

// Lists the routes counted by prepare: a block reserves its places of every
// expert at once and hands them out in shared memory.
__global__ void __launch_bounds__(kPlanThreads) fill_kernel(const Product p) {
  pdl_enter();
  extern __shared__ int sh[];  // counts[E]
  const int t = threadIdx.x;
  for (int e = t; e < p.E; e += kPlanThreads) sh[e] = 0;
  __syncthreads();
  const int64_t r0 = blockIdx.x * kPlanChunk, r1 = imin64(r0 + kPlanChunk, p.R);
  for (int64_t r = r0 + t; r < r1; r += kPlanThreads) {
    const int64_t e = expert_of(p, r);
    if (e >= 0 && e < p.E) atomicAdd(&sh[e], 1);
  }
  __syncthreads();
  for (int e = t; e < p.E; e += kPlanThreads)
    if (sh[e]) sh[e] = atomicAdd(&p.cursor[e], sh[e]);
  __syncthreads();
  for (int64_t r = r0 + t; r < r1; r += kPlanThreads) {
    const int64_t e = expert_of(p, r);
    if (e >= 0 && e < p.E) p.list[atomicAdd(&sh[e], 1)] = (int32_t)r;
    else bad_route(p, r, e);
  }
}

// ------------------------------------------------------------------ gemm
// Persistent, one CTA an SM, tiles of 128 routes x BN columns round-robin.
//   warp 0      gathers the tile's rows: 4 rows x 128 bytes (256 values) an
//               instruction, only the lanes that have rows;
//   warp 1      gathers their scale cells, 16 bytes a row ahead in registers,
//               and lays them out as tensor memory wants them: lane l takes rows
//               l, l + 32, l + 64, l + 96, whose cells are 16 consecutive bytes;
//   warp 2      lane 0 loads the weight tile (TMA) and its scales (bulk copies
//               of whole 512-byte pieces);
//   warp 3      allocates tensor memory; lane 0 copies each stage's scales there
//               (their own columns for every stage, so a copy never meets an MMA
//               that still reads) and issues the MMAs, K = 64 each;
//   warps 4-11  two groups read half the accumulator's columns each, round and
//               store them through shared memory in 64-byte row pieces.
constexpr int kThreads = 384;
constexpr int kEpilogueWarps = 8;
constexpr uint32_t kStagePitch = 80;  // 64-byte row piece + 16: 16-byte accesses meet no bank twice

template <int BN, int S, int NACC>
struct Layout {
  static constexpr int np = BN < 128 ? 1 : BN / 128;  // 128-row scale pieces of a weight tile
  static constexpr uint32_t a_bytes = kTile * 128, b_bytes = BN * 128;
  static constexpr uint32_t stage = a_bytes + b_bytes;
  static constexpr uint32_t sa = S * stage;                   // [S][2 pieces]
  static constexpr uint32_t sb = sa + S * 2 * kPiece;         // [S][np][2 pieces]
  static constexpr uint32_t staging = sb + S * np * 2 * kPiece;
  static constexpr uint32_t bars = staging + kEpilogueWarps * 32 * kStagePitch;
  static constexpr uint32_t misc = bars + (2 * S + 5) * 8;
  static constexpr uint32_t alloc = misc + 16 + 1024;
  static constexpr uint32_t sf_cols = 8 + 8 * np;  // tensor-memory columns of a stage's scales
  static constexpr uint32_t need = NACC * BN + S * sf_cols;
  static constexpr uint32_t cols = need <= 256 ? 256 : 512;
  static_assert(need <= 512, "tensor memory");
  static_assert(alloc <= 232448, "shared memory");
};

// One warp's 32 rows x 32 columns, rounded to 16 bits: lane l holds row l,
// `off` its first element (-1: none). ncols is the same for the whole warp.
__device__ __forceinline__ void store_rows(uint16_t* y, int dtype, int64_t off, const float (&v)[32], int ncols,
                                           uint32_t stage, bool vec) {
  const int lane = threadIdx.x & 31;
  if (!vec || ncols < 32) {
    if (off >= 0) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) y[off + j] = float_to_bits(v[j], dtype);
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    ptx::st_shared_v4(stage + lane * kStagePitch + 16 * q, pack2(v[8 * q], v[8 * q + 1], dtype),
                      pack2(v[8 * q + 2], v[8 * q + 3], dtype), pack2(v[8 * q + 4], v[8 * q + 5], dtype),
                      pack2(v[8 * q + 6], v[8 * q + 7], dtype));
  __syncwarp();
  const int q = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (lane >> 2) + 8 * i;
    const int64_t o = __shfl_sync(0xffffffffu, off, r);
    uint32_t w0, w1, w2, w3;
    ptx::ld_shared_v4(stage + r * kStagePitch + 16 * q, w0, w1, w2, w3);
    if (o >= 0) *reinterpret_cast<uint4*>(y + o + 8 * q) = make_uint4(w0, w1, w2, w3);
  }
  __syncwarp();
}

template <int BN, int S, int NACC>
__global__ void __launch_bounds__(kThreads, 1)
gemm_kernel(const Product p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            int n_n) {
  using L = Layout<BN, S, NACC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = umma::align_smem(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t* empty = full + S;
  uint64_t* accf = empty + S;
  uint64_t* acce = accf + 2;
  uint64_t* drain = acce + 2;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::misc);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::misc + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(&full[s], 3);  // rows, their scales, the weight tile
      ptx::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&accf[a], 1);
      ptx::mbar_init(&acce[a], kEpilogueWarps);
    }
    ptx::mbar_init(drain, 1);
    *abort = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 3) {
    ptx::tmem_alloc(const_cast<uint32_t*>(tmem_slot), L::cols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  const int total = p.header[0] * n_n;
  const int rb = (int)row_bytes(p.K), nkb = (rb + 127) / 128, kp = (int)pieces(p.K);
  auto tile = [&](int tt) -> int4 { return tt < total ? p.tiles[tt / n_n] : make_int4(0, 0, 0, 0); };
  const uint32_t base = ptx::smem_u32(smem);

  if (warp == 0) {
    // ------------------------------------------------------------ rows
    auto rows_of = [&](const int4& u, int (&r)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = 4 * lane + q;
        r[q] = i < u.z ? (int)((uint32_t)p.list[u.y + i] / (uint32_t)p.per_row) : -1;
      }
    };
    int4 u = tile(blockIdx.x);
    int rows[4], next[4];
    rows_of(u, rows);
    uint32_t it = 0;
    bool ok = true;
    for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x) {
      const int4 un = tile(tt + gridDim.x);
      rows_of(un, next);
      const int lanes = (u.z + 3) / 4;
      for (int kb = 0; kb < nkb; ++kb, ++it) {
        const int s = it % S;
        if (it >= S && !ptx::mbar_wait_or_abort(&empty[s], ((it / S) - 1) & 1, kTagEmpty, abort)) {
          ok = false;
          break;
        }
        if (lane == 0) ptx::mbar_arrive_expect_tx(&full[s], lanes * 512);
        __syncwarp();
        if (lane < lanes)
          ptx::tma_gather4(base + s * L::stage + lane * 512, &map_a, &full[s], kb * 128, rows[0], rows[1], rows[2],
                           rows[3]);
      }
      u = un;
#pragma unroll
      for (int q = 0; q < 4; ++q) rows[q] = next[q];
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ scales of the rows
    // Loads run three 16-byte chunks (of 512 values, two stages) ahead of the
    // stores, across tiles, so that their latency hides behind the stages.
    const int chunks = (nkb + 1) / 2;
    const uint4* src[4];
    int4 lu;                 // tile of the next load
    int lt = blockIdx.x, lc = 0;
    auto open = [&]() {
      lu = tile(lt);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = lane + 32 * q;
        src[q] = i < lu.z ? reinterpret_cast<const uint4*>(
                                p.xs + (int64_t)((uint32_t)p.list[lu.y + i] / (uint32_t)p.per_row) * p.cells * 4)
                          : nullptr;
      }
    };
    auto load = [&](uint4 (&v)[4]) {
      if (lt >= total) return;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = src[q] ? src[q][lc] : make_uint4(0, 0, 0, 0);
      if (++lc == chunks) {
        lc = 0;
        lt += gridDim.x;
        if (lt < total) open();
      }
    };
    uint4 v0[4] = {}, v1[4] = {}, v2[4] = {};
    if (lt < total) open();
    load(v0);
    load(v1);
    load(v2);
    uint32_t it = 0;
    bool ok = true;
    for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x) {
      for (int c = 0; c < chunks && ok; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (2 * c + h >= nkb) break;
          const int s = it % S;
          if (it >= S && !ptx::mbar_wait_or_abort(&empty[s], ((it / S) - 1) & 1, kTagEmpty, abort)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + L::sa + s * 2 * kPiece + lane * 16;
          if (h == 0) {
            ptx::st_shared_v4(dst, v0[0].x, v0[1].x, v0[2].x, v0[3].x);
            ptx::st_shared_v4(dst + kPiece, v0[0].y, v0[1].y, v0[2].y, v0[3].y);
          } else {
            ptx::st_shared_v4(dst, v0[0].z, v0[1].z, v0[2].z, v0[3].z);
            ptx::st_shared_v4(dst + kPiece, v0[0].w, v0[1].w, v0[2].w, v0[3].w);
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&full[s]);
          ++it;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v0[q] = v1[q];
          v1[q] = v2[q];
        }
        load(v2);
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ weight tiles
    if (lane == 0) {
      const int np_all = (int)pieces(p.N);
      const int64_t per_expert = scale_bytes(p.N, p.K);
      uint32_t it = 0;
      bool ok = true;
      int4 u = tile(blockIdx.x);
      for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x) {
        const int4 un = tile(tt + gridDim.x);
        const int n0 = tt % n_n * BN, np = min(L::np, np_all - n0 / 128);
        const uint8_t* sc = p.ks + u.x * per_expert + (int64_t)(n0 / 128) * kp * kPiece;
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % S;
          if (it >= S && !ptx::mbar_wait_or_abort(&empty[s], ((it / S) - 1) & 1, kTagEmpty, abort)) {
            ok = false;
            break;
          }
          const uint32_t bytes = min(2, kp - 2 * kb) * kPiece;
          ptx::mbar_arrive_expect_tx(&full[s], L::b_bytes + np * bytes);
          ptx::tma_load_3d(base + s * L::stage + L::a_bytes, &map_b, &full[s], kb * 128, n0, u.x);
          for (int q = 0; q < np; ++q)
            ptx::bulk_load(base + L::sb + (s * L::np + q) * 2 * kPiece, sc + ((int64_t)q * kp + 2 * kb) * kPiece, bytes,
                           &full[s]);
        }
        u = un;
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------ MMAs
    if (lane == 0) {
      const int np_all = (int)pieces(p.N);
      uint32_t it = 0;
      int local = 0;
      bool ok = true;
      for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x, ++local) {
        const int a = local % NACC;
        if (local >= NACC && !ptx::mbar_wait_or_abort(&acce[a], (local / NACC - 1) & 1, kTagAccEmpty, abort)) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + a * BN;
        const int n0 = tt % n_n * BN, np = min(L::np, np_all - n0 / 128);
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % S;
          if (!ptx::mbar_wait_or_abort(&full[s], (it / S) & 1, kTagFull, abort)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t sa = tmem + NACC * BN + s * L::sf_cols, sb = sa + 8;
          const int pc = min(2, kp - 2 * kb);
          for (int c = 0; c < pc; ++c) {
            ptx::tmem_cp_scales(sa + 4 * c, ptx::smem_desc_rows16(base + L::sa + (s * 2 + c) * kPiece));
            for (int q = 0; q < np; ++q)
              ptx::tmem_cp_scales(sb + 4 * (c * L::np + q),
                                  ptx::smem_desc_rows16(base + L::sb + ((s * L::np + q) * 2 + c) * kPiece));
          }
          const uint32_t a_u = base + s * L::stage, b_u = a_u + L::a_bytes;
          const int steps = min(4, (rb - kb * 128 + 31) / 32);
          // A 64-column tile reads the upper half of its 128-row scale piece at odd positions.
          const uint32_t half = BN == 64 ? (n0 / 64 % 2) * 2 : 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < steps)
              ptx::mma_mxf4(d, ptx::smem_desc_sw128(a_u + j * 32, 16, 1024), ptx::smem_desc_sw128(b_u + j * 32, 16, 1024),
                            ptx::instr_desc_mxf4(kTile, BN, (j & 1) * 2), sa + 4 * (j >> 1),
                            sb + 4 * (j >> 1) * L::np + half, (kb | j) != 0);
          }
          ptx::mma_commit(&empty[s]);
        }
        if (ok) ptx::mma_commit(&accf[a]);
      }
      // Everything issued must finish before tensor memory is released.
      ptx::mma_commit(drain);
      ptx::mbar_wait(drain, 0, kTagDrain);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3, group = (warp - 4) >> 2;
    const uint32_t stage = base + L::staging + (warp - 4) * 32 * kStagePitch;
    auto route_of = [&](const int4& u) -> int {
      const int i = quad * 32 + lane;
      return i < u.z ? p.list[u.y + i] : -1;
    };
    int route = route_of(tile(blockIdx.x));
    int local = 0;
    for (int tt = blockIdx.x; tt < total; tt += gridDim.x, ++local) {
      const int route_next = route_of(tile(tt + gridDim.x));
      const int a = local % NACC;
      const int64_t n0 = (int64_t)(tt % n_n) * BN;
      if (!ptx::mbar_wait_or_abort(&accf[a], (local / NACC) & 1, kTagAccFull, abort)) break;
      ptx::tc_fence_after();
      const int64_t off = route < 0 ? -1 : (int64_t)route * p.N + n0;
      for (int c = group * (BN / 2); c < (group + 1) * (BN / 2); c += 32) {
        if (n0 + c >= p.N) break;
        float v[32];
        umma::load_acc32(tmem + ((uint32_t)(quad * 32) << 16) + a * BN + c, v);
        store_rows(p.y, p.out_dtype, off < 0 ? -1 : off + c, v, (int)imin64(32, p.N - n0 - c), stage, p.y_vec);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&acce[a]);
      route = route_next;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort) {
    // A role gave up: copies already issued land well within this time.
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000) __nanosleep(1000);
  }
  if (warp == 3) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, L::cols);
  }
}

// out[t] = sum_j w[t, j] y[t k + j] in 32 bits, j ascending; 8 columns a thread.
__global__ void __launch_bounds__(256)
combine_kernel(const uint16_t* __restrict__ y, const void* __restrict__ w, int w_dtype, int64_t T, int64_t k, int64_t N,
               void* __restrict__ out, int dtype, bool vec) {
  pdl_enter();
  const int64_t groups = (N + 7) / 8;
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= T * groups) return;
  const int64_t t = i / groups, n0 = (i - t * groups) * 8;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const uint16_t* row = y + t * k * N + n0;
  if (vec) {
    for (int64_t j0 = 0; j0 < k; j0 += 4) {
      uint4 q[4];
      float wj[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j0 + u < k) q[u] = *reinterpret_cast<const uint4*>(row + (j0 + u) * N);
#pragma unroll
      for (int u = 0; u < 4; ++u) wj[u] = j0 + u < k ? load_as_float(w, w_dtype, t * k + j0 + u) : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u >= k) break;
        const uint32_t d[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          acc[2 * c] = fmaf(wj[u], bits_to_float((uint16_t)(d[c] & 0xffffu), dtype), acc[2 * c]);
          acc[2 * c + 1] = fmaf(wj[u], bits_to_float((uint16_t)(d[c] >> 16), dtype), acc[2 * c + 1]);
        }
      }
    }
    store8(reinterpret_cast<char*>(out) + (t * N + n0) * 2, dtype, acc);
  } else {
    for (int64_t j = 0; j < k; ++j) {
      const float wj = load_as_float(w, w_dtype, t * k + j);
      for (int c = 0; c < 8 && n0 + c < N; ++c) acc[c] = fmaf(wj, bits_to_float(row[j * N + c], dtype), acc[c]);
    }
    for (int c = 0; c < 8 && n0 + c < N; ++c) store_from_float(out, dtype, t * N + n0 + c, acc[c]);
  }
}

// ------------------------------------------------------------------ host side
// Byte maps of 128-byte pieces (256 values) in the 128-byte swizzle.
static bool rows_map(CUtensorMap* map, const void* base, int64_t rb, int64_t rows) {
  auto fn = umma::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)rb, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)rb};
  cuuint32_t box[2] = {128, 1}, estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool weights_map(CUtensorMap* map, const void* base, int64_t rb, int64_t N, int64_t E, int bn) {
  auto fn = umma::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)rb, (cuuint64_t)N, (cuuint64_t)E};
  cuuint64_t strides[2] = {(cuuint64_t)rb, (cuuint64_t)(rb * N)};
  cuuint32_t box[3] = {128, (cuuint32_t)bn, 1}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, int S, int NACC>
static int launch_gemm(const Product& p, int64_t max_tiles, cudaStream_t stream) {
  using L = Layout<BN, S, NACC>;
  CUtensorMap a, b;
  if (!rows_map(&a, p.xd, row_bytes(p.K), p.x_rows) || !weights_map(&b, p.kd, row_bytes(p.K), p.N, p.E, BN))
    return fail(CVMM_ERR_LAUNCH, "cvmm_mx_forward: tensor map");
  if (int rc = umma::set_smem(gemm_kernel<BN, S, NACC>, L::alloc)) return rc;
  const int n_n = (int)((p.N + BN - 1) / BN);
  const unsigned grid = (unsigned)std::min<int64_t>(max_tiles * n_n, umma::sm_count());
  launch(gemm_kernel<BN, S, NACC>, grid, kThreads, L::alloc, stream, p, a, b, n_n);
  return check_launch("cvmm_mx_forward: gemm");
}

// Workspace of one call, in order.
struct Sizes {
  size_t header, cursor, tiles, list, xd, xs, y, total;
  int64_t cells, max_tiles;
};
static Sizes sizes(int64_t x_rows, int64_t R, int64_t E, int64_t K, int64_t N, bool weighted) {
  Sizes z;
  z.cells = (pieces(K) + 3) / 4 * 4;
  z.max_tiles = R / kTile + std::min(E, R);
  z.header = 256;
  z.cursor = align_up((size_t)E * 4, 256);
  z.tiles = align_up((size_t)z.max_tiles * sizeof(int4), 256);
  z.list = align_up((size_t)R * 4, 256);
  z.xd = align_up((size_t)(x_rows * row_bytes(K)), 256);
  z.xs = align_up((size_t)(x_rows * z.cells * 4), 256);
  z.y = weighted ? align_up((size_t)(R * N) * 2, 256) : 0;
  z.total = z.header + z.cursor + z.tiles + z.list + z.xd + z.xs + z.y + 256;
  return z;
}

}  // namespace mx
}  // namespace cvmm

extern "C" {

size_t cvmm_mx_workspace_size(int64_t x_rows, int64_t n_routes, int64_t n_experts, int64_t k_dim, int64_t n_dim,
                              int weighted) {
  if (x_rows < 0 || n_routes < 0 || n_experts < 0 || k_dim < 0 || n_dim < 0) return 0;
  return cvmm::mx::sizes(x_rows, n_routes, n_experts, k_dim, n_dim, weighted != 0).total;
}

int cvmm_mx_forward(const void* x, int x_dtype, int64_t x_rows, int64_t x_ld, const void* sel, int sel_dtype,
                    int64_t n_routes, int64_t top_k, const void* w, int w_dtype, const uint8_t* keys_data,
                    const uint8_t* keys_scale, int64_t n_experts, int64_t k_dim, int64_t n_dim, void* out,
                    int out_dtype, void* workspace, size_t workspace_bytes, cvmm_stream_t stream) {
  using namespace cvmm;
  if (!is_float_dtype(x_dtype) || (w && !is_float_dtype(w_dtype)) || (out_dtype != CVMM_BF16 && out_dtype != CVMM_F16))
    return fail(CVMM_ERR_UNSUPPORTED_DTYPE, "cvmm_mx_forward: x and w must be float tensors, out bf16 or fp16");
  if (sel_dtype != CVMM_I64 && sel_dtype != CVMM_I32)
    return fail(CVMM_ERR_UNSUPPORTED_DTYPE, "cvmm_mx_forward: sel must be int64 or int32");
  if (x_rows < 0 || n_routes < 0 || top_k < 1 || n_experts < 1 || k_dim < 1 || n_dim < 1 || x_ld < k_dim ||
      n_routes % top_k != 0 || (n_routes > 0 && (x_rows < 1 || n_routes % x_rows != 0)))
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_forward: bad sizes");
  if (n_experts > mx::kMaxExperts) return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_forward: more than 4096 experts");
  if (n_routes == 0) return CVMM_OK;
  // Routes, K and N are 32-bit indices in the kernels, and so is tiles x column tiles.
  if (n_routes > (int64_t)INT32_MAX || k_dim > (int64_t)1 << 24 || n_dim > (int64_t)1 << 24 ||
      (n_routes / mx::kTile + std::min(n_experts, n_routes)) * ((n_dim + 63) / 64) > (int64_t)INT32_MAX / 2)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_forward: too many routes, k or n");
  if (!x || !sel || !keys_data || !keys_scale || !out)
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_forward: null pointer");
  if (!al16(keys_data) || !al16(keys_scale))
    return fail(CVMM_ERR_INVALID_ARG, "cvmm_mx_forward: keys must be 16-byte aligned");
  const mx::Sizes z = mx::sizes(x_rows, n_routes, n_experts, k_dim, n_dim, w != nullptr);
  if (!workspace || workspace_bytes < z.total)
    return fail(CVMM_ERR_WORKSPACE, "cvmm_mx_forward: workspace too small");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>(align_up((size_t)workspace, 256));
  auto take = [&](size_t bytes) {
    char* at = ws;
    ws += bytes;
    return at;
  };
  mx::Product p = {};
  p.x = x; p.x_dtype = x_dtype; p.x_rows = x_rows; p.x_ld = x_ld;
  p.x_vec = al16(x) && x_ld * (int64_t)dtype_size(x_dtype) % 16 == 0;
  p.per_row = (int)(n_routes / x_rows);
  p.cells = z.cells;
  p.sel = sel; p.sel_dtype = sel_dtype; p.R = n_routes; p.E = (int)n_experts;
  p.header = reinterpret_cast<int*>(take(z.header));
  p.cursor = reinterpret_cast<int*>(take(z.cursor));
  p.tiles = reinterpret_cast<int4*>(take(z.tiles));
  p.list = reinterpret_cast<int32_t*>(take(z.list));
  p.xd = reinterpret_cast<uint8_t*>(take(z.xd));
  p.xs = reinterpret_cast<uint8_t*>(take(z.xs));
  p.y = reinterpret_cast<uint16_t*>(w ? take(z.y) : static_cast<char*>(out));
  p.kd = keys_data; p.ks = keys_scale; p.K = k_dim; p.N = n_dim;
  p.out_dtype = out_dtype;
  p.y_vec = n_dim % 8 == 0 && al16(p.y);

  const int plan_blocks = (int)((n_routes + mx::kPlanChunk - 1) / mx::kPlanChunk);
  const int quant_blocks = grid_for(x_rows * z.cells, mx::kPlanThreads / 16);
  const size_t plan_smem = (size_t)(2 * n_experts + 1 + 34) * sizeof(int);
  if (plan_blocks > 1 && cudaMemsetAsync(p.header, 0, z.header + z.cursor, s) != cudaSuccess)
    return fail_cuda("cvmm_mx_forward: memset");
  launch(mx::prepare_kernel, plan_blocks + quant_blocks, mx::kPlanThreads, plan_smem, s, p, plan_blocks);
  if (plan_blocks > 1) launch(mx::fill_kernel, plan_blocks, mx::kPlanThreads, (size_t)n_experts * sizeof(int), s, p);
  if (int rc = check_launch("cvmm_mx_forward: prepare")) return rc;
  const int64_t m_tiles = std::max(n_routes / mx::kTile, std::min(n_experts, n_routes));
  int rc;
  if (n_dim > 128 && m_tiles * ((n_dim + 255) / 256) >= 148) rc = mx::launch_gemm<256, 4, 1>(p, z.max_tiles, s);
  else if (n_dim > 64 && m_tiles * ((n_dim + 127) / 128) >= 148) rc = mx::launch_gemm<128, 6, 2>(p, z.max_tiles, s);
  else rc = mx::launch_gemm<64, 7, 2>(p, z.max_tiles, s);
  if (rc || !w) return rc;
  const int64_t T = n_routes / top_k;
  launch(mx::combine_kernel, (unsigned)((T * ((n_dim + 7) / 8) + 255) / 256), 256, 0, s, p.y, w, w_dtype, T, top_k,
         n_dim, out, out_dtype, n_dim % 8 == 0 && al16(out));
  return check_launch("cvmm_mx_forward: combine");
}

}  // extern "C"
