// Expert product of 4-bit rows with 4-bit expert weights (cvmm_mx_forward).
//
//   y[r] = Q(x[r / per_row]) . W[sel[r]]^T;  out[r] = y[r], or with weights
//   out[t] = sum_j w[t, j] y[t top_k + j]
//
// Three or four launches:
//   prepare  quantises the rows of x once, in their own order (4 bits a value,
//            so that all route copies of a row are reads of the same bytes), and
//            lists the routes of every expert and the 128-route tiles they make;
//   fill     (many routes only) writes the lists that prepare laid out;
//   gemm     gathers a tile's rows and multiplies them with the
//            expert's weight tiles on the tensor cores, scales and all;
//   combine  (weights only) sums the route outputs, which the gemm then leaves in
//            32 bits: the sum is rounded once, and a route output past the 16-bit
//            range does not spoil a sum within it.
// The order of the routes within an expert's list is left to atomics: a row's
// output does not depend on where in a tile it stands.
#include "launch.h"
#include "mx.cuh"
#include "ptx.cuh"

namespace cvmm {
namespace mx {

constexpr int kTile = 128;           // routes of a tile (MMA M)
constexpr int64_t kMaxExperts = 4096;
constexpr int kPlanThreads = 512;
constexpr int64_t kPlanAlone = 4096;  // routes up to which one block ranks and lists them all
constexpr int64_t kPlanChunk = 1024;  // else routes of a block (16384 routes: 8.5 us at 1024, 11.8 at 4096)
constexpr int kBadIdTag = 31;         // status-word site: an expert id outside [0, n_experts)
enum : int { kTagEmpty = 40, kTagFull = 41, kTagAccFull = 42, kTagAccEmpty = 43, kTagDrain = 44 };

struct Product {
  // x
  const void* x;
  int x_dtype;
  int64_t x_rows, x_ld;
  int x_vec;
  Divisor per_row;  // routes that share a row
  uint8_t* xd;  // [x_rows][row_bytes]
  uint8_t* xs;  // [x_rows][cells] of 4 scale bytes, an even number of cells
  int64_t cells;
  // routing
  const void* sel;
  int sel_dtype;
  int64_t R;
  int E;
  int* header;   // [0] tiles, [1] blocks that have ranked their routes
  int* cursor;   // [E] counts, then the start of every expert's list
  int4* tiles;   // (expert, first place in list, routes, -)
  int32_t* list; // routes by expert
  int2* rank;    // (expert, place in its list) of every route, when several blocks rank
  // weights and output
  const uint8_t* kd;
  const uint8_t* ks;
  int64_t K, N;
  void* y;  // route outputs: 16-bit in out_dtype, or 32-bit for combine
  int64_t y_words;  // 16-bit words of a row of y: N, or 2 N
  int out_dtype;
  bool y_vec;
};

__device__ __forceinline__ int64_t expert_of(const Product& p, int64_t r) {
  return p.sel_dtype == CVMM_I64 ? static_cast<const int64_t*>(p.sel)[r]
                                 : (int64_t) static_cast<const int32_t*>(p.sel)[r];
}

// A route whose id names no expert: reported, and its output is zero.
// What it needs of registers prepare_kernel reserves (a choice by width here made
// that 47 for 40, two blocks an SM for three: 65 us for 57, 32768 tokens x 4096).
__device__ __noinline__ void bad_route(const Product& p, int64_t r, int64_t e) {
  report(CVMM_DEV_BAD_INDEX, kBadIdTag, (long long)e);
  for (int64_t n = 0; n < p.y_words; ++n) static_cast<uint16_t*>(p.y)[r * p.y_words + n] = 0;
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

// The up to kPer routes of a thread among r0 .. r1 - 1: their experts, -1 for
// none or an id out of range (reported and zeroed, once a call).
constexpr int kPer = (int)(kPlanAlone / kPlanThreads);
__device__ __forceinline__ void my_routes(const Product& p, int64_t r0, int64_t r1, int (&e)[kPer]) {
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int64_t r = r0 + threadIdx.x + j * kPlanThreads;
    int64_t v = -1;
    if (r < r1) {
      v = expert_of(p, r);
      if (v < 0 || v >= p.E) {
        bad_route(p, r, v);
        v = -1;
      }
    }
    e[j] = (int)v;
  }
}

// Blocks 0 .. plan_blocks - 1 rank their routes within their experts; the last
// of them to finish lays out the lists and tiles (and a lone one writes its
// list, too). The other blocks quantise x; scale cells stay in row order,
// which is how a gathered tile reads them.
template <int DT>
__global__ void __launch_bounds__(kPlanThreads)
prepare_kernel(const __grid_constant__ Product p, int plan_blocks, Divisor by_blocks) {
  pdl_enter();
  extern __shared__ int sh[];  // counts[E], tstart[E + 1], 34 ints of scratch
  const int t = threadIdx.x;
  if ((int)blockIdx.x < plan_blocks) {
    int* counts = sh;
    int* tstart = sh + p.E;
    int* scratch = tstart + p.E + 1;
    const int64_t r0 = blockIdx.x * kPlanChunk, r1 = plan_blocks == 1 ? p.R : imin64(r0 + kPlanChunk, p.R);
    int e[kPer], rank[kPer];
    my_routes(p, r0, r1, e);
    for (int i = t; i < p.E; i += kPlanThreads) counts[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) rank[j] = e[j] >= 0 ? atomicAdd(&counts[e[j]], 1) : 0;
    __syncthreads();
    if (plan_blocks == 1) {
      plan_tiles(p, counts, tstart, scratch);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (e[j] >= 0) p.list[counts[e[j]] + rank[j]] = (int32_t)(r0 + t + j * kPlanThreads);
      return;
    }
    // This block's places within every expert's list.
    for (int i = t; i < p.E; i += kPlanThreads)
      if (counts[i]) counts[i] = atomicAdd(&p.cursor[i], counts[i]);
    __threadfence();
    __syncthreads();
    if (t == 0) scratch[32] = atomicAdd(&p.header[1], 1);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t r = r0 + t + j * kPlanThreads;
      if (r < r1) p.rank[r] = e[j] >= 0 ? make_int2(e[j], counts[e[j]] + rank[j]) : make_int2(-1, 0);
    }
    __syncthreads();
    if (scratch[32] != plan_blocks - 1) return;
    __threadfence();
    for (int i = t; i < p.E; i += kPlanThreads) counts[i] = __ldcg(&p.cursor[i]);
    __syncthreads();
    plan_tiles(p, counts, tstart, scratch);
    for (int i = t; i < p.E; i += kPlanThreads) p.cursor[i] = counts[i];
    return;
  }
  const int64_t rb = row_bytes(p.K), blocks = by_blocks.d;  // 4 a cell
  auto at = [&](int64_t it) -> Block {
    const int64_t r = by_blocks.of(it);
    return {r * p.x_ld, p.xd + r * rb, reinterpret_cast<uint32_t*>(p.xs + (it & ~(int64_t)3)), it - r * blocks, true};
  };
  quantize_blocks<DT>(p.x, p.K, p.x_vec, p.x_rows * blocks,
                      (int64_t)(blockIdx.x - plan_blocks) * kPlanThreads + t,
                      (int64_t)(gridDim.x - plan_blocks) * kPlanThreads, at);
}

// Writes the lists that several blocks of prepare ranked.
__global__ void __launch_bounds__(256) fill_kernel(const __grid_constant__ Product p) {
  pdl_enter();
  const int64_t r = blockIdx.x * 256ll + threadIdx.x;
  if (r >= p.R) return;
  const int2 er = p.rank[r];
  if (er.x >= 0) p.list[p.cursor[er.x] + er.y] = (int32_t)r;
}

// ------------------------------------------------------------------ gemm
// Persistent, one CTA an SM, tiles of 128 routes x BN columns round-robin.
//   warps 0-3   gather the tile's rows, 16 bytes a copy into the 128-byte
//               swizzle, and their scale cells, 4 bytes a copy into the order
//               tensor memory wants (row r's at 16 (r % 32) + 4 (r / 32)); only
//               rows that exist. The copies arrive on the stage's barrier by
//               themselves. (Gathers by TMA, 4 rows an instruction, took 567 us
//               where plain rows took 403, 32768 tokens 4096 -> 512; arrivals a
//               warp one or two stages late, 391 and 397 against 375.)
//   warp 4      lane 0 loads the weight tile (TMA) and its scales (bulk copies
//               of whole 512-byte pieces);
//   warp 5      allocates tensor memory; lane 0 copies each stage's scales there
//               (their own columns for every stage, so a copy never meets an MMA
//               that still reads) and issues the MMAs, K = 64 each;
//   warps 6-13  two groups read half the accumulator's columns each, round them
//               into registers, hand the accumulator back and only then store,
//               through shared memory in 64-byte row pieces. 32-bit outputs, twice
//               the registers, are stored 32 columns at a time straight from them
//               before the accumulator goes back (32 tokens 512 -> 4096, the whole
//               call: 32 us; through shared memory, 52).
constexpr int kProducers = 128;
constexpr int kLoadWarp = 4, kMmaWarp = 5, kEpilogueWarp = 6, kEpilogueWarps = 8;
constexpr int kThreads = 32 * (kEpilogueWarp + kEpilogueWarps);
constexpr uint32_t kStagePitch = 80;  // 64-byte row piece + 16: 16-byte accesses meet no bank twice

// Position in a ring of S stages: phase is the parity of the round, which is
// what a consumer waits for; a producer waits for the other one, and in the
// first round for nothing.
template <int S>
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  bool first = true;
  __device__ __forceinline__ void next() {
    if (++s == S) {
      s = 0;
      phase ^= 1u;
      first = false;
    }
  }
};

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

// One warp's 32 rows x 32 columns of 16-bit values, two to a word: lane l holds
// row l, `off` its first element (-1: none). ncols is the same for the whole warp.
__device__ __forceinline__ void store_rows(uint16_t* y, int64_t off, const uint32_t* v, int ncols, uint32_t stage,
                                           bool vec) {
  const int lane = threadIdx.x & 31;
  if (!vec || ncols < 32) {
    if (off >= 0) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) y[off + j] = (uint16_t)(j & 1 ? v[j >> 1] >> 16 : v[j >> 1] & 0xffffu);
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    ptx::st_shared_v4(stage + lane * kStagePitch + 16 * q, v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
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

// The same in 32 bits: every lane stores its own row, a whole sector an instruction.
__device__ __forceinline__ void store_rows(float* y, int64_t off, const uint32_t* v, int ncols, bool vec) {
  if (off >= 0) {
    if (vec && ncols >= 32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) st_v8(y + off + 8 * q, v + 8 * q);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < ncols) y[off + j] = __uint_as_float(v[j]);
    }
  }
  __syncwarp();
}

template <int BN, int S, int NACC, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1)
gemm_kernel(const __grid_constant__ Product p, const __grid_constant__ CUtensorMap map_b, int n_n) {
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
      ptx::mbar_init(&full[s], kProducers + 1);  // the rows' copies, the weight tile
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
  if (warp == kMmaWarp) {
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

  if (warp < 4) {
    // ------------------------------------------------------------ rows and their scales
    // Thread t copies 16-byte piece t % 8 of rows t / 8 + 16 i, and the scales
    // of row t. The next tile's rows are looked up during the current tile.
    const int t = threadIdx.x, piece = (t & 7) * 16;
    // The tile after the next is looked up, too, so that neither lookup is waited for.
    auto look = [&](const int4& u, int (&r)[8], int& sr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = (t >> 3) + 16 * i < u.z ? p.list[u.y + (t >> 3) + 16 * i] : -1;
      sr = t < u.z ? p.list[u.y + t] : -1;
    };
    auto row_of = [&](int route) -> int { return route < 0 ? -1 : (int)p.per_row.of(route); };
    int next[8], snext;
    int4 un = tile(blockIdx.x + gridDim.x);
    look(tile(blockIdx.x), next, snext);
    Ring<S> ring;
    bool ok = true;
    for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x) {
      int rows[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) rows[i] = row_of(next[i]);
      const int srow = row_of(snext);
      look(un, next, snext);
      un = tile(tt + 2 * gridDim.x);
      const uint8_t* src[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) src[i] = p.xd + (int64_t)max(rows[i], 0) * rb + piece;
      const uint8_t* scales = p.xs + (int64_t)max(srow, 0) * p.cells * 4;
      for (int kb = 0; kb < nkb; ++kb, ring.next()) {
        const int s = ring.s;
        if (!ring.first && !ptx::mbar_wait_or_abort(&empty[s], ring.phase ^ 1u, kTagEmpty, abort)) {
          ok = false;
          break;
        }
        const uint32_t a_u = base + s * L::stage;
        const bool in = kb * 128 + piece < rb;  // past the row's end: zeros
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (rows[i] >= 0)
            ptx::cp_async_16(a_u + umma::swz((t >> 3) + 16 * i, t & 7, 0), in ? src[i] + kb * 128 : p.xd, in ? 16 : 0);
        if (srow >= 0) {
          const uint32_t dst = base + L::sa + s * 2 * kPiece + (t & 31) * 16 + (t >> 5) * 4;
          ptx::cp_async_4(dst, scales + kb * 8);
          ptx::cp_async_4(dst + kPiece, scales + kb * 8 + 4);
        }
        ptx::cp_async_arrive_noinc(&full[s]);
      }
    }
    ptx::cp_async_wait_all();
  } else if (warp == kLoadWarp) {
    // ------------------------------------------------------------ weight tiles
    if (lane == 0) {
      const int np_all = (int)pieces(p.N);
      const int64_t per_expert = scale_bytes(p.N, p.K);
      Ring<S> ring;
      bool ok = true;
      int4 u = tile(blockIdx.x);
      for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x) {
        const int4 un = tile(tt + gridDim.x);
        const int n0 = tt % n_n * BN, np = min(L::np, np_all - n0 / 128);
        const uint8_t* sc = p.ks + u.x * per_expert + (int64_t)(n0 / 128) * kp * kPiece;
        for (int kb = 0; kb < nkb; ++kb, ring.next()) {
          const int s = ring.s;
          if (!ring.first && !ptx::mbar_wait_or_abort(&empty[s], ring.phase ^ 1u, kTagEmpty, abort)) {
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
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMAs
    if (lane == 0) {
      // One thread issues everything, so its instructions a stage count: ring
      // positions and descriptors are carried along, not computed.
      // (Copying the scales of stage i + 1 ahead of the MMAs of stage i, or two
      // stages' scales ahead of two stages' MMAs, was slower, 609 and 468 us:
      // copies and MMAs drain one another.)
      const int np_all = (int)pieces(p.N);
      const uint64_t a0 = ptx::smem_desc_sw128(base, 16, 1024), b0 = ptx::smem_desc_sw128(base + L::a_bytes, 16, 1024);
      const uint64_t sa0 = ptx::smem_desc_rows16(base + L::sa), sb0 = ptx::smem_desc_rows16(base + L::sb);
      const uint32_t sf0 = tmem + NACC * BN;
      Ring<S> ring;
      int local = 0;
      bool ok = true;
      for (int tt = blockIdx.x; tt < total && ok; tt += gridDim.x, ++local) {
        const int a = local % NACC;
        if (local >= NACC && !ptx::mbar_wait_or_abort(&acce[a], (local / NACC - 1) & 1, kTagAccEmpty, abort)) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + a * BN;
        const int n = tt % n_n, np = min(L::np, np_all - n * BN / 128);
        // A 64-column tile reads the upper half of its 128-row scale piece at odd positions.
        const uint32_t half = BN == 64 ? (n & 1) * 2 : 0;
        // pc scale pieces, `steps` MMAs of K = 64; both constant but for a row's last stage.
        auto stage = [&](int pc, int steps, bool add) {
          const uint32_t sa = sf0 + ring.s * L::sf_cols, sb = sa + 8;
          const uint64_t ad = a0 + ring.s * (L::stage / 16), bd = b0 + ring.s * (L::stage / 16);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c >= pc) break;
            ptx::tmem_cp_scales(sa + 4 * c, sa0 + (ring.s * 2 + c) * (kPiece / 16));
#pragma unroll
            for (int q = 0; q < L::np; ++q)
              if (q < np)
                ptx::tmem_cp_scales(sb + 4 * (c * L::np + q), sb0 + ((ring.s * L::np + q) * 2 + c) * (kPiece / 16));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= steps) break;
            ptx::mma_mxf4(d, ad + 2 * j, bd + 2 * j, ptx::instr_desc_mxf4(kTile, BN, (j & 1) * 2), sa + 4 * (j >> 1),
                          sb + 4 * (j >> 1) * L::np + half, add || j > 0);
          }
        };
        for (int kb = 0; kb < nkb; ++kb) {
          if (!ptx::mbar_wait_or_abort(&full[ring.s], ring.phase, kTagFull, abort)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          ptx::fence_proxy_async_smem();  // the rows came through the generic proxy
          if (kb + 1 < nkb) stage(2, 4, kb != 0);
          else stage(min(2, kp - 2 * kb), min(4, (rb - kb * 128 + 31) / 32), kb != 0);
          ptx::mma_commit(&empty[ring.s]);
          ring.next();
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
    const int quad = warp & 3, group = (warp - kEpilogueWarp) >> 2;
    const uint32_t stage = base + L::staging + (warp - kEpilogueWarp) * 32 * kStagePitch;
    auto route_of = [&](const int4& u) -> int {
      const int i = quad * 32 + lane;
      return i < u.z ? p.list[u.y + i] : -1;
    };
    int route = route_of(tile(blockIdx.x));
    int local = 0;
    for (int tt = blockIdx.x; tt < total; tt += gridDim.x, ++local) {
      const int route_next = route_of(tile(tt + gridDim.x));
      const int a = local % NACC;
      const int64_t n0 = (int64_t)(tt % n_n) * BN + group * (BN / 2);
      if (!ptx::mbar_wait_or_abort(&accf[a], (local / NACC) & 1, kTagAccFull, abort)) break;
      ptx::tc_fence_after();
      uint32_t v[WIDE ? 32 : BN / 4];
      const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + a * BN + group * (BN / 2);
#pragma unroll
      for (int c = 0; c < BN / 64; ++c) {
        if (n0 + 32 * c >= p.N) break;
        if constexpr (WIDE) {
          ptx::tmem_ld_32x32b_x32(from + 32 * c, v);
          ptx::tmem_wait_ld();
          store_rows(static_cast<float*>(p.y), route < 0 ? -1 : (int64_t)route * p.N + n0 + 32 * c, v,
                     (int)imin64(32, p.N - n0 - 32 * c), p.y_vec);
        } else {
          float f[32];
          umma::load_acc32(from + 32 * c, f);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[16 * c + j] = pack2(f[2 * j], f[2 * j + 1], p.out_dtype);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&acce[a]);
      if constexpr (!WIDE) {
        const int64_t off = route < 0 ? -1 : (int64_t)route * p.N + n0;
#pragma unroll
        for (int c = 0; c < BN / 64; ++c) {
          if (n0 + 32 * c >= p.N) break;
          store_rows(static_cast<uint16_t*>(p.y), off < 0 ? -1 : off + 32 * c, v + 16 * c,
                     (int)imin64(32, p.N - n0 - 32 * c), stage, p.y_vec);
        }
      }
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
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, L::cols);
  }
}

// out[t] = sum_j w[t, j] y[t k + j] in 32 bits, j ascending, rounded once; 8 columns a thread.
__global__ void __launch_bounds__(256)
combine_kernel(const float* __restrict__ y, const void* __restrict__ w, int w_dtype, int64_t T, int64_t k, int64_t N,
               void* __restrict__ out, int dtype, bool vec) {
  pdl_enter();
  const int64_t groups = (N + 7) / 8;
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= T * groups) return;
  const int64_t t = i / groups, n0 = (i - t * groups) * 8;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float* row = y + t * k * N + n0;
  if (vec) {
    for (int64_t j0 = 0; j0 < k; j0 += 4) {
      uint32_t q[4][8];
      float wj[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j0 + u < k) ld_v8(q[u], row + (j0 + u) * N);
#pragma unroll
      for (int u = 0; u < 4; ++u) wj[u] = j0 + u < k ? load_as_float(w, w_dtype, t * k + j0 + u) : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u >= k) break;
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = fmaf(wj[u], __uint_as_float(q[u][c]), acc[c]);
      }
    }
    store8(reinterpret_cast<char*>(out) + (t * N + n0) * 2, dtype, acc);
  } else {
    for (int64_t j = 0; j < k; ++j) {
      const float wj = load_as_float(w, w_dtype, t * k + j);
      for (int c = 0; c < 8 && n0 + c < N; ++c) acc[c] = fmaf(wj, row[j * N + c], acc[c]);
    }
    for (int c = 0; c < 8 && n0 + c < N; ++c) store_from_float(out, dtype, t * N + n0 + c, acc[c]);
  }
}

// ------------------------------------------------------------------ host side
// Byte map of the weights: boxes of 128 bytes (256 values) x bn rows in the 128-byte swizzle.
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
  CUtensorMap b;
  if (!weights_map(&b, p.kd, row_bytes(p.K), p.N, p.E, BN))
    return fail(CVMM_ERR_LAUNCH, "cvmm_mx_forward: tensor map");
  const auto kernel = p.y_words != p.N ? gemm_kernel<BN, S, NACC, true> : gemm_kernel<BN, S, NACC, false>;
  if (int rc = umma::set_smem(kernel, L::alloc)) return rc;
  const int n_n = (int)((p.N + BN - 1) / BN);
  const unsigned grid = (unsigned)std::min<int64_t>(max_tiles * n_n, umma::sm_count());
  launch(kernel, grid, kThreads, L::alloc, stream, p, b, n_n);
  return check_launch("cvmm_mx_forward: gemm");
}

// Columns of a tile: a stage takes 0.48, 0.50 and 0.67 us at 64, 128 and 256
// (32768 tokens 4096 -> 512: 877, 464 and 312 us), so wide tiles where they
// fill the SMs and narrow ones where those would leave SMs idle: 1 token 10.9,
// 11.3 and 13.2 us, 8 tokens 25.3, 19.0 and 13.5 us.
static int tile_columns(int64_t R, int64_t E, int64_t N, int64_t sms) {
  const int64_t used = std::min(E, R), m_tiles = std::max(R / kTile + used / 2, used);
  const auto cost = [&](int64_t bn, int64_t stage) { return (m_tiles * ((N + bn - 1) / bn) + sms - 1) / sms * stage; };
  const int64_t c64 = cost(64, 48), c128 = cost(128, 50), c256 = cost(256, 67);
  return c256 < c128 && c256 < c64 ? 256 : c128 < c64 ? 128 : 64;
}

// Workspace of one call, in order.
struct Sizes {
  size_t header, cursor, tiles, list, rank, xd, xs, y, total;
  int64_t cells, max_tiles;
};
static Sizes sizes(int64_t x_rows, int64_t R, int64_t E, int64_t K, int64_t N, bool weighted) {
  Sizes z;
  z.cells = (pieces(K) + 1) / 2 * 2;  // two a stage
  z.max_tiles = R / kTile + std::min(E, R);
  z.header = 256;
  z.cursor = align_up((size_t)E * 4, 256);
  z.tiles = align_up((size_t)z.max_tiles * sizeof(int4), 256);
  z.list = align_up((size_t)R * 4, 256);
  z.rank = R > kPlanAlone ? align_up((size_t)R * sizeof(int2), 256) : 0;
  z.xd = align_up((size_t)(x_rows * row_bytes(K)), 256);
  z.xs = align_up((size_t)(x_rows * z.cells * 4), 256);
  z.y = weighted ? align_up((size_t)(R * N) * 4, 256) : 0;
  z.total = z.header + z.cursor + z.tiles + z.list + z.rank + z.xd + z.xs + z.y + 256;
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

int cvmm_mx_launches(int64_t n_routes, int weighted) {
  return n_routes <= 0 ? 0 : 2 + (n_routes > cvmm::mx::kPlanAlone) + (weighted != 0);
}

int cvmm_mx_tile_columns(int64_t n_routes, int64_t n_experts, int64_t n_dim, int64_t sms) {
  if (n_routes < 1 || n_experts < 1 || n_dim < 1 || sms < 1) return 0;
  return cvmm::mx::tile_columns(n_routes, n_experts, n_dim, sms);
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
  p.x_vec = mx::vector_bytes(x, x_ld * (int64_t)dtype_size(x_dtype), 0);
  p.per_row = mx::Divisor(n_routes / x_rows);
  p.cells = z.cells;
  p.sel = sel; p.sel_dtype = sel_dtype; p.R = n_routes; p.E = (int)n_experts;
  p.header = reinterpret_cast<int*>(take(z.header));
  p.cursor = reinterpret_cast<int*>(take(z.cursor));
  p.tiles = reinterpret_cast<int4*>(take(z.tiles));
  p.list = reinterpret_cast<int32_t*>(take(z.list));
  p.rank = reinterpret_cast<int2*>(take(z.rank));
  p.xd = reinterpret_cast<uint8_t*>(take(z.xd));
  p.xs = reinterpret_cast<uint8_t*>(take(z.xs));
  p.y = w ? take(z.y) : out;
  p.y_words = w ? 2 * n_dim : n_dim;
  p.kd = keys_data; p.ks = keys_scale; p.K = k_dim; p.N = n_dim;
  p.out_dtype = out_dtype;
  p.y_vec = n_dim % 8 == 0 && al16(p.y);

  const int plan_blocks =
      n_routes <= mx::kPlanAlone ? 1 : (int)((n_routes + mx::kPlanChunk - 1) / mx::kPlanChunk);
  const int quant_blocks = grid_for(x_rows * z.cells * 4, mx::kPlanThreads);
  const size_t plan_smem = (size_t)(2 * n_experts + 1 + 34) * sizeof(int);
  if (plan_blocks > 1 && cudaMemsetAsync(p.header, 0, z.header + z.cursor, s) != cudaSuccess)
    return fail_cuda("cvmm_mx_forward: memset");
  const auto prepare = x_dtype == CVMM_F32 ? mx::prepare_kernel<F32>
                       : x_dtype == CVMM_BF16 ? mx::prepare_kernel<BF16> : mx::prepare_kernel<F16>;
  launch(prepare, plan_blocks + quant_blocks, mx::kPlanThreads, plan_smem, s, p, plan_blocks,
         mx::Divisor(z.cells * 4));
  if (plan_blocks > 1) launch(mx::fill_kernel, (unsigned)((n_routes + 255) / 256), 256, 0, s, p);
  if (int rc = check_launch("cvmm_mx_forward: prepare")) return rc;
  const int columns = mx::tile_columns(n_routes, n_experts, n_dim, umma::sm_count());
  const int rc = columns == 256   ? mx::launch_gemm<256, 4, 1>(p, z.max_tiles, s)
                 : columns == 128 ? mx::launch_gemm<128, 6, 2>(p, z.max_tiles, s)
                                  : mx::launch_gemm<64, 7, 2>(p, z.max_tiles, s);
  if (rc || !w) return rc;
  const int64_t T = n_routes / top_k;
  launch(mx::combine_kernel, (unsigned)((T * ((n_dim + 7) / 8) + 255) / 256), 256, 0, s,
         static_cast<const float*>(p.y), w, w_dtype, T, top_k,
         n_dim, out, out_dtype, n_dim % 8 == 0 && al16(out));
  return check_launch("cvmm_mx_forward: combine");
}

}  // extern "C"
