// Low-rank adapters of many requests beside a shared projection (k_lora_rows): out[r] = base[r] + scale B (A x[r]) with
// the adapter that row r names, A [rank][n] and B [d][rank] in fp32, bf16 or fp16. Products and sums are fp32.
//
// One launch: a cluster of CTAs per row, or per tile of up to 64 rows of one adapter. Each CTA takes a slice of n for
// A x, the cluster sums the slices' partial vectors through distributed shared memory in CTA order (no atomics: the same
// bits on every call), and each CTA then takes a slice of d for B. The rank-long vectors between the two products never
// leave the SMs.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRank = 256;
constexpr int kCtas = 8;  // of a tile's cluster
constexpr int kRowCtas = 4;  // an SM's CTAs of the row kernel
constexpr int kMaxColumns = 0x7fffffff - 65536;  // slices and steps are numbered past the last one

struct LoraArgs {
  float *out;
  const float *base, *x;
  long long ldo, ldb, ldx;
  const int *index;
  const LoraAdapter *adapters;
  int count, max_rank, n, d, rows;
  int from, to;  // the tile kernel's part of n
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// Eight neighbouring weights from a 16-byte aligned address.
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename H2>
__device__ __forceinline__ void halves(const void *p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    H2 h;
    *reinterpret_cast<unsigned *>(&h) = w[i];
    v[2 * i] = to_float(h.x), v[2 * i + 1] = to_float(h.y);
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) { halves<__nv_bfloat162>(p, v); }
__device__ __forceinline__ void load8(const __half *p, float (&v)[8]) { halves<__half2>(p, v); }

__host__ __device__ __forceinline__ bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The weights of a unit: 16 bytes, or 8.
__device__ __forceinline__ void load_unit(const float *p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4 *>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
__device__ __forceinline__ void load_unit(const __nv_bfloat16 *p, float (&v)[8]) { load8(p, v); }
__device__ __forceinline__ void load_unit(const __half *p, float (&v)[8]) { load8(p, v); }
template <typename W>
__device__ __forceinline__ void load_unit(const W *p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2 *>(p);
  const W *w = reinterpret_cast<const W *>(&a);
#pragma unroll
  for (int i = 0; i < 4; i++)
    v[i] = to_float(w[i]);
}

// out = base + B h for the outputs [d0, d1) of a row, rows of B in units of E weights: P lanes take a row together, so
// that a warp's reads are whole lines, and keep their part of h in registers. After P steps every lane has one of 32
// outputs; K such groups are under way at once.
template <typename W, int E, int P, int K = 1>
__device__ __forceinline__ void expand_rows(const W *B, const float *h, int rank, int d0, int d1, const float *base,
                                            float *out) {
  constexpr int G = 32 / P;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, p = lane % P, g = lane / P, units = rank / E;
  float hv[E];
#pragma unroll
  for (int e = 0; e < E; e++)
    hv[e] = p < units ? h[p * E + e] : 0.0f;
  for (int i0 = d0 + 32 * K * warp; i0 < d1; i0 += 32 * K * kWarps) {
    const int own = i0 + p * G + g;
    float before[K], mine[K];
#pragma unroll
    for (int k = 0; k < K; k++)
      before[k] = base && own + 32 * k < d1 ? base[own + 32 * k] : 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
      mine[k] = 0.0f;
#pragma unroll 8
      for (int step = 0; step < P; step++) {
        const int i = i0 + 32 * k + step * G + g;
        float s = 0.0f;
        if (i < d1 && p < units) {
          const W *row = B + (size_t)i * rank;
          float wv[E];
          load_unit(row + p * E, wv);
#pragma unroll
          for (int e = 0; e < E; e++)
            s = fmaf(wv[e], hv[e], s);
          if constexpr (P == 32)
            for (int u = p + 32; u < units; u += 32) {
              load_unit(row + u * E, wv);
#pragma unroll
              for (int e = 0; e < E; e++)
                s = fmaf(wv[e], h[u * E + e], s);
            }
        }
#pragma unroll
        for (int o = P / 2; o; o >>= 1)
          s += __shfl_xor_sync(0xffffffffu, s, o);
        mine[k] = p == step ? s : mine[k];
      }
    }
#pragma unroll
    for (int k = 0; k < K; k++)
      if (own + 32 * k < d1)
        out[own + 32 * k] = before[k] + mine[k];
  }
}

// A cluster of C CTAs per row. 33 rows of rank 32 fp32, 4096 to 14336: 10.4 us, 7.5 TB/s of adapters from L2, which
// bounds it; 64 rows of rank 16 bf16, 4096 to 4096: 6.9 us, the chain index, adapter, A, cluster, B in one wave.
template <typename W, int C>
__global__ void __launch_bounds__(kThreads, 4) lora_row_kernel(const LoraArgs a, int) {
  __shared__ float part[kMaxRank], h[kMaxRank];
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int ctas = C;
  const int rank = cluster.block_rank(), row = blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int id = a.index[row];
  LoraAdapter w = {nullptr, nullptr, 0, 0.0f};
  bool bad = id < -1 || id >= a.count;
  if (!bad && id >= 0) {
    w = a.adapters[id];
    bad = w.rank < 0 || w.rank > a.max_rank || (w.rank > 0 && (!w.a || !w.b));
  }
  if (bad) {
    w.rank = 0;
    if (rank == 0 && threadIdx.x == 0)
      kc_raise(KC_ERR_BAD_ARGS);
  }
  // A x over this CTA's slice of n, a warp per row of A.
  const W *A = static_cast<const W *>(w.a), *B = static_cast<const W *>(w.b);
  const float *x = a.x + (long long)row * a.ldx;
  const int n_slice = ((a.n + ctas - 1) / ctas + 7) & ~7;
  const int n0 = min(rank * n_slice, a.n), n1 = min(n0 + n_slice, a.n);
  const bool wide = aligned16(A) && aligned16(x) && a.n % 8 == 0;
  constexpr int R = sizeof(W) == 4 ? 2 : 4;  // rows of A at once: their reads are under way together
  for (int k0 = warp; k0 < w.rank; k0 += R * kWarps) {
    float s[R];
    const W *ak[R];
#pragma unroll
    for (int r = 0; r < R; r++)
      s[r] = 0.0f, ak[r] = A + (size_t)min(k0 + r * kWarps, w.rank - 1) * a.n;
    if (wide) {
      for (int i = n0 + 8 * lane; i < n1; i += 256) {
        float xv[8], wv[R][8];
        load8(x + i, xv);
#pragma unroll
        for (int r = 0; r < R; r++)
          if (k0 + r * kWarps < w.rank)
            load8(ak[r] + i, wv[r]);
#pragma unroll
        for (int r = 0; r < R; r++)
          if (k0 + r * kWarps < w.rank)
#pragma unroll
            for (int j = 0; j < 8; j++)
              s[r] = fmaf(wv[r][j], xv[j], s[r]);
      }
    } else {
#pragma unroll 2
      for (int i = n0 + lane; i < n1; i += 32) {
        const float xi = x[i];
#pragma unroll
        for (int r = 0; r < R; r++)
          s[r] = fmaf(to_float(ak[r][i]), xi, s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
      for (int o = 16; o; o >>= 1)
        s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
      if (lane == 0 && k0 + r * kWarps < w.rank)
        part[k0 + r * kWarps] = s[r];
    }
  }
  cluster.sync();
  for (int k = threadIdx.x; k < w.rank; k += kThreads) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < ctas; c++)
      s += *cluster.map_shared_rank(&part[k], c);
    h[k] = s * w.scale;
  }
  cluster.sync();  // the slices are read: a CTA may leave, and h is whole
  const int d_slice = (a.d + ctas - 1) / ctas;
  const int d0 = min(rank * d_slice, a.d), d1 = min(d0 + d_slice, a.d);
  const float *base = a.base ? a.base + (long long)row * a.ldb : nullptr;
  float *out = a.out + (long long)row * a.ldo;
  constexpr int E = 16 / sizeof(W);
  if (w.rank && aligned16(B) && w.rank % E == 0) {
    const int units = w.rank / E;
    const bool many = d1 - d0 >= 4 * kThreads;
    if (units <= 1 && many)
      expand_rows<W, E, 1, 4>(B, h, w.rank, d0, d1, base, out);
    else if (units <= 1)
      expand_rows<W, E, 1>(B, h, w.rank, d0, d1, base, out);
    else if (units <= 2 && many)
      expand_rows<W, E, 2, 2>(B, h, w.rank, d0, d1, base, out);
    else if (units <= 2)
      expand_rows<W, E, 2>(B, h, w.rank, d0, d1, base, out);
    else if (units <= 4)
      expand_rows<W, E, 4>(B, h, w.rank, d0, d1, base, out);
    else if (units <= 8)
      expand_rows<W, E, 8>(B, h, w.rank, d0, d1, base, out);
    else if (units <= 16)
      expand_rows<W, E, 16>(B, h, w.rank, d0, d1, base, out);
    else
      expand_rows<W, E, 32>(B, h, w.rank, d0, d1, base, out);
    return;
  }
  if (sizeof(W) == 2 && w.rank == 4 && ((uintptr_t)B & 7) == 0) {
    expand_rows<W, 4, 1, 4>(B, h, w.rank, d0, d1, base, out);
    return;
  }
  constexpr int K = 4;  // outputs under way
  for (int i0 = d0 + threadIdx.x; i0 < d1; i0 += K * kThreads) {
    float s[K], before[K];
#pragma unroll
    for (int j = 0; j < K; j++) {
      s[j] = 0.0f;
      before[j] = base && i0 + j * kThreads < d1 ? base[i0 + j * kThreads] : 0.0f;
    }
#pragma unroll 4
    for (int k = 0; k < w.rank; k++)
#pragma unroll
      for (int j = 0; j < K; j++)
        s[j] = fmaf(to_float(B[(size_t)min(i0 + j * kThreads, d1 - 1) * w.rank + k]), h[k], s[j]);
#pragma unroll
    for (int j = 0; j < K; j++)
      if (i0 + j * kThreads < d1)
        out[i0 + j * kThreads] = before[j] + s[j];
  }
}

// ---- tiles of rows ------------------------------------------------------------------------------------------------

// Many rows: tiles of up to 64 rows of one adapter, wherever they lie in the batch, so that a tile reads its adapter
// once. Every CTA finds its tile in the index array by itself (a histogram of the adapters, then the tile's rows in
// order): no sorting launch and no workspace. Rows without an adapter form tiles too, which copy their base.
//
// Both products run on tcgen05 with the weights as the M operand, as they lie in memory for bf16, and the tile's vectors
// as the N operand: D = A x' is [ranks][rows], then D = B h' [128 outputs][rows], whose lanes are neighbouring outputs
// of one row for the epilogue's reads and writes. fp32 values are three bf16 parts (24 bits: x = x0 + x1 + x2 with no
// scaling), fp16 weights two, fp32 weights three; a product is the sum of the parts' products up to 2^-24 of it
// (x_i w_j with i + j <= 2). The tensor cores' sums truncate, always towards zero: in the first product, whose sums are
// long, the small parts' sums have an accumulator of their own, so that a large one is cut once for sixteen elements
// only, and the large ones are three in turn, 48 cuts each at most (n = 10624: the result 1.2e-6 off with one, 0.4e-6
// with three). Beyond kMaxSum elements another launch adds the product over the next ones.
constexpr int kTileRows = 64;
constexpr int kTileRank = 128;       // ranks the tile kernel takes
constexpr int kMaxBins = 2048;       // adapters + 1 of the histogram
constexpr int kMaxTileRows = 16384;  // rows of a launch: every CTA reads their indices
constexpr int kStep = 64;            // elements of n a step: one 128-byte row of bf16
constexpr uint32_t kTmemCols = 256;  // four accumulators of 64 rows
constexpr int kTmemSmall = 192;      // the fourth takes the small parts of the first product
constexpr int kMaxSum = 16384;       // elements of n that a launch sums in the three others

// Parts of a weight.
template <typename W>
constexpr int kParts = std::is_same_v<W, __nv_bfloat16> ? 1 : sizeof(W) == 2 ? 2 : 3;

__host__ __device__ constexpr int rank_rows(int max_rank) { return max_rank <= 64 ? 64 : 128; }
__host__ __device__ constexpr int h_stride(int max_rank) { return rank_rows(max_rank) + 4; }

// Shared memory: `work` holds two stages of the first product (weights, then vectors), then the partial vectors, then a
// weight tile of the second product and a tile of outputs; behind it the operand of the vectors h and this CTA's own
// rows of h.
constexpr int kOutBytes = kTileRows * 128 * 4;
template <typename W>
struct TileSmem {
  int stage, tile, work, operand, total;
  __host__ __device__ explicit TileSmem(int max_rank) {
    const int r = rank_rows(max_rank);
    stage = kParts<W> * r * 128 + 3 * kTileRows * 128;
    tile = kParts<W> * 128 * r * 2;
    work = 2 * stage > tile + kOutBytes ? 2 * stage : tile + kOutBytes;
    operand = 3 * kTileRows * r * 2;
    total = work + operand + kTileRows / 8 * h_stride(max_rank) * 4 + 1024;
  }
};

struct LoraTile {
  uint64_t bar[2];
  uint32_t tmem;
  int abort_flag;
  int rows[kTileRows];
  int warp_sums[kWarps];
  int adapter, part, n;  // the cluster's tile: its adapter (`count`: rows without one) and its rows in order
  bool direct[kTileRows], any_direct;  // rows whose vector is not finite
};

// False: no such tile. bins: kMaxBins words. A thread takes a run of neighbouring rows, whose adapters it keeps as long
// as there are no more than kKept.
__device__ bool find_tile(const LoraArgs &a, LoraTile *t, int *bins, int tile) {
  constexpr int kKept = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = a.count + 1;
  const int per = (a.rows + kThreads - 1) / kThreads, r0 = min((int)threadIdx.x * per, a.rows), r1 = min(r0 + per, a.rows);
  int kept[kKept];
  auto read = [&](int r) {
    const int id = a.index[r];
    return id >= 0 && id < a.count ? id : a.count;
  };
#pragma unroll
  for (int i = 0; i < kKept; i++)
    kept[i] = r0 + i < r1 ? read(r0 + i) : -1;
  for (int i = threadIdx.x; i < count; i += kThreads)
    bins[i] = 0;
  if (threadIdx.x == 0)
    t->adapter = -1;
  __syncthreads();
  int last = -1, run = 0;  // neighbours of one adapter are added at once
  auto add = [&](int bin) {
    if (bin != last && run)
      atomicAdd(&bins[last], run);
    run = bin == last ? run + 1 : 1;
    last = bin;
  };
#pragma unroll
  for (int i = 0; i < kKept; i++)
    if (kept[i] >= 0)
      add(kept[i]);
  for (int r = r0 + kKept; r < r1; r++)
    add(read(r));
  if (run)
    atomicAdd(&bins[last], run);
  __syncthreads();
  // The adapter whose tiles hold number `tile`: a running sum over the adapters' tiles.
  int before = 0;
  for (int i0 = 0; i0 < count; i0 += kThreads) {
    const int i = i0 + threadIdx.x, tiles = i < count ? (bins[i] + kTileRows - 1) / kTileRows : 0;
    int upto = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o)
        upto += other;
    }
    if (lane == 31)
      t->warp_sums[warp] = upto;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kWarps; w++) {
      if (w < warp)
        upto += t->warp_sums[w];
      all += t->warp_sums[w];
    }
    if (tile >= before + upto - tiles && tile < before + upto) {
      t->adapter = i;
      t->part = tile - (before + upto - tiles);
      t->n = min(kTileRows, bins[i] - t->part * kTileRows);
    }
    before += all;
    __syncthreads();
  }
  if (t->adapter < 0)
    return false;
  // Its rows, ranked by the matches before them.
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kKept; i++)
    mine += kept[i] == t->adapter;
  for (int r = r0 + kKept; r < r1; r++)
    mine += read(r) == t->adapter;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o)
      upto += other;
  }
  if (lane == 31)
    t->warp_sums[warp] = upto;
  __syncthreads();
  int rank = upto - mine - t->part * kTileRows;
  for (int w = 0; w < warp; w++)
    rank += t->warp_sums[w];
  if (mine && rank < kTileRows && rank + mine > 0) {
    auto take = [&](int r) {
      if (rank >= 0 && rank < kTileRows)
        t->rows[rank] = r;
      rank++;
    };
#pragma unroll
    for (int i = 0; i < kKept; i++)
      if (kept[i] == t->adapter)
        take(r0 + i);
    for (int r = r0 + kKept; r < r1; r++)
      if (read(r) == t->adapter)
        take(r);
  }
  __syncthreads();
  return true;
}

// kind::f16 instruction descriptor: bf16 A and B, both K-major, fp32 accumulators, M x N.
__host__ __device__ constexpr uint32_t umma_idesc_bf16(int m, int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_bf16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// A CTA's wait for its MMAs, with one answer for a warp's lanes: false once any wait of the CTA has given up.
__device__ __forceinline__ bool tile_wait(uint64_t *bar, unsigned parity, volatile int *abort_flag) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    ok = *abort_flag == 0;
    if (ok && !mbar_wait_bounded(bar, parity)) {
      *abort_flag = 1;
      ok = false;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Two values as N packed bf16 parts. The first part of a finite value is finite (the largest ones would round up to an
// infinity); those of an infinity or NaN have a NaN among them where N is 3, so that none passes unseen.
template <int N>
__device__ __forceinline__ void parts2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (i == 0)
      asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(p[0]) : "f"(y), "f"(x));
    else
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p[i]) : "f"(y), "f"(x));
    if (i + 1 < N) {
      x -= __uint_as_float(p[i] << 16);
      y -= __uint_as_float(p[i] & 0xffff0000u);
    }
  }
}

// Byte offset of element (row, col) of a K-major operand of 128-byte rows in the 128-byte swizzle, `rows` rows to a
// block of 64 columns.
__device__ __forceinline__ uint32_t operand_at(int rows, int row, int col) {
  return (col >> 6) * rows * 128 + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}

// A thread's share of a weight operand: up to N runs of eight neighbouring elements in registers, read ahead of their
// use. The operand is the first `runs` runs, 1 << log a row at most, of columns from c0 on of `rows` rows of a row-major
// matrix (row stride ld); zeros from column `end` on.
template <typename W, int N>
struct WeightRuns {
  uint4 v[N][sizeof(W) / 2];

  __device__ __forceinline__ void load(int first, const W *w, size_t ld, int rows, int c0, int runs, int log, int end,
                                       bool wide) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int id = first + n * kThreads + threadIdx.x, row = id >> log, run = id & ((1 << log) - 1), c = c0 + run * 8;
      if (row >= rows || run >= runs)
        continue;
      const W *src = w + row * ld + c;
      if (wide && c < end) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(W) / 2); j++)
          v[n][j] = __ldg(reinterpret_cast<const uint4 *>(src) + j);
      } else {
        W *at = reinterpret_cast<W *>(v[n]);
#pragma unroll
        for (int j = 0; j < 8; j++)
          at[j] = c + j < end ? src[j] : W(0.0f);
      }
    }
  }
  // As operand parts of blocks of `high` rows, `bytes` apart.
  __device__ __forceinline__ void store(int first, uint8_t *at, int bytes, int high, int rows, int runs, int log) const {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int id = first + n * kThreads + threadIdx.x, row = id >> log, run = id & ((1 << log) - 1);
      if (row >= rows || run >= runs)
        continue;
      uint8_t *dst = at + operand_at(high, row, run * 8);
      if constexpr (kParts<W> == 1) {
        *reinterpret_cast<uint4 *>(dst) = v[n][0];
      } else {
        const unsigned *u = reinterpret_cast<const unsigned *>(v[n]);
        uint32_t p[4][kParts<W>];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float x, y;
          if constexpr (sizeof(W) == 4) {
            x = __uint_as_float(u[2 * j]), y = __uint_as_float(u[2 * j + 1]);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
            x = f.x, y = f.y;
          }
          parts2(x, y, p[j]);
        }
#pragma unroll
        for (int i = 0; i < kParts<W>; i++)
          *reinterpret_cast<uint4 *>(dst + i * bytes) = make_uint4(p[0][i], p[1][i], p[2][i], p[3][i]);
      }
    }
  }
};

// Four neighbouring floats of a row, `left` of them inside; 16-byte units where `wide`.
__device__ __forceinline__ float4 read4(const float *p, int left, bool wide) {
  if (wide && left >= 4)
    return *reinterpret_cast<const float4 *>(p);
  return make_float4(left > 0 ? p[0] : 0.0f, left > 1 ? p[1] : 0.0f, left > 2 ? p[2] : 0.0f, left > 3 ? p[3] : 0.0f);
}
__device__ __forceinline__ void write4(float *p, float4 v, int left, bool wide) {
  if (wide && left >= 4) {
    *reinterpret_cast<float4 *>(p) = v;
    return;
  }
  if (left > 0)
    p[0] = v.x;
  if (left > 1)
    p[1] = v.y;
  if (left > 2)
    p[2] = v.z;
  if (left > 3)
    p[3] = v.w;
}

// The whole CTA: a row's product over [n0, n1) of x by fp32 FMAs, added to its outputs [d0, d1). Where a row's vector is
// not finite its bf16 parts say nothing, and the formula decides which outputs are infinities, numbers or NaN. h: 128
// floats of shared memory.
template <typename W>
__device__ __forceinline__ void row_directly(const LoraArgs &a, const W *A, const W *B, int rank, float scale, int row, int n0,
                                             int n1, int d0, int d1, float *h) {
  const float *x = a.x + (long long)row * a.ldx;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  for (int k = warp; k < rank; k += kWarps) {
    float s = 0.0f;
    for (int i = n0 + lane; i < n1; i += 32)
      s = fmaf(to_float(A[(size_t)k * a.n + i]), x[i], s);
#pragma unroll
    for (int o = 16; o; o >>= 1)
      s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0)
      h[k] = s * scale;
  }
  __syncthreads();
  for (int i = d0 + threadIdx.x; i < d1; i += kThreads) {
    float s = 0.0f;
    for (int k = 0; k < rank; k++)
      s = fmaf(to_float(B[(size_t)i * rank + k]), h[k], s);
    a.out[(long long)row * a.ldo + i] += s;
  }
}

// 2048 rows of 4 adapters of rank 64 bf16, 4096 to 4096: 45 us, 2.4 TB/s of the rows' own bytes, the tensor pipe 8 % and
// the issue slots 24 % busy: the phases (rows, first product, the cluster's sum, second product) follow one another, two
// CTAs an SM.
// parts clusters share a tile: each computes its vectors and takes a part of d. kPart: of n, the launch takes a part.
template <typename W, bool kPart>
__global__ void __launch_bounds__(kThreads, 2) lora_tile_kernel(const LoraArgs a, int parts) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ LoraTile t;
  constexpr int P = kParts<W>;
  const TileSmem<W> L(a.max_rank);
  const int rank_high = rank_rows(a.max_rank), hs = h_stride(a.max_rank);
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int ctas = kCtas;
  const int rank = cluster.block_rank(), id = blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort_flag = &t.abort_flag;
  if (threadIdx.x == 0) {
    mbar_init(&t.bar[0], 1);
    mbar_init(&t.bar[1], 1);
    t.abort_flag = 0;
    t.any_direct = false;
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < kTileRows; i += kThreads)
    t.direct[i] = false;
  pdl_wait();
  pdl_launch_dependents();
  if (!find_tile(a, &t, reinterpret_cast<int *>(smem), id / parts))
    return;  // the whole cluster
  if (warp == 0)
    tmem_alloc(&t.tmem, kTmemCols);
  const int part = id % parts, rows = t.n, n16 = (rows + 15) / 16 * 16;
  LoraAdapter w = {nullptr, nullptr, 0, 0.0f};
  bool bad = false;
  if (t.adapter < a.count) {
    w = a.adapters[t.adapter];
    bad = w.rank < 0 || w.rank > a.max_rank || (w.rank > 0 && (!w.a || !w.b));
  } else if (part == 0 && rank == 0) {
    for (int i = threadIdx.x; i < rows; i += kThreads)
      bad |= a.index[t.rows[i]] != -1;
  }
  if (bad) {
    w.rank = 0;
    if (part == 0 && rank == 0)
      kc_raise(KC_ERR_BAD_ARGS);
  }
  const W *A = static_cast<const W *>(w.a), *B = static_cast<const W *>(w.b);
  const int rank16 = (w.rank + 15) / 16 * 16;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = t.tmem;
  uint8_t *operand = smem + L.work;
  float *partial = reinterpret_cast<float *>(smem), *own_h = reinterpret_cast<float *>(operand + L.operand);
  int phase[2] = {0, 0};  // of the two barriers, the same in all threads
  bool ok = true;

  // This CTA's slices of n and d. Its vectors' and its base's lines start on their way to L2 now.
  const int d_all = parts * ctas, d_slice = ((a.d + d_all - 1) / d_all + 31) / 32 * 32;
  const int d0 = min((part * ctas + rank) * d_slice, a.d), d1 = min(d0 + d_slice, a.d), tiles = (d1 - d0 + 127) / 128;
  const int from_n = kPart ? a.from : 0, to_n = kPart ? a.to : a.n;
  const int n_slice = ((to_n - from_n + ctas - 1) / ctas + kStep - 1) / kStep * kStep;
  const int n0 = min(from_n + rank * n_slice, to_n), n1 = min(n0 + n_slice, to_n);
  const int steps = w.rank ? (n1 - n0 + kStep - 1) / kStep : 0;
  auto prefetch = [&](const float *from, long long ld, int c0, int c1) {
    const int lines = (c1 - c0 + 31) / 32;
    for (int e = threadIdx.x; e < rows * lines; e += kThreads) {
      const int i = e / lines;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(from + t.rows[i] * ld + c0 + 32 * (e - i * lines)));
    }
  };
  if (w.rank)
    prefetch(a.x, a.ldx, n0, n1);
  if (a.base)
    prefetch(a.base, a.ldb, d0, d1);
  const bool x_wide = aligned16(a.x) && a.ldx % 4 == 0 && a.n % 4 == 0, a_wide = aligned16(A) && a.n % 8 == 0;
  const int a_bytes = rank_high * 128, x_bytes = kTileRows * 128;
  if (steps) {
    // This thread's share of a step's vectors: four neighbouring elements of rows r0, r0 + 16, ...
    const int r0 = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * 4;
    const float *src[4];
    float4 x[2][4];
#pragma unroll
    for (int p = 0; p < 4; p++)
      src[p] = a.x + (long long)t.rows[min(r0 + 16 * p, rows - 1)] * a.ldx + c0;
    auto load_x = [&](float4 (&v)[4], int j) {
      const int c = n0 + j * kStep;
#pragma unroll
      for (int p = 0; p < 4; p++) {
        v[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j >= steps || r0 + 16 * p >= rows)
          continue;
        if (x_wide) {
          if (c + c0 < n1)
            v[p] = __ldcg(reinterpret_cast<const float4 *>(src[p] + c));
        } else {
          v[p].x = c + c0 < n1 ? src[p][c] : 0.0f;
          v[p].y = c + c0 + 1 < n1 ? src[p][c + 1] : 0.0f;
          v[p].z = c + c0 + 2 < n1 ? src[p][c + 2] : 0.0f;
          v[p].w = c + c0 + 3 < n1 ? src[p][c + 3] : 0.0f;
        }
      }
    };
    // Its share of the weights: two runs a step up to 64 ranks, read two steps ahead; the others as they are needed.
    WeightRuns<W, 2> runs2[2];
    auto load_w = [&](WeightRuns<W, 2> &r, int first, int j) {
      r.load(first, A, (size_t)a.n, w.rank, n0 + j * kStep, kStep / 8, 3, n1, a_wide);
    };
    const uint32_t idesc = umma_idesc_bf16(128, n16);
    auto step = [&](auto odd, float4 (&v)[4], WeightRuns<W, 2> &runs, int j) {
      constexpr int s = odd;  // j & 1
      uint8_t *stage = smem + s * L.stage, *xs = stage + P * a_bytes;
      if (j > 1) {  // the stage is free once the MMAs of two steps ago are done
        ok &= tile_wait(&t.bar[s], phase[s] & 1, abort_flag);
        phase[s]++;
      }
#pragma unroll
      for (int p = 0; p < 4; p++)
        if (16 * p < n16) {
          uint32_t p0[3], p1[3];
          parts2(v[p].x, v[p].y, p0);
          parts2(v[p].z, v[p].w, p1);
          uint8_t *dst = xs + operand_at(kTileRows, r0 + 16 * p, c0);
#pragma unroll
          for (int i = 0; i < 3; i++)
            *reinterpret_cast<uint2 *>(dst + i * x_bytes) = make_uint2(p0[i], p1[i]);
        }
      runs.store(0, stage, a_bytes, rank_high, w.rank, kStep / 8, 3);
      if (w.rank > 64) {
        load_w(runs, 2 * kThreads, j);
        runs.store(2 * kThreads, stage, a_bytes, rank_high, w.rank, kStep / 8, 3);
      }
      fence_proxy_async_smem();
      __syncthreads();
      if (warp == 0 && ok) {
        if (elect_one()) {
          const uint64_t ad = umma_desc_sw128(stage), bd = umma_desc_sw128(xs);
#pragma unroll
          for (int s2 = 2; s2 >= 0; s2--)
#pragma unroll
            for (int i = 0; i < P; i++) {  // part i of the weights, s2 - i of the vectors
              if (i > s2)
                continue;
#pragma unroll
              for (int k = 0; k < kStep / 16; k++)
                umma_bf16(tmem + (s2 ? kTmemSmall : 64 * ((4 * s + k) % 3)), ad + (i * a_bytes + 32 * k) / 16,
                          bd + ((s2 - i) * x_bytes + 32 * k) / 16, idesc,
                          j > 0 || (s2 ? s2 < 2 || i > 0 || k > 0 : k > 2));
            }
          umma_commit(&t.bar[s]);
        }
        __syncwarp();
      }
      load_x(v, j + 2);
      if (j + 2 < steps)
        load_w(runs, 0, j + 2);
    };
    load_w(runs2[0], 0, 0);
    load_x(x[0], 0);
    if (steps > 1)
      load_w(runs2[1], 0, 1);
    load_x(x[1], 1);
    for (int j = 0; j < steps; j += 2) {
      step(std::integral_constant<int, 0>(), x[0], runs2[0], j);
      if (j + 1 < steps)
        step(std::integral_constant<int, 1>(), x[1], runs2[1], j + 1);
    }
    // The last two steps' MMAs.
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int uses = (steps + 1 - i) / 2;
      for (; phase[i] < uses; phase[i]++)
        ok &= tile_wait(&t.bar[i], phase[i] & 1, abort_flag);
    }
    __syncthreads();
    tc_fence_after();
    // Lanes are ranks, columns rows: into this CTA's partial vectors, 32 columns for each half of the warps.
    const int k = 32 * (warp & 3) + lane, column = 32 * (warp >> 2);
    if (32 * (warp & 3) < rank16 && column < n16) {
      const uint32_t from = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + column;
#pragma unroll
      for (int c = 0; c < 32; c += 16) {
        float sum[16];
#pragma unroll
        for (int l = 0; l < 4; l++) {
          uint32_t e[16];
          tmem_ld16(from + 64 * l + c, e);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++)
            sum[i] = l ? sum[i] + __uint_as_float(e[i]) : __uint_as_float(e[i]);
        }
        if (k < rank16)
#pragma unroll
          for (int i = 0; i < 16; i++)
            partial[(column + c + i) * hs + k] = k < w.rank ? sum[i] : 0.0f;
      }
    }
    tc_fence_before();
  } else {
    for (int e = threadIdx.x; e < rows * rank16; e += kThreads)
      partial[e / rank16 * hs + e % rank16] = 0.0f;
  }
  // The cluster's sums: CTA c adds up its share of the rows from all CTAs in their order, then everyone fetches them as
  // the second product's operand.
  cluster.sync();
  const int own = (rows - rank + ctas - 1) / ctas;  // rows rank, rank + ctas, ...: a warp each
  if (warp < own)
    for (int k = lane; k < rank16; k += 32) {
      float s = 0.0f;
#pragma unroll 8
      for (int c = 0; c < ctas; c++)
        s += *cluster.map_shared_rank(&partial[(rank + warp * ctas) * hs + k], c);
      own_h[warp * hs + k] = s * w.scale;
    }
  cluster.sync();
  const int h_bytes = kTileRows * rank_high * 2;
  unsigned direct = 0;  // a bit for each of this warp's rows that has a number which is not finite
  for (int k = 2 * lane; k < rank16; k += 64) {
#pragma unroll
    for (int n = 0; n < kTileRows / kWarps; n++) {
      const int i = warp + kWarps * n;
      if (i >= n16)
        break;
      float2 v = make_float2(0.0f, 0.0f);
      if (i < rows)
        v = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(&own_h[i / ctas * hs + k], i % ctas));
      if (!(fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY))
        direct |= 1u << n;
      uint32_t p[3];
      parts2(v.x, v.y, p);
      uint8_t *dst = operand + operand_at(kTileRows, i, k);
#pragma unroll
      for (int j = 0; j < 3; j++)
        *reinterpret_cast<uint32_t *>(dst + j * h_bytes) = p[j];
    }
  }
  auto fetched = cluster.barrier_arrive();  // a CTA may leave once everybody has fetched everything
  if (__any_sync(0xffffffffu, direct != 0)) {  // those rows get their base for now
    direct = __reduce_or_sync(0xffffffffu, direct);
    for (int n = 0; n < kTileRows / kWarps; n++) {
      if (lane == 0)
        t.direct[warp + kWarps * n] = direct >> n & 1;
      if (direct >> n & 1)
        for (int k = 2 * lane; k < rank16; k += 64)
          for (int j = 0; j < 3; j++)
            *reinterpret_cast<uint32_t *>(operand + j * h_bytes + operand_at(kTileRows, warp + kWarps * n, k)) = 0;
    }
    t.any_direct = true;
  }

  // B h over this CTA's slice of d, 128 outputs at a time.
  const bool b_wide = aligned16(B) && w.rank % 8 == 0;
  const int b_bytes = 128 * rank_high * 2, per = rank16 / 8, log = rank_high == 64 ? 3 : 4;
  const uint32_t idesc = umma_idesc_bf16(128, n16);
  const int column = 32 * (warp >> 2), lane_d = 32 * (warp & 3) + lane;
  const bool base_wide = aligned16(a.base) && a.ldb % 4 == 0, out_wide = aligned16(a.out) && a.ldo % 4 == 0;
  float *tile_out = reinterpret_cast<float *>(smem + L.tile);  // [64][128]
  // This thread's share of a weight tile: four runs up to 64 ranks, read a tile ahead.
  WeightRuns<W, 4> runs;
  auto load_w = [&](int first, int j) {
    const int d = d0 + 128 * j;
    if (per && d < d1)
      runs.load(first, B + (size_t)d * w.rank, (size_t)w.rank, min(128, d1 - d), 0, per, log, w.rank, b_wide);
  };
  // A warp per row, four outputs a lane: this lane's base, read a tile ahead.
  int r[kTileRows / kWarps];
  float4 y[kTileRows / kWarps];
#pragma unroll
  for (int n = 0; n < kTileRows / kWarps; n++)
    r[n] = t.rows[min(warp + kWarps * n, rows - 1)];
  auto load_base = [&](int j) {
    const int at = d0 + 128 * j + 4 * lane, left = d1 - at;
#pragma unroll
    for (int n = 0; n < kTileRows / kWarps; n++) {
      y[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (a.base && warp + kWarps * n < rows)
        y[n] = read4(a.base + r[n] * a.ldb + at, left, base_wide);
    }
  };
  load_w(0, 0);
  load_base(0);
  for (int j = 0; j < tiles; j++) {
    const int d = d0 + 128 * j;
    if (per) {
      runs.store(0, smem, b_bytes, 128, min(128, d1 - d), per, log);
      if (rank_high > 64) {
        load_w(4 * kThreads, j);
        runs.store(4 * kThreads, smem, b_bytes, 128, min(128, d1 - d), per, log);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncthreads();
      if (warp == 0 && ok) {
        if (elect_one()) {
          tc_fence_after();
          const uint64_t ad = umma_desc_sw128(smem), bd = umma_desc_sw128(operand);
          const int ks = rank16 / 16;
#pragma unroll
          for (int s = 2; s >= 0; s--)
#pragma unroll
            for (int i = 0; i < P; i++) {
              if (i > s)
                continue;
              const uint64_t ai = ad + i * b_bytes / 16, bi = bd + (s - i) * h_bytes / 16;
#pragma unroll
              for (int k = 0; k < kTileRank / 16; k++)
                if (k < ks)
                  umma_bf16(tmem, ai + ((k >> 2) * 128 * 128 + 32 * (k & 3)) / 16,
                            bi + ((k >> 2) * kTileRows * 128 + 32 * (k & 3)) / 16, idesc, s < 2 || i > 0 || k > 0);
            }
          umma_commit(&t.bar[0]);
        }
        __syncwarp();
      }
      load_w(0, j + 1);
    }
    if (per) {
      ok &= tile_wait(&t.bar[0], phase[0] & 1, abort_flag);
      phase[0]++;
      tc_fence_after();
      if (column < n16) {  // lanes are outputs, columns rows: by way of shared memory
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
          uint32_t v[16];
          tmem_ld16(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + column + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++)
            tile_out[(column + c + i) * 128 + lane_d] = __uint_as_float(v[i]);
        }
      }
      __syncthreads();
    }
    const int at = d + 4 * lane;
#pragma unroll
    for (int n = 0; n < kTileRows / kWarps; n++) {
      const int i = warp + kWarps * n;
      if (i >= rows)
        break;
      if (per) {
        const float4 v = *reinterpret_cast<const float4 *>(tile_out + i * 128 + 4 * lane);
        y[n].x += v.x, y[n].y += v.y, y[n].z += v.z, y[n].w += v.w;
      }
      write4(a.out + r[n] * a.ldo + at, y[n], d1 - at, out_wide);
    }
    if (j + 1 < tiles)
      load_base(j + 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (t.any_direct)
    for (int i = 0; i < rows; i++)
      if (t.direct[i])
        row_directly(a, A, B, w.rank, w.scale, t.rows[i], from_n, to_n, d0, d1, reinterpret_cast<float *>(smem));
  cluster.barrier_wait(std::move(fetched));
}

template <typename W>
cudaError_t launch(void (*kernel)(LoraArgs, int), const LoraArgs &a, unsigned clusters, int parts, size_t smem,
                   int ctas = kCtas) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = kc_stream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = kc_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, a, parts);
}

// At most this many tiles: the full ones, and one more for each adapter and the rows without one.
int most_tiles(const LoraArgs &a) {
  const int some = a.count + 1 < a.rows ? a.count + 1 : a.rows;
  return (a.rows - some) / kTileRows + some;
}
int parts_for(int tiles) {
  const int few = kc_device_sms() / (kCtas * tiles);
  return few < 1 ? 1 : few > 4 ? 4 : few;
}

// The two kernels' times in microseconds, fitted to 70 shapes (1 to 2048 rows, 1 to 64 adapters of rank 4 to 64, 256 to
// 14336 columns, the three types) to 17 % on average; where the estimates choose wrongly the two are close (1 % lost on
// average over the same shapes, 27 % at most). Ranks 65 to 128 lie outside the fit: right for 8 rows and from 256 on, but
// of 33 to 128 rows of 4 to 8 adapters many go to the row kernel where tiles take half the time (128 rows of 8 adapters of
// rank 128 bf16, 4096 to 4096: 48 us, 29 as tiles; fp32, 2048 to 8192: 127 us, 57 as tiles). A row's adapter comes from
// L2 for every row. 33 rows, rank 32 fp32, 4096 to 14336: 11 us here, 38 as tiles.
template <typename W>
double row_us(const LoraArgs &a) {
  const double mb = 1e-6 * a.rows;
  return 5.7 + mb * (0.79 * 4 * a.n + 0.27 * 8 * a.d + sizeof(W) * (double)a.max_rank * (0.058 * a.n + 0.108 * a.d));
}
// A tile reads its adapter once, in steps over the n and d columns; a wave of clusters after another. 2048 rows of rank
// 64 bf16, 4096 to 4096: 45 us here, 319 as rows.
template <typename W>
double tile_us(const LoraArgs &a) {
  const int tiles = most_tiles(a), parts = parts_for(tiles);
  const double ctas = (double)kCtas * tiles * parts / kc_device_sms();
  const bool wide = aligned16(a.out) && a.ldo % 4 == 0 && aligned16(a.base) && a.ldb % 4 == 0;  // else one value at a time
  return 9.5 + (ctas > 1.0 ? ctas : 1.0) * (2.1 + 1.1e-3 * kParts<W> * a.n +
                                            ((wide ? 2.0e-3 : 4.6e-3) + 1.44e-5 * kParts<W> * a.max_rank) * a.d / parts);
}

// The largest cluster, 16 CTAs to one, with which all rows are resident at once, at kRowCtas CTAs an SM (291 rows of
// rank 4: 7 us with two CTAs a row, 11 with four); with two waves where a row's adapter is large (236 rows of rank 64
// fp16, 22 thousand columns: 76 us with four, 113 with two).
template <typename W, int C = 16>
cudaError_t launch_rows(const LoraArgs &a) {
  if constexpr (C > 1) {
    const bool large = C < 16 && sizeof(W) * (double)a.max_rank * ((double)a.n + a.d) > 1e6;
    if ((long long)a.rows * C > (large ? 2 : 1) * kRowCtas * kc_device_sms())
      return launch_rows<W, C / 2>(a);
  }
  if (C > 8) {
    const cudaError_t e = kc_allow_clusters(reinterpret_cast<const void *>(lora_row_kernel<W, C>));
    if (e != cudaSuccess)
      return e;
  }
  return launch<W>(lora_row_kernel<W, C>, a, (unsigned)a.rows, 1, 0, C);
}

// Ranks above kTileRank and kMaxBins adapters or more go to the row kernel whatever the rows (2048 rows of rank 256 bf16,
// 4096 to 4096: 1340 us, of rank 128 as tiles 130).
template <typename W>
cudaError_t run(const LoraArgs &a) {
  if (a.count >= kMaxBins || a.max_rank > kTileRank || row_us<W>(a) <= tile_us<W>(a))
    return launch_rows<W>(a);
  const size_t smem = TileSmem<W>(a.max_rank).total;
  void (*const kernel)(LoraArgs, int) = a.n > kMaxSum ? lora_tile_kernel<W, true> : lora_tile_kernel<W, false>;
  cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(kernel), TileSmem<W>(kTileRank).total);
  for (int r = 0; r < a.rows && e == cudaSuccess; r += kMaxTileRows) {
    LoraArgs b = a;
    b.rows = a.rows - r < kMaxTileRows ? a.rows - r : kMaxTileRows;
    b.x += (long long)r * a.ldx, b.out += (long long)r * a.ldo, b.index += r;
    if (b.base)
      b.base += (long long)r * a.ldb;
    const int tiles = most_tiles(b), parts = parts_for(tiles);
    for (int from = 0; from < a.n && e == cudaSuccess; from += kMaxSum) {
      b.from = from, b.to = a.n - from < kMaxSum ? a.n : from + kMaxSum;
      e = launch<W>(kernel, b, (unsigned)(tiles * parts), parts, smem);
      if (e == cudaSuccess && (r + kMaxTileRows < a.rows || from + kMaxSum < a.n))
        kc_count_launch();
      b.base = b.out, b.ldb = b.ldo;
    }
  }
  return e;
}

}  // namespace

extern "C" {

void k_lora_rows(float *out, size_t ldo, const float *base, size_t ldb, const float *x, size_t ldx, const int *index,
                 const LoraAdapter *adapters, int count, int type, int max_rank, int n, int d, int rows) {
  const char *name = "k_lora_rows";
  if (type != K_F32 && type != K_BF16 && type != K_F16) {
    kc_fail("%s: invalid weight type %d", name, type);
    return;
  }
  if (rows < 0 || rows > (1 << 24) || n <= 0 || n > kMaxColumns || d <= 0 || d > kMaxColumns || count < 0 ||
      max_rank <= 0 || max_rank > kMaxRank || ldx < (size_t)n || ldo < (size_t)d || (base && ldb < (size_t)d)) {
    kc_fail("%s: invalid shape rows=%d n=%d d=%d count=%d max_rank=%d (at most %d)", name, rows, n, d, count, max_rank,
            kMaxRank);
    return;
  }
  if (!rows)
    return;
  if (!out || !x || !index || (count && !adapters)) {
    kc_fail("%s: missing output, activations, row indices or adapters", name);
    return;
  }
  const LoraArgs a = {out, base, x, (long long)ldo, (long long)ldb, (long long)ldx, index, adapters, count, max_rank,
                      n, d, rows, 0, n};
  const cudaError_t e = type == K_F32 ? run<float>(a) : type == K_BF16 ? run<__nv_bfloat16>(a) : run<__half>(a);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
