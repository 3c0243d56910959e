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

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRank = 256;

struct LoraArgs {
  float *out;
  const float *base, *x;
  long long ldo, ldb, ldx;
  const int *index;
  const LoraAdapter *adapters;
  int count, max_rank, n, d, rows;
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

__device__ __forceinline__ bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename W>
__global__ void __launch_bounds__(kThreads) lora_row_kernel(const LoraArgs a, int) {
  __shared__ float part[kMaxRank], h[kMaxRank];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ctas;
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
  for (int k = warp; k < w.rank; k += kWarps) {
    const W *ak = A + (long long)k * a.n;
    float s = 0.0f;
    if (wide) {
      for (int i = n0 + 8 * lane; i < n1; i += 256) {
        float wv[8], xv[8];
        load8(ak + i, wv);
        load8(x + i, xv);
#pragma unroll
        for (int j = 0; j < 8; j++)
          s = fmaf(wv[j], xv[j], s);
      }
    } else {
      for (int i = n0 + lane; i < n1; i += 32)
        s = fmaf(to_float(ak[i]), x[i], s);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
      s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0)
      part[k] = s;
  }
  cluster.sync();
  for (int k = threadIdx.x; k < w.rank; k += kThreads) {
    float s = 0.0f;
    for (int c = 0; c < ctas; c++)
      s += *cluster.map_shared_rank(&part[k], c);
    h[k] = s * w.scale;
  }
  cluster.sync();  // the slices are read: a CTA may leave, and h is whole
  const int d_slice = (a.d + ctas - 1) / ctas;
  const int d0 = min(rank * d_slice, a.d), d1 = min(d0 + d_slice, a.d);
  const bool wide_b = aligned16(B) && w.rank % 8 == 0;
  for (int i = d0 + threadIdx.x; i < d1; i += kThreads) {
    const W *bi = B + (long long)i * w.rank;
    float s = 0.0f;
    if (wide_b) {
      for (int k = 0; k < w.rank; k += 8) {
        float wv[8];
        load8(bi + k, wv);
#pragma unroll
        for (int j = 0; j < 8; j++)
          s = fmaf(wv[j], h[k + j], s);
      }
    } else {
      for (int k = 0; k < w.rank; k++)
        s = fmaf(to_float(bi[k]), h[k], s);
    }
    const float before = a.base ? a.base[(long long)row * a.ldb + i] : 0.0f;
    a.out[(long long)row * a.ldo + i] = before + s;
  }
}

// ---- tiles of rows ------------------------------------------------------------------------------------------------

// Many rows: tiles of up to 64 rows of one adapter, wherever they lie in the batch, so that a tile reads its adapter
// once. Every CTA finds its tile in the index array by itself (a histogram of the adapters, then the tile's rows in
// order): no sorting launch and no workspace. Rows without an adapter form tiles too, which copy their base.
//
// Products on mma.sync m16n8k8 tf32 with both operands' 24 bits kept: x = hi + lo with hi its upper 11 bits, bf16 and
// fp16 weights are exact in tf32, fp32 ones split like x: hi w + lo w (+ hi w_lo), off by 2^-22 of a product. The tensor
// core's sums truncate, so they run over 32 elements only and are added up in fp32 registers. The k index of a
// fragment is free as long as both operands agree: a lane's two fragment columns of four steps are eight neighbouring
// elements, one 16- or 32-byte read, without a pass through shared memory.
constexpr int kTileRows = 64;
constexpr int kMaxBins = 2048;       // adapters + 1 of the histogram
constexpr int kMaxTileRows = 16384;  // rows of a launch: every CTA reads their indices

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t tf32_hi(float x) { return __float_as_uint(x) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_lo(float x) { return __float_as_uint(x - __uint_as_float(tf32_hi(x))); }

// This lane's eight elements of rows g and g + 8, split.
struct Split16 {
  uint32_t hi[2][8], lo[2][8];
  __device__ __forceinline__ void set(int r, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++)
      hi[r][j] = tf32_hi(v[j]), lo[r][j] = tf32_lo(v[j]);
  }
};

// Values 2 j and 2 j + 1 of words u.
template <typename W>
__device__ __forceinline__ void two(const unsigned *u, int j, float &x, float &y) {
  if constexpr (sizeof(W) == 4) {
    x = __uint_as_float(u[2 * j]), y = __uint_as_float(u[2 * j + 1]);
  } else if constexpr (std::is_same_v<W, __nv_bfloat16>) {
    x = __uint_as_float(u[j] << 16), y = __uint_as_float(u[j] & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
    x = f.x, y = f.y;
  }
}

// Eight elements of a row as they lie in memory, so that many can be under way.
template <typename W>
struct Raw8 {
  uint4 v[sizeof(W) / 2];

  // Whole groups of eight at 16-byte addresses.
  __device__ __forceinline__ void load(const W *at) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(W) / 2); j++)
      v[j] = __ldg(reinterpret_cast<const uint4 *>(at) + j);
  }
  // From element i on, zeros from `end` on. `wide`: as above.
  __device__ __forceinline__ void load(const W *row, int i, int end, bool wide) {
    if (wide && i + 8 <= end) {
#pragma unroll
      for (int j = 0; j < (int)(sizeof(W) / 2); j++)
        v[j] = __ldg(reinterpret_cast<const uint4 *>(row + i) + j);
    } else {
      W *at = reinterpret_cast<W *>(v);
#pragma unroll
      for (int j = 0; j < 8; j++)
        at[j] = i + j < end ? row[i + j] : W(0.0f);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const unsigned *u = reinterpret_cast<const unsigned *>(v);
#pragma unroll
    for (int j = 0; j < 4; j++)
      two<W>(u, j, f[2 * j], f[2 * j + 1]);
  }
};

// 16 rows x 8 columns += 32 elements of the 16 rows times those of the 8 columns (this lane's eight of column g).
// SPLIT: the weights have more bits than tf32.
template <bool SPLIT>
__device__ __forceinline__ void product32(float (&sum)[4], const Split16 &x, const float (&w)[8]) {
  float d[4], small[4];  // two chains of MMAs
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const int e = 2 * s;
    const uint32_t lo[4] = {x.lo[0][e], x.lo[1][e], x.lo[0][e + 1], x.lo[1][e + 1]};
    const uint32_t hi[4] = {x.hi[0][e], x.hi[1][e], x.hi[0][e + 1], x.hi[1][e + 1]};
    const uint32_t b0 = SPLIT ? tf32_hi(w[e]) : __float_as_uint(w[e]);
    const uint32_t b1 = SPLIT ? tf32_hi(w[e + 1]) : __float_as_uint(w[e + 1]);
    if (s == 0) {
      mma_tf32_first(small, lo, b0, b1);
      mma_tf32_first(d, hi, b0, b1);
    } else {
      mma_tf32(small, lo, b0, b1);
      mma_tf32(d, hi, b0, b1);
    }
    if (SPLIT)
      mma_tf32(small, hi, tf32_lo(w[e]), tf32_lo(w[e + 1]));
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    sum[i] += d[i] + small[i];
}

// The cluster's tile: its adapter (`count`: rows without one) and its rows in order. False: no such tile.
struct LoraTile {
  int bins[kMaxBins];
  int rows[kTileRows];
  int warp_sums[kWarps];
  int adapter, part, n;
};

__device__ bool find_tile(const LoraArgs &a, LoraTile *t, int tile) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bins = a.count + 1;
  auto bin_of = [&](int r) {
    const int id = a.index[r];
    return id >= 0 && id < a.count ? id : a.count;
  };
  for (int i = threadIdx.x; i < bins; i += kThreads)
    t->bins[i] = 0;
  if (threadIdx.x == 0)
    t->adapter = -1;
  __syncthreads();
  for (int r = threadIdx.x; r < a.rows; r += kThreads)
    atomicAdd(&t->bins[bin_of(r)], 1);
  __syncthreads();
  // The adapter whose tiles hold number `tile`: a running sum over the adapters' tiles.
  int before = 0;
  for (int i0 = 0; i0 < bins; i0 += kThreads) {
    const int i = i0 + threadIdx.x, tiles = i < bins ? (t->bins[i] + kTileRows - 1) / kTileRows : 0;
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
      t->n = min(kTileRows, t->bins[i] - t->part * kTileRows);
    }
    before += all;
    __syncthreads();
  }
  if (t->adapter < 0)
    return false;
  // Its rows: every thread a run of neighbouring rows, ranked by the matches before it.
  const int per = (a.rows + kThreads - 1) / kThreads, r0 = min((int)threadIdx.x * per, a.rows), r1 = min(r0 + per, a.rows);
  int mine = 0;
  for (int r = r0; r < r1; r++)
    mine += bin_of(r) == t->adapter;
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
  for (int r = r0; r < r1; r++)
    if (bin_of(r) == t->adapter) {
      if (rank >= 0 && rank < kTileRows)
        t->rows[rank] = r;
      rank++;
    }
  __syncthreads();
  return true;
}

// Floats of a row of the tile's vectors: the rank in whole 32s, and 4 so that neighbouring rows lie in other banks.
__host__ __device__ constexpr int h_stride(int max_rank) { return (max_rank + 31) / 32 * 32 + 4; }

// parts clusters share a tile: each computes its vectors and takes a part of d.
template <typename W>
__global__ void __launch_bounds__(kThreads, 2) lora_tile_kernel(const LoraArgs a, int parts) {
  extern __shared__ __align__(16) float smem[];
  __shared__ LoraTile t;
  constexpr bool kSplit = sizeof(W) == 4;
  constexpr int kFlight = kSplit ? 2 : 4;  // column groups whose weights are under way at once
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank(), id = blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  if (!find_tile(a, &t, id / parts))
    return;  // the whole cluster
  const int part = id % parts, rows = t.n, hs = h_stride(a.max_rank);
  // [64][hs] each: this CTA's partial vectors (then the low parts), the vectors, their high parts.
  float *partial = smem, *h = smem + kTileRows * hs, *high = h + kTileRows * hs, *low = partial;
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
  const int rank32 = (w.rank + 31) / 32 * 32;
  // This warp's 16 rows, and its share of the work along n or d: the warps that a small tile leaves over take shares.
  const int groups = rows > 32 ? 4 : rows > 16 ? 2 : 1, ways = kWarps / groups, rg = warp % groups, way = warp / groups;
  const int i0 = 16 * rg + g, i1 = i0 + 8;
  const bool busy = 16 * rg < rows;

  // A x: this CTA's slice of n in steps of 32, the ways in turn; 64 rows of A at a time.
  const int n_slice = ((a.n + ctas - 1) / ctas + 31) / 32 * 32;
  const int n0 = min(rank * n_slice, a.n), n1 = min(n0 + n_slice, a.n);
  const bool x_wide = aligned16(a.x) && a.ldx % 4 == 0, a_wide = aligned16(A) && a.n % 8 == 0;
  for (int k0 = 0; k0 < w.rank; k0 += 64) {
    float sum[8][4];
#pragma unroll
    for (int c = 0; c < 8; c++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        sum[c][i] = 0.0f;
    if (busy) {
      const float *x0 = a.x + (long long)t.rows[min(i0, rows - 1)] * a.ldx;
      const float *x1 = a.x + (long long)t.rows[min(i1, rows - 1)] * a.ldx;
      // Whole steps first: every register is loaded again, for a step or half a step ahead, as soon as its value is
      // used.
      const int r1 = w.rank - 1, step = 32 * ways, first = n0 + 32 * way;
      const int whole = x_wide && a_wide && w.rank % 8 == 0 ? n1 - 31 : 0;  // steps that start below it
      const W *rows_a = A + (size_t)min(k0 + g, r1) * a.n + 8 * q;
      const size_t rows8 = (size_t)8 * a.n;
      auto row_of = [&](int c) { return rows_a + c * rows8; };
      Raw8<float> x[2];
      Raw8<W> wr[kFlight];
      x0 += 8 * q, x1 += 8 * q;
      if (first < whole) {
        x[0].load(x0 + first);
        x[1].load(x1 + first);
#pragma unroll
        for (int c = 0; c < kFlight; c++)
          if (k0 + 8 * c < w.rank)
            wr[c].load(row_of(c) + first);
      }
      int i = first;
      for (; i < whole; i += step) {
        const int next = i + step < whole ? i + step : first;  // past the end: any step's, which nothing uses
        Split16 xs;
        float v[8];
        x[0].get(v);
        xs.set(0, v);
        x[1].get(v);
        xs.set(1, v);
        x[0].load(x0 + next);
        x[1].load(x1 + next);
#pragma unroll
        for (int c = 0; c < 8; c++) {
          if (k0 + 8 * c < w.rank) {
            wr[c % kFlight].get(v);
            product32<kSplit>(sum[c], xs, v);
          }
          const int ahead = (c + kFlight) % 8;
          if (k0 + 8 * ahead < w.rank)
            wr[c % kFlight].load(row_of(ahead) + (c + kFlight < 8 ? i : next));
        }
      }
      for (; i < n1; i += step) {
        Split16 xs;
        float v[8];
#pragma unroll
        for (int r = 0; r < 2; r++) {
          x[r].load(r ? x1 : x0, i, n1 - 8 * q, x_wide);
          x[r].get(v);
          xs.set(r, v);
        }
#pragma unroll
        for (int c = 0; c < 8; c++)
          if (k0 + 8 * c < w.rank) {
            wr[0].load(A + (size_t)min(k0 + 8 * c + g, r1) * a.n + 8 * q, i, n1 - 8 * q, a_wide);
            wr[0].get(v);
            product32<kSplit>(sum[c], xs, v);
          }
      }
    }
    // The last way's sums, then the others' on top, into this CTA's partial vectors.
    for (int turn = ways - 1; turn >= 0; turn--) {
      if (busy && way == turn)
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int k = k0 + 8 * c + 2 * q + (i & 1);
            float *at = partial + (i < 2 ? i0 : i1) * hs + k;
            if (k < rank32)
              *at = k >= w.rank ? 0.0f : turn == ways - 1 ? sum[c][i] : *at + sum[c][i];
          }
      __syncthreads();
    }
  }
  // The cluster's sums: CTA c adds up its share of the rows from all CTAs in their order, then everyone fetches them.
  cluster.sync();
  const int own = (rows - rank + ctas - 1) / ctas;  // rows rank, rank + ctas, ...
  for (int e = threadIdx.x; e < own * rank32; e += kThreads) {
    const int n = e / rank32, at = (rank + n * ctas) * hs + e - n * rank32;
    float s = 0.0f;
#pragma unroll 8
    for (int c = 0; c < ctas; c++)
      s += *cluster.map_shared_rank(&partial[at], c);
    h[at] = s * w.scale;
  }
  cluster.sync();
#pragma unroll 4
  for (int e = threadIdx.x; e < rows * rank32; e += kThreads) {
    const int i = e / rank32, at = i * hs + e - i * rank32;
    const float v = *cluster.map_shared_rank(&h[at], i % ctas);
    high[at] = __uint_as_float(tf32_hi(v)), low[at] = __uint_as_float(tf32_lo(v));
  }
  cluster.sync();  // everything is fetched: a CTA may leave
  if (!busy)
    return;

  // B h: this CTA's slice of d, 32 columns at a time, the ways in turn.
  const int d_all = parts * ctas, d_slice = ((a.d + d_all - 1) / d_all + 31) / 32 * 32;
  const int d0 = min((part * ctas + rank) * d_slice, a.d), d1 = min(d0 + d_slice, a.d);
  const bool b_wide = aligned16(B) && w.rank % 8 == 0;
  const bool pairs = a.ldo % 2 == 0 && ((uintptr_t)a.out & 7) == 0 && (!a.base || (a.ldb % 2 == 0 && ((uintptr_t)a.base & 7) == 0));
  const long long r0 = t.rows[min(i0, rows - 1)], r1 = t.rows[min(i1, rows - 1)];
  float *const out[2] = {a.out + r0 * a.ldo + 2 * q, a.out + r1 * a.ldo + 2 * q};
  const float *const base[2] = {a.base ? a.base + r0 * a.ldb + 2 * q : nullptr, a.base ? a.base + r1 * a.ldb + 2 * q : nullptr};
  // As above: the weights of the first kAhead ranks and the base of the next step come during this one.
  constexpr int kAhead = 1;
  const int step = 32 * ways;
  Raw8<W> wr[kAhead][4];
  float2 y[4][2];
  const bool b_whole = b_wide && w.rank == rank32;
  auto load_b = [&](Raw8<W> &r, int d, int c, int k) {
    const W *row = B + (size_t)min(d + 8 * c + g, a.d - 1) * w.rank;
    if (b_whole)
      r.load(row + min(k, rank32 - 32) + 8 * q);
    else if (k < rank32)
      r.load(row, k + 8 * q, w.rank, b_wide);
  };
  auto load_base = [&](int d) {
    const bool whole = pairs && d + 32 <= d1;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const float *at = base[r] + d + 8 * c;
        const int left = d1 - (d + 8 * c + 2 * q);
        y[c][r] = make_float2(0.0f, 0.0f);
        if (a.base && whole) {
          y[c][r] = *reinterpret_cast<const float2 *>(at);
        } else if (a.base) {
          y[c][r].x = left > 0 ? at[0] : 0.0f;
          y[c][r].y = left > 1 ? at[1] : 0.0f;
        }
      }
  };
  const int first = d0 + 32 * way;
  if (rank32 && first < d1)
#pragma unroll
    for (int k = 0; k < kAhead; k++)
#pragma unroll
      for (int c = 0; c < 4; c++)
        load_b(wr[k][c], first, c, 32 * k);
  if (first < d1)
    load_base(first);
  for (int d = first; d < d1; d += step) {
    float prod[4][4];
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        prod[c][i] = 0.0f;
    for (int k0 = 0; k0 < rank32; k0 += 32 * kAhead) {
      const bool last = k0 + 32 * kAhead >= rank32;
#pragma unroll
      for (int n = 0; n < kAhead; n++) {
        const int k = k0 + 32 * n;
        if (k >= rank32)
          break;
        Split16 hv;
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int at = (r ? i1 : i0) * hs + k + 8 * q;
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(high + at + j), z = *reinterpret_cast<const uint4 *>(low + at + j);
            hv.hi[r][j] = x.x, hv.hi[r][j + 1] = x.y, hv.hi[r][j + 2] = x.z, hv.hi[r][j + 3] = x.w;
            hv.lo[r][j] = z.x, hv.lo[r][j + 1] = z.y, hv.lo[r][j + 2] = z.z, hv.lo[r][j + 3] = z.w;
          }
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
          float wv[8];
          wr[n][c].get(wv);
          product32<kSplit>(prod[c], hv, wv);
          load_b(wr[n][c], last ? d + step : d, c, last ? 32 * n : k + 32 * kAhead);
        }
      }
    }
    const bool whole = pairs && d + 32 <= d1;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const float2 o = make_float2(y[c][r].x + prod[c][2 * r], y[c][r].y + prod[c][2 * r + 1]);
        float *at = out[r] + d + 8 * c;
        const int left = (r ? i1 : i0) < rows ? d1 - (d + 8 * c + 2 * q) : 0;
        if (whole) {
          if (left)
            *reinterpret_cast<float2 *>(at) = o;
        } else {
          if (left > 0)
            at[0] = o.x;
          if (left > 1)
            at[1] = o.y;
        }
      }
    if (d + step < d1)
      load_base(d + step);
  }
}

template <typename W>
cudaError_t launch(void (*kernel)(LoraArgs, int), const LoraArgs &a, unsigned clusters, int ctas, int parts, size_t smem) {
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

template <typename W>
cudaError_t run(const LoraArgs &a) {
  constexpr int kCtas = 8;
  // Four rows an adapter make a tile worth its search (measured at d = n = 4096, rank 16).
  if (a.rows < 16 || a.rows < 4 * a.count || a.count >= kMaxBins)
    return launch<W>(lora_row_kernel<W>, a, (unsigned)a.rows, kCtas, 1, 0);
  const size_t smem = 3 * sizeof(float) * kTileRows * h_stride(a.max_rank);
  cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(lora_tile_kernel<W>),
                                (int)(3 * sizeof(float) * kTileRows * h_stride(kMaxRank)));
  for (int r = 0; r < a.rows && e == cudaSuccess; r += kMaxTileRows) {
    LoraArgs b = a;
    b.rows = a.rows - r < kMaxTileRows ? a.rows - r : kMaxTileRows;
    b.x += (long long)r * a.ldx, b.out += (long long)r * a.ldo, b.index += r;
    if (b.base)
      b.base += (long long)r * a.ldb;
    // At most this many tiles: the full ones, and one more for each adapter and the rows without one.
    const int some = b.count + 1 < b.rows ? b.count + 1 : b.rows, tiles = (b.rows - some) / kTileRows + some;
    const int few = kc_device_sms() / (kCtas * tiles), parts = few < 1 ? 1 : few > 4 ? 4 : few;
    e = launch<W>(lora_tile_kernel<W>, b, (unsigned)(tiles * parts), kCtas, parts, smem);
    if (e == cudaSuccess && r + kMaxTileRows < a.rows)
      kc_count_launch();
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
  if (rows < 0 || rows > (1 << 24) || n <= 0 || d <= 0 || count < 0 || max_rank <= 0 || max_rank > kMaxRank ||
      ldx < (size_t)n || ldo < (size_t)d || (base && ldb < (size_t)d)) {
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
                      n, d, rows};
  const cudaError_t e = type == K_F32 ? run<float>(a) : type == K_BF16 ? run<__nv_bfloat16>(a) : run<__half>(a);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
