// Attention of a batch of requests that share a prefix (k_attention_shared_rows). Row r of request b attends to the
// prefix [0, prefix) of one cache that all requests read and to positions [0, starts[b] + r] of the request's own
// cache. The prefix is read once for all rows of the batch and not once a request: its query vectors are gathered over
// the whole batch per KV head.
//
// Both parts give partial results per query vector and split of the positions: a reference m near the maximum of the
// scores (in units of log 2), the sum l of 2^(score - m) and the vector sum o of 2^(score - m) v. A merge joins them:
// out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i with M the largest m_i. Statistics and accumulators are fp32.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"
#include "tcgen05.cuh"

namespace {

constexpr int kMaxHd = 256;
constexpr int kPlanSms = 148;      // the plan is a function of the shape alone, so that the workspace's size is too
constexpr int kMaxSplits = 64;     // of the prefix, or of a request's own positions

constexpr float kLog2e = 1.44269504088896341f;

constexpr int kGenericThreads = 128;
constexpr int kGenericVecs = 32;   // query vectors per CTA
constexpr int kGenericPos = 32;    // positions per tile

struct SharedArgs {
  const float *q;             // [batch][rows][n_heads][hd]
  const float *pk, *pv;       // [n_kv][prefix_seq][hd]
  const float *k, *v;         // [batch][n_kv][seq][hd]
  const int *starts, *counts;
  float *out;                 // as q
  int8_t *oq;
  float *os;
  float2 *ml;                 // [splits][vectors]: the pairs (m, l)
  float *acc;                 // [splits][vectors][hd]
  int n_heads, n_kv, group, hd, prefix_seq, prefix, seq, batch, rows, gs;
  int vectors;                // batch * rows * n_heads
  int prefix_splits, own_splits;  // splits of the positions
  int tiles, own_tiles;           // query tiles per KV head: of the prefix part, of a request's own part
};

__device__ __forceinline__ int rows_of(const SharedArgs &a, int b) { return a.counts ? a.counts[b] : a.rows; }
// A request whose rows the kernels compute: a row count within the call and own positions within the cache.
__device__ __forceinline__ bool request_ok(const SharedArgs &a, int b, int count) {
  return count > 0 && count <= a.rows && a.starts[b] >= 0 && a.starts[b] <= a.seq - count;
}

// One work item: up to a tile of query vectors of one KV head against a range of one cache's positions.
struct Item {
  const float *k, *v;  // the KV head's rows
  int kv, split;       // split: index of the partial result
  int b;               // the request, or -1: the prefix
  int first, vecs;     // tile vectors: the flat (b, r, group member) index of the first, and how many
  int p0, p1;          // positions
};

// Vector i of KV head kv's flat list: index in the [batch][rows][n_heads] order.
__device__ __forceinline__ int vector_at(const SharedArgs &a, int kv, int i) {
  return (i / a.group) * a.n_heads + kv * a.group + i % a.group;
}

// Items 0 .. n_kv * tiles * prefix_splits - 1 are the prefix's, then one per (request, KV head, query tile, split).
// False: nothing to do.
__device__ __forceinline__ bool item_at(const SharedArgs &a, int id, int tile, Item *it) {
  const int prefix_items = a.n_kv * a.tiles * a.prefix_splits;
  if (id < prefix_items) {
    it->split = id % a.prefix_splits;
    id /= a.prefix_splits;
    it->kv = id % a.n_kv;
    it->b = -1;
    it->first = id / a.n_kv * tile;
    it->vecs = min(tile, a.batch * a.rows * a.group - it->first);
    it->k = a.pk + (size_t)it->kv * a.prefix_seq * a.hd;
    it->v = a.pv + (size_t)it->kv * a.prefix_seq * a.hd;
    it->p0 = (int)((long long)a.prefix * it->split / a.prefix_splits);
    it->p1 = (int)((long long)a.prefix * (it->split + 1) / a.prefix_splits);
    return true;
  }
  id -= prefix_items;
  const int split = id % a.own_splits;
  id /= a.own_splits;
  it->split = a.prefix_splits + split;
  const int own_tile = id % a.own_tiles * tile;
  id /= a.own_tiles;
  it->kv = id % a.n_kv;
  it->b = id / a.n_kv;
  const int count = rows_of(a, it->b);
  if (!request_ok(a, it->b, count)) {
    if (count != 0 && threadIdx.x == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    return false;
  }
  it->first = it->b * a.rows * a.group + own_tile;
  it->vecs = min(tile, count * a.group - own_tile);
  if (it->vecs <= 0)
    return false;
  const size_t head = ((size_t)it->b * a.n_kv + it->kv) * a.seq * a.hd;
  it->k = a.k + head;
  it->v = a.v + head;
  const int length = a.starts[it->b] + count;
  it->p0 = (int)((long long)length * split / a.own_splits);
  it->p1 = (int)((long long)length * (split + 1) / a.own_splits);
  return true;
}

// Positions of the item that its vector i (a flat index) sees: [p0, limit).
__device__ __forceinline__ int limit_of(const SharedArgs &a, const Item &it, int i) {
  if (it.b < 0)
    return it.p1;
  return min(it.p1, a.starts[it.b] + (i - it.b * a.rows * a.group) / a.group + 1);
}

// Any head_dim up to 256 and any alignment, in fp32 FMAs: a warp takes 8 of the tile's 32 vectors in turn, its lanes
// the 32 positions of a tile for the scores and the head's elements for the sums.
__global__ void __launch_bounds__(kGenericThreads) shared_generic_kernel(const SharedArgs a) {
  extern __shared__ float smem[];
  pdl_wait();
  pdl_launch_dependents();
  Item it;
  if (!item_at(a, blockIdx.x, kGenericVecs, &it))
    return;
  const int hd = a.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *ks = smem;                                 // [32][hd + 1]
  float *vs = ks + kGenericPos * (hd + 1);          // [32][hd]
  float *qs = vs + kGenericPos * hd;                // [4 warps][hd]
  const float scale = rsqrtf((float)hd) * kLog2e;
  for (int v0 = 0; v0 < it.vecs; v0 += 4) {
    // One vector a warp at a time; the tiles come again from the cache for the next four.
    const int i = it.first + v0 + warp;
    const bool have = v0 + warp < it.vecs;
    const int vec = have ? vector_at(a, it.kv, i) : 0;
    const int limit = have ? limit_of(a, it, i) : it.p0;
    float m = -INFINITY, l = 0.0f, acc[kMaxHd / 32];
#pragma unroll
    for (int e = 0; e < kMaxHd / 32; e++)
      acc[e] = 0.0f;
    for (int e = lane; e < hd; e += 32)
      qs[warp * hd + e] = have ? a.q[(size_t)vec * hd + e] * scale : 0.0f;
    for (int t0 = it.p0; t0 < it.p1; t0 += kGenericPos) {
      const int n = min(kGenericPos, it.p1 - t0);
      __syncthreads();
      for (int e = threadIdx.x; e < n * hd; e += kGenericThreads) {
        const int p = e / hd, c = e - p * hd;
        ks[p * (hd + 1) + c] = it.k[(size_t)t0 * hd + e];
        vs[e] = it.v[(size_t)t0 * hd + e];
      }
      __syncthreads();
      const bool seen = t0 + lane < limit;
      float s = 0.0f;
      if (seen)
        for (int e = 0; e < hd; e++)
          s = fmaf(qs[warp * hd + e], ks[lane * (hd + 1) + e], s);
      float top = seen ? s : -INFINITY;
#pragma unroll
      for (int o = 16; o; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (top == -INFINITY && t0 >= limit)
        continue;
      const float m_new = fmaxf(m, top);
      const float keep = m == -INFINITY ? 0.0f : exp2f(m - m_new);
      const float p = seen ? exp2f(s - m_new) : 0.0f;
      float sum = p;
#pragma unroll
      for (int o = 16; o; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = l * keep + sum;
      m = m_new;
#pragma unroll
      for (int e = 0; e < kMaxHd / 32; e++)
        acc[e] *= keep;
      const int live = min(n, limit - t0);
      for (int j = 0; j < live; j++) {
        const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
        for (int e = 0; e < kMaxHd / 32; e++)
          if (32 * e + lane < hd)
            acc[e] = fmaf(pj, vs[j * hd + 32 * e + lane], acc[e]);
      }
    }
    if (have) {
      const size_t at = (size_t)it.split * a.vectors + vec;
#pragma unroll
      for (int e = 0; e < kMaxHd / 32; e++)
        if (32 * e + lane < hd)
          a.acc[at * hd + 32 * e + lane] = acc[e];
      if (lane == 0)
        a.ml[at] = make_float2(m, l);
    }
    __syncthreads();
  }
}


// ---- tensor-core kernel -------------------------------------------------------------------------------------------

// head_dim <= 128 in whole 16-byte units. A CTA takes one item: up to 128 query vectors of a KV head against a range of
// positions in tiles of 64, S = Q K^T and O += P V on tcgen05 with accumulators in TMEM.
//
// fp32 products on half-precision tensor cores: x = 2^-k (hi + lo) with hi and lo fp16, 22 bits of x, and
// x y = 2^-(k + k') (hi hi' + hi lo' + lo hi') up to 2^-22 of the product (what is dropped, lo lo', is below the
// rounding of lo). The power 2^k puts the largest magnitude of a query vector, of a tile of keys or of a tile of values
// just below 2^15, so no finite input overflows and a value 2^-17 of the largest still keeps its 22 bits. k of the
// keys goes into the scores' scale; k of the values into the probabilities (exact powers of two both).
//
// Warps: 0-3 the softmax, a thread per query vector (TMEM lane); 4 issues the MMAs; 5-12 read keys and values from
// global memory, split them and store them as the MMA's operands (values transposed, so both are K-major), two stages.
// The running maximum is a reference m that moves only when a score exceeds it by 8 (a factor of 256): O in TMEM is
// seldom rescaled.
constexpr int kTcVecs = 128, kTcPos = 64;
constexpr int kSoftWarps = 4, kConvWarps = 8;
constexpr int kTcThreads = 32 * (kSoftWarps + 1 + kConvWarps);
constexpr int kConvThreads = 32 * kConvWarps;
constexpr uint32_t kTmemS = 0, kTmemP = 128, kTmemO = 256, kTmemCols = 512;
constexpr int kPShift = 7;  // probabilities are up to 2^8 (the lazy reference) and carry this power of two more

template <int HD>
struct TcSmem {
  static constexpr int q_bytes = kTcVecs * HD * 2;  // hi or lo
  static constexpr int kv_bytes = kTcPos * HD * 2;  // hi or lo of K or V
  static constexpr int stage = 4 * kv_bytes;
  static constexpr int stages_at = 2 * q_bytes;
  static constexpr int tail_at = stages_at + 2 * stage;
  static constexpr int total = tail_at + 2048 + 1024;  // the tail, and room to align the start to 1 KiB
};

struct TcTail {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], sempty[2], pfull[2], pvdone[2];
  uint32_t tmem;
  int abort_flag;
  int kshift[4], vshift[4];      // powers of two of the keys' and values' tiles
  unsigned wmax[4][kConvWarps];  // magnitudes while they are agreed on
  int qshift[kTcVecs];
};
static_assert(sizeof(TcTail) <= 2048, "the tail's room");

// A whole warp's bounded wait, with one answer for all lanes: false once any wait of the CTA has given up.
__device__ __forceinline__ bool tc_wait(uint64_t *bar, unsigned parity, volatile int *abort_flag) {
  bool ok = *abort_flag == 0;
  if (ok && !mbar_wait_sleep_bounded(bar, parity)) {
    *abort_flag = 1;
    ok = false;
  }
  return __all_sync(0xffffffffu, ok);
}

// kind::f16 instruction descriptor: fp16 A and B, both K-major, fp32 accumulators, M x N.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// A from TMEM: lane = row, a 32-bit column holds two neighbouring elements.
__device__ __forceinline__ void umma_f16_ta(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Writes 32 lanes (this warp's quadrant) x 32 consecutive columns.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// The power k for a largest magnitude (its bits): magnitudes times 2^k below 2^15. At most 126, so that 2^k is a
// number; tiny and zero maxima take that.
__device__ __forceinline__ int shift_for(unsigned max_bits) {
  const int e = (int)(max_bits >> 23) - 127;
  return min(14 - e, 126);
}
__device__ __forceinline__ float pow2(int k) { return ldexpf(1.0f, k); }

// Two scaled values as packed fp16 high parts and the packed rest.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The largest of the converters' magnitudes (bits), agreed over their warps. `slot` alternates, so that a value is not
// overwritten while another warp still reads it.
__device__ __forceinline__ unsigned agree_max(TcTail *t, int slot, unsigned mine, int cw, int lane) {
  mine = __reduce_max_sync(0xffffffffu, mine);
  if (lane == 0)
    t->wmax[slot][cw] = mine;
  asm volatile("bar.sync 1, %0;" ::"n"(kConvThreads) : "memory");
  unsigned m = 0;
#pragma unroll
  for (int w = 0; w < kConvWarps; w++)
    m = max(m, t->wmax[slot][w]);
  return m;
}

template <int HD>
__global__ void __launch_bounds__(kTcThreads, 1) shared_tc_kernel(const SharedArgs a) {
  using L = TcSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  TcTail *t = reinterpret_cast<TcTail *>(smem + L::tail_at);
  volatile int *abort_flag = &t->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  Item it;
  if (!item_at(a, blockIdx.x, kTcVecs, &it))
    return;
  const int tiles = (it.p1 - it.p0 + kTcPos - 1) / kTcPos;
  if (tiles <= 0) {
    for (int i = threadIdx.x; i < it.vecs; i += kTcThreads)
      a.ml[(size_t)it.split * a.vectors + vector_at(a, it.kv, it.first + i)] = make_float2(-INFINITY, 0.0f);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&t->kfull[i], kConvWarps);
      mbar_init(&t->vfull[i], kConvWarps);
      mbar_init(&t->kempty[i], 1);
      mbar_init(&t->vempty[i], 1);
      mbar_init(&t->sfull[i], 1);
      mbar_init(&t->sempty[i], kSoftWarps);
      mbar_init(&t->pfull[i], kSoftWarps);
      mbar_init(&t->pvdone[i], 1);
    }
    t->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kSoftWarps)
    tmem_alloc(&t->tmem, kTmemCols);

  const int hd = a.hd;
  // The queries: a warp per vector, split with the vector's own power of two. Vectors not in use are zeros.
  for (int i = warp; i < kTcVecs; i += kTcThreads / 32) {
    constexpr int E = HD / 32;  // 4 or 2 elements a lane
    float x[E];
    bool use = i < it.vecs;
    if (use) {
      const int flat = it.first + i, row = flat / a.group, b = row / a.rows;
      const int count = rows_of(a, b);
      use = row - b * a.rows < count && request_ok(a, b, count);
    }
    const float *src = a.q + (size_t)(use ? vector_at(a, it.kv, it.first + i) : 0) * hd;
    unsigned mx = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
      x[e] = use && lane * E + e < hd ? src[lane * E + e] : 0.0f;
      mx = max(mx, __float_as_uint(fabsf(x[e])));
    }
    const int k = shift_for(__reduce_max_sync(0xffffffffu, mx));
    const float f = pow2(k);
    if (lane == 0)
      t->qshift[i] = k;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      uint32_t hi, lo;
      split2(x[e] * f, x[e + 1] * f, hi, lo);
      const int c = lane * E + e;
      const int at = (c >> 6) * (kTcVecs * 128) + i * 128 + ((((c & 63) >> 3) ^ (i & 7)) << 4) + (c & 7) * 2;
      *reinterpret_cast<uint32_t *>(smem + at) = hi;
      *reinterpret_cast<uint32_t *>(smem + L::q_bytes + at) = lo;
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = t->tmem;

  if (warp > kSoftWarps) {
    // ---- converters ----
    const int ct = threadIdx.x - 32 * (kSoftWarps + 1), cw = warp - kSoftWarps - 1;
    constexpr int kChunks = kTcPos * HD / 8 / kConvThreads;  // chunks of 8 values per thread: 4 or 2
    float kx[kChunks][8], vx[kChunks][8];
    auto load_k = [&](int tile) {
      const int p0 = it.p0 + tile * kTcPos;
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        const int c = i * kConvThreads + ct, r = c / (HD / 8), e = c % (HD / 8) * 8;
        const float *src = it.k + (size_t)(p0 + r) * hd + e;
        const bool in = p0 + r < it.p1;
        float4 x = make_float4(0, 0, 0, 0), y = x;
        if (in && e < hd)
          x = *reinterpret_cast<const float4 *>(src);
        if (in && e + 4 < hd)
          y = *reinterpret_cast<const float4 *>(src + 4);
        kx[i][0] = x.x, kx[i][1] = x.y, kx[i][2] = x.z, kx[i][3] = x.w;
        kx[i][4] = y.x, kx[i][5] = y.y, kx[i][6] = y.z, kx[i][7] = y.w;
      }
    };
    auto load_v = [&](int tile) {
      const int p0 = it.p0 + tile * kTcPos;
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        const int c = i * kConvThreads + ct, d = c % HD, r = c / HD * 8;
#pragma unroll
        for (int j = 0; j < 8; j++)
          vx[i][j] = p0 + r + j < it.p1 && d < hd ? it.v[(size_t)(p0 + r + j) * hd + d] : 0.0f;
      }
    };
    auto largest = [&](const float (&x)[kChunks][8]) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < kChunks; i++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          m = max(m, __float_as_uint(fabsf(x[i][j])));
      return m;
    };
    auto store = [&](uint8_t *hi_at, uint8_t *lo_at, const float (&x)[8], float f) {
      uint4 hi, lo;
      split2(x[0] * f, x[1] * f, hi.x, lo.x);
      split2(x[2] * f, x[3] * f, hi.y, lo.y);
      split2(x[4] * f, x[5] * f, hi.z, lo.z);
      split2(x[6] * f, x[7] * f, hi.w, lo.w);
      *reinterpret_cast<uint4 *>(hi_at) = hi;
      *reinterpret_cast<uint4 *>(lo_at) = lo;
    };
    load_k(0);
    load_v(0);
    for (int j = 0; j < tiles; j++) {
      const int s = j & 1, use = j >> 1;
      uint8_t *stage = smem + L::stages_at + s * L::stage;
      const int ks = shift_for(agree_max(t, 2 * s, largest(kx), cw, lane));
      const float kf = pow2(ks);
      tc_wait(&t->kempty[s], (use & 1) ^ 1, abort_flag);
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        const int c = i * kConvThreads + ct, r = c / (HD / 8), e8 = c % (HD / 8);
        uint8_t *at = stage + (e8 >> 3) * (kTcPos * 128) + r * 128 + (((e8 & 7) ^ (r & 7)) << 4);
        store(at, at + L::kv_bytes, kx[i], kf);
      }
      if (ct == 0)
        t->kshift[j & 3] = ks;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->kfull[s]);
      if (j + 1 < tiles)
        load_k(j + 1);
      const int vs = shift_for(agree_max(t, 2 * s + 1, largest(vx), cw, lane));
      const float vf = pow2(vs);
      tc_wait(&t->vempty[s], (use & 1) ^ 1, abort_flag);
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        const int c = i * kConvThreads + ct, d = c % HD, r8 = c / HD;
        uint8_t *at = stage + 2 * L::kv_bytes + d * 128 + ((r8 ^ (d & 7)) << 4);
        store(at, at + L::kv_bytes, vx[i], vf);
      }
      if (ct == 0)
        t->vshift[j & 3] = vs;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->vfull[s]);
      if (j + 1 < tiles)
        load_v(j + 1);
    }
  } else if (warp == kSoftWarps) {
    // ---- MMA issue: the scores of tile j + 1 go out before the sums of tile j, so that they run under its softmax ----
    const uint32_t idesc_s = umma_idesc_f16(kTcVecs, kTcPos), idesc_o = umma_idesc_f16(kTcVecs, HD);
    auto scores = [&](int j) {
      const int s = j & 1, use = j >> 1;
      if (!tc_wait(&t->kfull[s], use & 1, abort_flag) || !tc_wait(&t->sempty[s], (use & 1) ^ 1, abort_flag))
        return;
      tc_fence_after();
      if (lane == 0) {
        const uint8_t *k = smem + L::stages_at + s * L::stage;
        const uint32_t d = tmem + kTmemS + 64 * s;
#pragma unroll
        for (int term = 0; term < 3; term++) {  // lo hi, hi lo, hi hi: the small terms first
          const uint8_t *qa = smem + (term == 0 ? L::q_bytes : 0), *kb = k + (term == 1 ? L::kv_bytes : 0);
#pragma unroll
          for (int c = 0; c < HD / 16; c++)
            umma_f16(d, umma_desc_sw128(qa + (c >> 2) * (kTcVecs * 128)) + 2 * (c & 3),
                     umma_desc_sw128(kb + (c >> 2) * (kTcPos * 128)) + 2 * (c & 3), idesc_s, term || c);
        }
        umma_commit(&t->sfull[s]);
        umma_commit(&t->kempty[s]);
      }
      __syncwarp();
    };
    scores(0);
    for (int j = 0; j < tiles; j++) {
      if (j + 1 < tiles)
        scores(j + 1);
      const int s = j & 1, use = j >> 1;
      if (!tc_wait(&t->vfull[s], use & 1, abort_flag) || !tc_wait(&t->pfull[s], use & 1, abort_flag))
        break;
      tc_fence_after();
      if (lane == 0) {
        const uint8_t *v = smem + L::stages_at + s * L::stage + 2 * L::kv_bytes;
        const uint32_t p = tmem + kTmemP + 64 * s;
#pragma unroll
        for (int term = 0; term < 3; term++) {
          const uint32_t pa = p + (term == 0 ? 32 : 0);
          const uint8_t *vb = v + (term == 1 ? L::kv_bytes : 0);
#pragma unroll
          for (int c = 0; c < kTcPos / 16; c++)
            umma_f16_ta(tmem + kTmemO, pa + 8 * c, umma_desc_sw128(vb) + 2 * c, idesc_o, j || term || c);
        }
        umma_commit(&t->pvdone[s]);
        umma_commit(&t->vempty[s]);
      }
      __syncwarp();
    }
  } else {
    // ---- softmax: a thread per query vector ----
    const uint32_t quadrant = tmem + ((uint32_t)(32 * warp) << 16);
    const int i = 32 * warp + lane;
    const bool have = i < it.vecs, busy = 32 * warp < it.vecs;
    const int limit = have ? limit_of(a, it, it.first + i) : it.p0;
    const int lowest = __reduce_min_sync(0xffffffffu, have ? limit : 0x7fffffff);
    const int qs = t->qshift[i];
    const float scale = rsqrtf((float)hd) * kLog2e;
    float m = -INFINITY, l = 0.0f;
    int vref = 0;  // O holds sums times 2^(kPShift + vref)
    for (int j = 0; j < tiles; j++) {
      const int s = j & 1, use = j >> 1;
      if (!tc_wait(&t->sfull[s], use & 1, abort_flag))
        break;
      tc_fence_after();
      uint32_t r0[32], r1[32];
      if (busy) {
        tmem_ld32(quadrant + kTmemS + 64 * s, r0);
        tmem_ld32(quadrant + kTmemS + 64 * s + 32, r1);
        tmem_wait_ld();
      }
      const int ks = t->kshift[j & 3];
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->sempty[s]);
      // The values' power of two for the probabilities.
      if (!tc_wait(&t->vfull[s], use & 1, abort_flag))
        break;
      const int vs = t->vshift[j & 3];
      if (busy) {
        const int p0 = it.p0 + j * kTcPos;
        if (p0 + kTcPos > lowest) {
#pragma unroll
          for (int c = 0; c < 32; c++) {
            r0[c] = p0 + c < limit ? r0[c] : 0xff800000u;
            r1[c] = p0 + 32 + c < limit ? r1[c] : 0xff800000u;
          }
        }
        const float factor = ldexpf(scale, -(qs + ks));
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 32; c++)
          top = fmaxf(top, fmaxf(__uint_as_float(r0[c]), __uint_as_float(r1[c])));
        top *= factor;
        // Move the reference when a score exceeds it by more than 8, and O's power when the values have grown.
        const bool up = top > m + 8.0f || (m == -INFINITY && top > m);
        const float m_new = up ? top : m;
        const int vref_new = j == 0 || vs < vref ? vs - 1 : vref;
        const float keep = !up ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - m_new);
        if (j > 0 && (vref_new != vref || __any_sync(0xffffffffu, up))) {
          if (!tc_wait(&t->pvdone[s ^ 1], ((j - 1) >> 1) & 1, abort_flag))
            break;
          tc_fence_after();
          const float f = keep * pow2(vref_new - vref);
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(quadrant + kTmemO + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(quadrant + kTmemO + c, o);
          }
        }
        l *= keep;
        m = m_new;
        vref = vref_new;
        const float base = m == -INFINITY ? 0.0f : m, grow = pow2(kPShift - vs + vref);
        float sum = 0.0f;
        uint32_t hi[32], lo[32];
#pragma unroll
        for (int c = 0; c < 16; c++) {
          const float x = ex2(fmaf(__uint_as_float(r0[2 * c]), factor, -base));
          const float y = ex2(fmaf(__uint_as_float(r0[2 * c + 1]), factor, -base));
          sum += x + y;
          split2(x * grow, y * grow, hi[c], lo[c]);
        }
#pragma unroll
        for (int c = 0; c < 16; c++) {
          const float x = ex2(fmaf(__uint_as_float(r1[2 * c]), factor, -base));
          const float y = ex2(fmaf(__uint_as_float(r1[2 * c + 1]), factor, -base));
          sum += x + y;
          split2(x * grow, y * grow, hi[16 + c], lo[16 + c]);
        }
        l += sum;
        // The probabilities' buffer: free once the sums of two tiles ago are done.
        if (j > 1 && !tc_wait(&t->pvdone[s], ((j - 2) >> 1) & 1, abort_flag))
          break;
        tmem_st32(quadrant + kTmemP + 64 * s, hi);
        tmem_st32(quadrant + kTmemP + 64 * s + 32, lo);
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->pfull[s]);
    }
    if (busy && tc_wait(&t->pvdone[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, abort_flag)) {
      tc_fence_after();
      const size_t at = (size_t)it.split * a.vectors + (have ? vector_at(a, it.kv, it.first + i) : 0);
      if (have)
        a.ml[at] = make_float2(m, l);
      const int down = -(kPShift + vref);
      const float f0 = pow2(down / 2), f1 = pow2(down - down / 2);  // 2^down itself may not be a number
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        tmem_ld32(quadrant + kTmemO + c, o);
        tmem_wait_ld();
        if (have)
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (c + e < hd)
              *reinterpret_cast<float4 *>(a.acc + at * hd + c + e) =
                  make_float4(__uint_as_float(o[e]) * f0 * f1, __uint_as_float(o[e + 1]) * f0 * f1,
                              __uint_as_float(o[e + 2]) * f0 * f1, __uint_as_float(o[e + 3]) * f0 * f1);
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == kSoftWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int HD>
cudaError_t launch_tc(const SharedArgs &a, unsigned items) {
  const cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(shared_tc_kernel<HD>), TcSmem<HD>::total);
  return e != cudaSuccess ? e
                          : kc_launch_pdl(shared_tc_kernel<HD>, dim3(items), dim3(kTcThreads), TcSmem<HD>::total,
                                          kc_stream(), a);
}

// Heads of whole 16-byte units at 16-byte addresses.
bool tc_shape(const SharedArgs &a) {
  const uintptr_t at = (uintptr_t)a.k | (uintptr_t)a.v | (a.prefix ? (uintptr_t)a.pk | (uintptr_t)a.pv : 0);
  return a.hd <= 128 && a.hd % 4 == 0 && !(at & 15);
}

// A warp per output vector: the splits joined in their order, and optionally quantized in gs-groups as k_quantize does.
__global__ void __launch_bounds__(256) shared_merge_kernel(const SharedArgs a) {
  __shared__ float weights[8][2 * kMaxSplits], outs[8][kMaxHd];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vec = blockIdx.x * 8 + warp;
  if (vec >= a.vectors)
    return;
  const int row = vec / a.n_heads, b = row / a.rows, r = row - b * a.rows;
  const int count = rows_of(a, b);
  if (!request_ok(a, b, count) || r >= count)
    return;  // rows out of use stay as they were
  const int splits = a.prefix_splits + a.own_splits, hd = a.hd;
  float top = -INFINITY;
  for (int s = lane; s < splits; s += 32)
    top = fmaxf(top, a.ml[(size_t)s * a.vectors + vec].x);
#pragma unroll
  for (int o = 16; o; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.0f;
  for (int s = lane; s < splits; s += 32) {
    const float2 ml = a.ml[(size_t)s * a.vectors + vec];
    const float w = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - top);
    weights[warp][s] = w;
    sum += w * ml.y;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncwarp();
  for (int e = lane; e < hd; e += 32) {
    float o = 0.0f;
    for (int s = 0; s < splits; s++)
      if (weights[warp][s] != 0.0f)
        o = fmaf(weights[warp][s], a.acc[((size_t)s * a.vectors + vec) * hd + e], o);
    o /= sum;
    a.out[(size_t)vec * hd + e] = o;
    outs[warp][e] = o;
  }
  if (!a.oq)
    return;
  __syncwarp();
  for (int g = 0; g < hd; g += a.gs) {
    float mx = 0.0f;
    bool bad = false;
    for (int e = lane; e < a.gs; e += 32) {
      const float v = outs[warp][g + e];
      bad |= !(fabsf(v) < INFINITY);
      mx = fmaxf(mx, fabsf(v));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (bad)
      kc_raise(KC_ERR_NONFINITE);
    const float scale = __fdiv_rn(mx, 127.0f);
    const size_t at = (size_t)vec * hd + g;
    for (int e = lane; e < a.gs; e += 32)
      a.oq[at + e] = (int8_t)quantize_value(outs[warp][g + e], scale);
    if (lane == 0)
      a.os[at / a.gs] = scale;
  }
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// How many ways a work's partial results split the prefix and each request's own positions at most.
int most_prefix_splits(int n_kv, int group, int batch, int rows) {
  const int tiles = ceil_div(batch * rows * group, 128);
  const int s = 2 * kPlanSms / (n_kv * tiles);
  return s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s;
}
int most_own_splits(int n_kv, int batch) {
  const int s = 2 * kPlanSms / (n_kv * batch);
  return s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s;
}

bool shape_ok(int n_heads, int n_kv, int hd, int batch, int rows) {
  return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && hd > 0 && hd <= kMaxHd && batch > 0 && rows > 0 &&
         (long long)batch * rows * n_heads <= (1 << 24);
}

// Floats of n (m, l) pairs, to a whole number of 16-byte units: the accumulators behind them stay aligned.
size_t pairs_floats(size_t n) { return (2 * n + 3) & ~(size_t)3; }

size_t partial_floats(int n_heads, int n_kv, int hd, int batch, int rows) {
  const size_t splits = (size_t)most_prefix_splits(n_kv, n_heads / n_kv, batch, rows) + most_own_splits(n_kv, batch);
  const size_t pairs = splits * ((size_t)batch * rows * n_heads);
  return pairs_floats(pairs) + pairs * hd;
}

size_t generic_smem(int hd) { return sizeof(float) * ((size_t)kGenericPos * (2 * hd + 1) + 4 * (size_t)hd); }

}  // namespace

extern "C" {

size_t k_attention_shared_bytes(int n_heads, int n_kv_heads, int head_dim, int batch, int rows) {
  if (!shape_ok(n_heads, n_kv_heads, head_dim, batch, rows))
    return 0;
  return sizeof(float) * partial_floats(n_heads, n_kv_heads, head_dim, batch, rows);
}

void k_attention_shared_init(AttentionWork *work, int n_heads, int n_kv_heads, int head_dim, int batch, int rows,
                             void *memory) {
  const size_t bytes = k_attention_shared_bytes(n_heads, n_kv_heads, head_dim, batch, rows);
  memset(work, 0, sizeof(*work));
  if (!bytes) {
    kc_fail("k_attention_shared_init: invalid shape");
    return;
  }
  if ((uintptr_t)memory & 15) {
    kc_fail("k_attention_shared_init: the memory must be 16-byte aligned");
    return;
  }
  void *base = memory;
  if (!base && cudaMalloc(&base, bytes) != cudaSuccess) {
    cudaGetLastError();
    kc_fail("k_attention_shared_init: cannot allocate %zu bytes of attention work", bytes);
    return;
  }
  work->partial = static_cast<float *>(base);
  work->max_chunks = most_prefix_splits(n_kv_heads, n_heads / n_kv_heads, batch, rows) +
                     most_own_splits(n_kv_heads, batch);
  work->n_heads = n_heads;
  work->head_dim = head_dim;
  work->workers = 1;
  work->external = memory != nullptr;
  work->capacity = bytes / sizeof(float);
}

void k_attention_shared_rows(float *out, int8_t *oq, float *os, const float *q, const float *prefix_key,
                             const float *prefix_value, int prefix_seq_len, int prefix, const float *key_cache,
                             const float *value_cache, const int *starts, const int *counts, AttentionWork *work,
                             int n_heads, int n_kv_heads, int head_dim, int seq_len, int batch, int rows, int gs) {
  const char *name = "k_attention_shared_rows";
  if (batch == 0 || rows == 0)
    return;
  if (!shape_ok(n_heads, n_kv_heads, head_dim, batch, rows) || seq_len <= 0 || rows > seq_len || prefix < 0 ||
      prefix > prefix_seq_len) {
    kc_fail("%s: invalid shape heads=%d/%d head_dim=%d batch=%d rows=%d seq_len=%d prefix=%d of %d", name, n_heads,
            n_kv_heads, head_dim, batch, rows, seq_len, prefix, prefix_seq_len);
    return;
  }
  if (!out || !q || !key_cache || !value_cache || !starts || (prefix && (!prefix_key || !prefix_value)) ||
      (oq && !os)) {
    kc_fail("%s: missing output, queries, caches or starts", name);
    return;
  }
  if (oq && (gs <= 0 || head_dim % gs)) {
    kc_fail("%s: group size %d does not divide the head's %d outputs", name, gs, head_dim);
    return;
  }
  if (!work || !work->partial || work->n_heads != n_heads || work->head_dim != head_dim ||
      work->capacity < partial_floats(n_heads, n_kv_heads, head_dim, batch, rows)) {
    kc_fail("%s: the attention work is missing or too small for this shape", name);
    return;
  }
  SharedArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q, a.pk = prefix_key, a.pv = prefix_value, a.k = key_cache, a.v = value_cache;
  a.starts = starts, a.counts = counts, a.out = out, a.oq = oq, a.os = os;
  a.n_heads = n_heads, a.n_kv = n_kv_heads, a.group = n_heads / n_kv_heads, a.hd = head_dim;
  a.prefix_seq = prefix_seq_len, a.prefix = prefix, a.seq = seq_len, a.batch = batch, a.rows = rows, a.gs = gs;
  a.vectors = batch * rows * n_heads;
  const int most_p = most_prefix_splits(n_kv_heads, a.group, batch, rows), most_o = most_own_splits(n_kv_heads, batch);
  a.prefix_splits = prefix ? (ceil_div(prefix, 64) < most_p ? ceil_div(prefix, 64) : most_p) : 0;
  a.own_splits = ceil_div(seq_len, 64) < most_o ? ceil_div(seq_len, 64) : most_o;
  const size_t splits = (size_t)a.prefix_splits + a.own_splits;
  a.ml = reinterpret_cast<float2 *>(work->partial);
  a.acc = work->partial + pairs_floats(splits * a.vectors);
  const bool tc = tc_shape(a);
  const int tile = tc ? kTcVecs : kGenericVecs;
  a.tiles = ceil_div(batch * rows * a.group, tile);
  a.own_tiles = ceil_div(rows * a.group, tile);
  const long long items = (long long)n_kv_heads * ((long long)a.tiles * a.prefix_splits +
                                                   (long long)batch * a.own_tiles * a.own_splits);
  if (items > 0x7fffffff) {
    kc_fail("%s: batch %d of %d rows is too large", name, batch, rows);
    return;
  }
  cudaError_t e;
  if (tc) {
    e = head_dim > 64 ? launch_tc<128>(a, (unsigned)items) : launch_tc<64>(a, (unsigned)items);
  } else {
    e = kc_allow_smem(reinterpret_cast<const void *>(shared_generic_kernel), (int)generic_smem(kMaxHd));
    if (e == cudaSuccess)
      e = kc_launch_pdl(shared_generic_kernel, dim3((unsigned)items), dim3(kGenericThreads), generic_smem(head_dim),
                        kc_stream(), a);
  }
  if (e == cudaSuccess) {
    kc_count_launch();
    e = kc_launch_pdl(shared_merge_kernel, dim3((unsigned)ceil_div(a.vectors, 8)), dim3(256), 0, kc_stream(), a);
    if (e == cudaSuccess)
      kc_count_launch();
  }
  if (e != cudaSuccess)
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
