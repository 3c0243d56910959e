// Serving from a paged K/V cache: keys and values stored into their pages with the rotation of queries and keys
// (k_rope_kv_store_paged), and attention over the pages (k_attention_paged_rows).
//
// A cache is [pages][n_kv][page_size][hd]; position p of request b lies in row p % page_size of page
// table[b][p / page_size].
//
// Attention, per query vector q (already rotated) with scores s_p = q . k_p / sqrt(hd) over the positions that it sees:
// out = sum_p 2^(s'_p - m) v_p / sum_p 2^(s'_p - m), s' = s log2(e), m a running maximum. The work is cut into segments,
// a KV head of a request with up to `block` of its query vectors, and each segment's positions into tiles; the tiles of
// all segments form one row, of which every CTA takes an equal, contiguous share, whatever the requests' lengths are. A
// segment that lies in several shares leaves partial results (m, l = sum 2^(s' - m), o = sum 2^(s' - m) v) that the CTA
// to finish last joins, in the order of the shares.
//
// Times in these files are device times in a graph of calls, except where "back to back" stands: calls of the Python mirror one
// after another, whose own work is 6 to 8 us each.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"
#include "paged.cuh"
#include "tcgen05.cuh"

using namespace paged;

namespace {

constexpr int kMaxPositions = 0x7fffffff - 1024;  // tiles are numbered past the last one

// ---- storing ------------------------------------------------------------------------------------------------------

struct StoreArgs {
  float *q_out;
  const float *q, *k, *v, *rope;
  void *key, *value;
  const int *table, *starts, *counts;
  long long q_out_ld, q_ld, kv_ld;
  size_t page_stride;
  int pages, page_size, max_pages, positions, n_heads, n_kv, hd, batch, rows, per_row;
  Divisor by_rows, by_page, by_units;  // units: of four elements, to a head
};

__device__ __forceinline__ void put(float *at, float a, float b) { at[0] = a, at[1] = b; }
__device__ __forceinline__ void put(__nv_bfloat16 *at, float a, float b) {
  at[0] = __float2bfloat16_rn(a), at[1] = __float2bfloat16_rn(b);
}
__device__ __forceinline__ void put(__half *at, float a, float b) {
  at[0] = __float2half_rn(a), at[1] = __float2half_rn(b);
}

__device__ __forceinline__ void put4(float *at, float4 x) { *reinterpret_cast<float4 *>(at) = x; }
__device__ __forceinline__ void put4(__nv_bfloat16 *at, float4 x) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(x.z, x.w);
  *reinterpret_cast<uint2 *>(at) =
      make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}
__device__ __forceinline__ void put4(__half *at, float4 x) {
  const __half2 lo = __floats2half2_rn(x.x, x.y), hi = __floats2half2_rn(x.z, x.w);
  *reinterpret_cast<uint2 *>(at) =
      make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}

// head_dim a multiple of four and everything aligned to four elements: a CTA, or a few with few rows, to a row; each thread
// has kStoreUnits units of four elements on their way at once (by the kernel for any alignment below, a thread per pair of
// elements, 2048 rows of 32/8 heads of 128 in bf16 take 57 us instead of 22, 514 rows 33 instead of 8.6).
// What bounds it: memory, with two waves of CTAs, 2048 rows 22 us, 4.3 TB/s; with few rows the chain starts, page and rotation,
// store (one row 1.7 us).
constexpr int kStoreThreads = 256, kStoreUnits = 6;
template <typename T>
__global__ void __launch_bounds__(kStoreThreads) paged_store4_kernel(const StoreArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x;
  int r = row;
  const int b = divide(r, a.by_rows);
  const Request request = request_of(a.starts, a.counts, b, a.rows, a.positions);
  if (request.bad && r == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    kc_raise(KC_ERR_BAD_ARGS);
  if (r >= request.count)
    return;
  const int position = request.start + r;
  int within = position;
  const int at = divide(within, a.by_page), page = a.table[(size_t)b * a.max_pages + at];
  const float *table = a.rope + (size_t)position * 2 * a.hd;
  const int units = a.per_row / 2, heads = a.n_heads + a.n_kv;
  for (int u0 = blockIdx.y * kStoreThreads + threadIdx.x; u0 < units; u0 += gridDim.y * kStoreThreads * kStoreUnits) {
    float4 x[kStoreUnits], c[kStoreUnits], s[kStoreUnits];
    int head[kStoreUnits], j[kStoreUnits];
#pragma unroll
    for (int i = 0; i < kStoreUnits; i++) {
      const int u = u0 + i * gridDim.y * kStoreThreads;
      if (u >= units)
        break;
      j[i] = u;
      head[i] = divide(j[i], a.by_units);
      j[i] *= 4;
      const float *src = head[i] < a.n_heads ? a.q + row * a.q_ld + (size_t)head[i] * a.hd
                         : head[i] < heads   ? a.k + row * a.kv_ld + (size_t)(head[i] - a.n_heads) * a.hd
                                             : a.v + row * a.kv_ld + (size_t)(head[i] - heads) * a.hd;
      x[i] = *reinterpret_cast<const float4 *>(src + j[i]);
      if (head[i] < heads) {
        c[i] = *reinterpret_cast<const float4 *>(table + j[i]);
        s[i] = *reinterpret_cast<const float4 *>(table + a.hd + j[i]);
      }
    }
    if (page < 0 || page >= a.pages) {
      if (threadIdx.x == 0)
        kc_raise(KC_ERR_BAD_ARGS);
      return;
    }
    const size_t place = (size_t)page * a.page_stride + (size_t)within * a.hd;
#pragma unroll
    for (int i = 0; i < kStoreUnits; i++) {
      if (u0 + i * gridDim.y * kStoreThreads >= units)
        break;
      float4 y = x[i];
      if (head[i] < heads) {  // (a, b) to (a cos - b sin, a sin + b cos), each product rounded
        y.x = __fsub_rn(__fmul_rn(x[i].x, c[i].x), __fmul_rn(x[i].y, s[i].y));
        y.y = __fadd_rn(__fmul_rn(x[i].x, s[i].y), __fmul_rn(x[i].y, c[i].x));
        y.z = __fsub_rn(__fmul_rn(x[i].z, c[i].z), __fmul_rn(x[i].w, s[i].w));
        y.w = __fadd_rn(__fmul_rn(x[i].z, s[i].w), __fmul_rn(x[i].w, c[i].z));
      }
      if (head[i] < a.n_heads) {
        *reinterpret_cast<float4 *>(a.q_out + row * a.q_out_ld + (size_t)head[i] * a.hd + j[i]) = y;
      } else {
        const bool is_k = head[i] < heads;
        T *cache = static_cast<T *>(is_k ? a.key : a.value);
        put4(cache + place + (size_t)(head[i] - (is_k ? a.n_heads : heads)) * a.page_size * a.hd + j[i], y);
      }
    }
  }
}

// A thread per pair of a row's queries, keys or values: any even head_dim and any alignment.
template <typename T>
__global__ void __launch_bounds__(256) paged_store_kernel(const StoreArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long row = id / a.per_row;
  if (row >= (long long)a.batch * a.rows)
    return;
  int pair = (int)(id - row * a.per_row);
  const int b = (int)(row / a.rows), r = (int)(row - (long long)b * a.rows);
  const Request request = request_of(a.starts, a.counts, b, a.rows, a.positions);
  if (request.bad && r == 0 && pair == 0)
    kc_raise(KC_ERR_BAD_ARGS);
  if (r >= request.count)
    return;
  const int position = request.start + r, at = position / a.page_size;
  const int page = a.table[(size_t)b * a.max_pages + at];
  if (page < 0 || page >= a.pages) {
    if (pair == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    return;
  }
  const int half = a.hd / 2, head = pair / half, j = 2 * (pair - head * half);
  const float *table = a.rope + (size_t)position * 2 * a.hd;
  const size_t place = (size_t)page * a.page_stride + (size_t)(position - at * a.page_size) * a.hd + j;
  const size_t head_stride = (size_t)a.page_size * a.hd;
  if (head < a.n_heads + a.n_kv) {
    const bool is_k = head >= a.n_heads;
    const int h = is_k ? head - a.n_heads : head;
    const float *src = (is_k ? a.k + row * a.kv_ld : a.q + row * a.q_ld) + (size_t)h * a.hd + j;
    const float c = table[j], s = table[a.hd + j + 1], x = src[0], y = src[1];
    const float o0 = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)), o1 = __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c));
    if (is_k)
      put(static_cast<T *>(a.key) + place + h * head_stride, o0, o1);
    else
      put(a.q_out + row * a.q_out_ld + (size_t)h * a.hd + j, o0, o1);
  } else {
    const int h = head - a.n_heads - a.n_kv;
    const float *src = a.v + row * a.kv_ld + (size_t)h * a.hd + j;
    put(static_cast<T *>(a.value) + place + h * head_stride, src[0], src[1]);
  }
}

// ---- attention ----------------------------------------------------------------------------------------------------

// The kernel on the CUDA cores: any type, head_dim up to 256, any alignment. LANES lanes take a position, 16 of its
// elements each, so that a score costs log2(LANES) shuffles for 16 LANES products, and its weight meets the values in the
// same lanes without another; four query vectors in registers share each key and value (eight with eight elements to a lane,
// half the passes over the keys and values, took longer: 24 requests of 28/4 heads of 96 up to 3001 positions 108 us back to
// back against 75). Every warp has a ring of its own in shared memory, which each lane fills for itself, asynchronously, and reads itself:
// no barrier until the end of a piece. What bounds it: its instructions, three warps to a scheduler that issue one every
// 2.8 cycles (32/8 heads of 96 in bf16, 24 requests: 82 us, 1.7 TB/s; 28/4 heads of 96 76 us).
constexpr int kVecs = 4, kElems = 16, kPairs = kElems / 2;
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kTile = 64;       // positions
constexpr int kCtas = 148 * 3;  // the shares; a function of nothing else, so that the workspace's size is known
constexpr int kStages = 4;

// A pair of elements in 32 bits each.
__device__ __forceinline__ uint64_t pair_of(uint32_t x, __nv_bfloat16) { return f2_pack_bits(x << 16, x & 0xffff0000u); }
__device__ __forceinline__ uint64_t pair_of(uint32_t x, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x));
  return f2_pack(f.x, f.y);
}
__device__ __forceinline__ float one_of(float x) { return x; }
__device__ __forceinline__ float one_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float one_of(__half x) { return __half2float(x); }

// 16 bytes from global to shared memory, asynchronously; zeros without `in`.
__device__ __forceinline__ void copy16(void *dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// This lane's kElems elements of a row: wide, 16-byte units LANES apart; else elements LANES apart.
template <typename T, int LANES, bool WIDE>
struct Row {
  static constexpr int kUnit = 16 / sizeof(T);
  static constexpr int kUnits = kElems / kUnit;
  uint4 raw[WIDE ? kUnits : 1];
  T one[WIDE ? 1 : kElems];

  // The element behind index i of the lane's.
  static __device__ __forceinline__ int element(int lane, int i) {
    return WIDE ? (lane + LANES * (i / kUnit)) * kUnit + i % kUnit : lane + LANES * i;
  }
  // Starts this lane's copies to a slot of kUnits times 32 units, and reads them back.
  static __device__ __forceinline__ void copy(uint4 *slot, const T *row, bool in, int hd, int sub, int lane) {
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
      const int at = (sub + LANES * u) * kUnit;
      copy16(slot + 32 * u + lane, row + (at < hd ? at : 0), in && at < hd);
    }
  }
  __device__ __forceinline__ void take(const uint4 *slot, int lane) {
#pragma unroll
    for (int u = 0; u < kUnits; u++)
      raw[u] = slot[32 * u + lane];
  }
  __device__ __forceinline__ void load(const T *row, bool in, int hd, int lane) {
#pragma unroll
    for (int i = 0; i < kElems; i++)
      one[i] = in && lane + LANES * i < hd ? row[lane + LANES * i] : T(0.0f);
  }
  __device__ __forceinline__ uint64_t pair(int i) const {  // elements 2 i, 2 i + 1
    if (!WIDE)
      return f2_pack(one_of(one[2 * i]), one_of(one[2 * i + 1]));
    if constexpr (sizeof(T) == 4) {
      const uint4 x = raw[i / 2];
      return i % 2 ? f2_pack_bits(x.z, x.w) : f2_pack_bits(x.x, x.y);
    } else {
      const uint4 x = raw[i / 4];
      return pair_of(i % 4 == 0 ? x.x : i % 4 == 1 ? x.y : i % 4 == 2 ? x.z : x.w, T(0.0f));
    }
  }
};

// Shared memory: the warps' rings (nothing where they are not used), and over them their results at the end of a piece.
template <typename T, int LANES, bool WIDE>
struct RowsSmem {
  using R = Row<T, LANES, WIDE>;
  static constexpr int slot = 32 * R::kUnits;                            // units of a key or a value
  static constexpr int ring = WIDE ? kStages * 2 * slot * 16 : 0;        // bytes to a warp
  static constexpr int sums = kVecs * LANES * kElems * (int)sizeof(float);  // of a warp
  static constexpr int total = kWarps * (ring > sums ? ring : sums);
};

template <typename T, int LANES, bool WIDE>
__global__ void __launch_bounds__(kThreads, 3) paged_rows_kernel(const PagedArgs a) {
  using S = RowsSmem<T, LANES, WIDE>;
  using R = typename S::R;
  constexpr int kAt = 32 / LANES, kStep = kWarps * kAt;  // positions of a warp, of all warps at a time
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ RangeRoom room;
  __shared__ float wm[kWarps][kVecs], wl[kWarps][kVecs], m_all[kVecs], l_all[kVecs];
  __shared__ int bad, last;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, sub = lane % LANES, at = lane / LANES;
  uint4 *const ring = reinterpret_cast<uint4 *>(smem + warp * S::ring);
  if (t == 0)
    bad = 0;
  __syncthreads();  // any warp may set it in its first fetch, and find_range need not hold a barrier
  pdl_wait();
  pdl_launch_dependents();
  Range range;
  if (!find_range(a, kTile, &range, &room))
    return;
  const int hd = a.hd;
  const float scale = rsqrtf((float)hd) * kLog2e;
  Walk walk(&range);
  Piece p;
  while (walk.next(a, &range, kTile, &p)) {
    const int end = min(p.t1 * kTile, p.start + p.count), first = p.t0 * kTile + warp * kAt + at;
    const int steps = (end - p.t0 * kTile + kStep - 1) / kStep;
    const float guard = guard_of(p.start + p.count);
    const int *pages = a.table + (size_t)p.b * a.max_pages;
    const size_t head = (size_t)p.head * a.page_size * hd;
    // Step i's page (-2: no position of the piece; a page below 0 is -1), and where its row lies.
    auto page_of = [&](int i) {
      int position = first + i * kStep;
      return position < end ? max(pages[divide(position, a.by_page)], -1) : -2;
    };
    auto row_of = [&](int i, int page, bool *in) {
      int within = first + i * kStep;
      *in = page >= 0 && page < a.pages;
      if (!*in && page != -2)
        bad = 1;
      divide(within, a.by_page);
      return *in ? (size_t)page * a.page_stride + head + (size_t)within * hd : 0;
    };
    auto fetch = [&](int i, int page) {
      bool in;
      const size_t place = row_of(i, page, &in);
      uint4 *slot = ring + (i % kStages) * 2 * S::slot;
      R::copy(slot, static_cast<const T *>(a.key) + place, in, hd, sub, lane);
      R::copy(slot + S::slot, static_cast<const T *>(a.value) + place, in, hd, sub, lane);
    };
    int page = page_of(0);  // of the step fetched next
    if (WIDE) {
#pragma unroll
      for (int i = 0; i < kStages - 1; i++) {
        const int next = page_of(i + 1);
        fetch(i, page);
        asm volatile("cp.async.commit_group;" ::: "memory");
        page = next;
      }
    }
    uint64_t q[kVecs][kPairs], acc[kVecs][kPairs];
    float m[kVecs], l[kVecs];
    int limit[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; v++) {
      int row = 0;
      const size_t vec = v < p.vecs ? vector_at(a, p, v, &row) : 0;
      limit[v] = v < p.vecs ? p.start + row + 1 : 0;
      m[v] = -INFINITY, l[v] = 0.0f;
#pragma unroll
      for (int i = 0; i < kPairs; i++) {
        const int e0 = R::element(sub, 2 * i), e1 = R::element(sub, 2 * i + 1);
        const float x = v < p.vecs && e0 < hd ? a.q[vec * hd + e0] * scale : 0.0f;
        const float y = v < p.vecs && e1 < hd ? a.q[vec * hd + e1] * scale : 0.0f;
        q[v][i] = f2_pack(x, y), acc[v][i] = 0;
      }
    }
    for (int i = 0; i < steps; i++) {
      const int position = first + i * kStep;
      R k, x;
      if (WIDE) {
        const int next = page_of(i + kStages);
        fetch(i + kStages - 1, page);
        asm volatile("cp.async.commit_group;" ::: "memory");
        page = next;
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        const uint4 *slot = ring + (i % kStages) * 2 * S::slot;
        k.take(slot, lane);
        x.take(slot + S::slot, lane);
      } else {
        bool in;
        const size_t place = row_of(i, page, &in);
        page = page_of(i + 1);
        k.load(static_cast<const T *>(a.key) + place, in, hd, sub);
        x.load(static_cast<const T *>(a.value) + place, in, hd, sub);
      }
      float s[kVecs];
      uint64_t part[kVecs];
#pragma unroll
      for (int v = 0; v < kVecs; v++)
        part[v] = 0;
#pragma unroll
      for (int j = 0; j < kPairs; j++) {
        const uint64_t kj = k.pair(j);
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          part[v] = f2_fma(q[v][j], kj, part[v]);
      }
      bool rises = false;
#pragma unroll
      for (int v = 0; v < kVecs; v++) {
        float lo, hi;
        f2_unpack(part[v], lo, hi);
        s[v] = lo + hi;
      }
#pragma unroll
      for (int o = LANES / 2; o; o >>= 1)
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          s[v] += __shfl_xor_sync(0xffffffffu, s[v], o);
#pragma unroll
      for (int v = 0; v < kVecs; v++) {
        s[v] = position < min(limit[v], end) ? s[v] : -INFINITY;
        rises |= s[v] > m[v];
      }
      if (rises) {
#pragma unroll
        for (int v = 0; v < kVecs; v++) {
          if (!(s[v] > m[v]))
            continue;
          const float keep = ex2(m[v] - s[v]);  // 0 at the first
          m[v] = s[v];
          l[v] *= keep;
#pragma unroll
          for (int j = 0; j < kPairs; j++)
            acc[v][j] = f2_mul(acc[v][j], f2_pack(keep, keep));
        }
      }
#pragma unroll
      for (int v = 0; v < kVecs; v++) {
        s[v] = s[v] == -INFINITY ? 0.0f : ex2(s[v] - m[v]) * guard;
        l[v] += s[v];
      }
      if (position <= p.start) {  // every row sees it
#pragma unroll
        for (int j = 0; j < kPairs; j++) {
          const uint64_t xj = x.pair(j);
#pragma unroll
          for (int v = 0; v < kVecs; v++)
            acc[v][j] = f2_fma(f2_pack(s[v], s[v]), xj, acc[v][j]);
        }
      } else if (position < end) {
        // What a row does not see may be anything: its product is left out, not made with a weight of zero.
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          if (position < limit[v])
#pragma unroll
            for (int j = 0; j < kPairs; j++)
              acc[v][j] = f2_fma(f2_pack(s[v], s[v]), x.pair(j), acc[v][j]);
      }
    }
    if (WIDE)
      asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the rings' room is free
    // The lane groups' results, then the warps'.
    float *const sums = reinterpret_cast<float *>(smem);  // [warps][kVecs][LANES * kElems]
    constexpr int kLine = LANES * kElems;
#pragma unroll
    for (int v = 0; v < kVecs; v++) {
      float top = m[v];
#pragma unroll
      for (int o = 16; o >= LANES; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float f = m[v] == -INFINITY ? 0.0f : ex2(m[v] - top);
      float sum = l[v] * f;
#pragma unroll
      for (int o = 16; o >= LANES; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0)
        wm[warp][v] = top, wl[warp][v] = sum;
#pragma unroll
      for (int j = 0; j < kPairs; j++) {
        float lo, hi;
        f2_unpack(f2_mul(acc[v][j], f2_pack(f, f)), lo, hi);
#pragma unroll
        for (int o = 16; o >= LANES; o >>= 1)
          lo += __shfl_xor_sync(0xffffffffu, lo, o), hi += __shfl_xor_sync(0xffffffffu, hi, o);
        if (at == 0) {
          sums[(warp * kVecs + v) * kLine + R::element(sub, 2 * j)] = lo;
          sums[(warp * kVecs + v) * kLine + R::element(sub, 2 * j + 1)] = hi;
        }
      }
    }
    __syncthreads();
    if (t < kVecs) {
      float top = -INFINITY, sum = 0.0f;
      for (int w = 0; w < kWarps; w++)
        top = fmaxf(top, wm[w][t]);
      for (int w = 0; w < kWarps; w++) {
        const float f = wm[w][t] == -INFINITY ? 0.0f : ex2(wm[w][t] - top);
        sum += wl[w][t] * f;
        wl[w][t] = f;
      }
      m_all[t] = top, l_all[t] = sum;
    }
    __syncthreads();
    // Joined in place: [vecs][hd] over the first warps' results, each thread's numbers read before any is written.
    constexpr int kEach = kVecs * kLine / kThreads;
    float y[kEach];
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      const int i = t + j * kThreads, v = i / kLine;
      y[j] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++)
        y[j] = fmaf(wl[w][v], sums[w * kVecs * kLine + i], y[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      const int i = t + j * kThreads, v = i / kLine, e = i % kLine;
      if (e < hd && v < p.vecs)
        sums[v * hd + e] = y[j];
    }
    __syncthreads();
    finish<kThreads, 0, 0>(a, &range, p, m_all, l_all, sums, &bad, &last, t);
    if (t == 0)
      bad = 0;
    __syncthreads();
  }
}

bool heads_ok(int n_heads, int n_kv, int hd, int batch, int rows) {
  constexpr long long most = 1 << 24;  // vectors; the product of two of the numbers does not wrap
  return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && hd > 0 && hd <= kMaxHd && batch > 0 && rows > 0 &&
         (long long)batch * rows <= most && (long long)batch * rows * n_heads <= most;
}

template <typename T>
cudaError_t launch_store(const StoreArgs &a) {
  const uintptr_t wide = (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.rope |
                         (a.q_ld | a.q_out_ld | a.kv_ld | a.hd) * sizeof(float);
  const uintptr_t cache = (uintptr_t)a.key | (uintptr_t)a.value | a.page_stride * sizeof(T);
  const long long rows = (long long)a.batch * a.rows;
  if (wide % 16 == 0 && cache % (4 * sizeof(T)) == 0) {
    // About two CTAs to an SM with few rows (one row of 32/8 heads of 64: three CTAs).
    const long long most = (a.per_row / 2 + kStoreThreads - 1) / kStoreThreads, want = 2 * kc_device_sms() / rows;
    const long long parts = want < 1 ? 1 : want < most ? want : most;
    return kc_launch_pdl(paged_store4_kernel<T>, dim3((unsigned)rows, (unsigned)parts), dim3(kStoreThreads), 0, kc_stream(),
                         a);
  }
  return kc_launch_pdl(paged_store_kernel<T>, dim3((unsigned)((rows * a.per_row + 255) / 256)), dim3(256), 0, kc_stream(), a);
}

const char *cache_fault(const PagedCache *c, int n_kv, int hd) {
  if (!c || !c->key || !c->value || !c->table)
    return "missing keys, values or page table";
  if (c->type != K_F32 && c->type != K_BF16 && c->type != K_F16)
    return "invalid cache type";
  if (c->pages <= 0 || c->page_size <= 0 || c->max_pages <= 0 ||
      (long long)c->max_pages * c->page_size > kMaxPositions)
    return "invalid pages";
  if (c->page_stride / hd / n_kv < (size_t)c->page_size || c->page_stride > ((size_t)1 << 62) / c->pages)
    return "invalid page stride";
  return nullptr;
}

template <typename T, int LANES, bool WIDE>
cudaError_t launch_rows(const PagedArgs &a) {
  const auto kernel = paged_rows_kernel<T, LANES, WIDE>;
  constexpr int smem = RowsSmem<T, LANES, WIDE>::total;
  const cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(kernel), smem);
  return e != cudaSuccess ? e : kc_launch_pdl(kernel, dim3(kCtas), dim3(kThreads), smem, kc_stream(), a);
}
template <typename T, bool WIDE>
cudaError_t launch_rows_of(const PagedArgs &a) {
  return a.hd <= 64    ? launch_rows<T, 4, WIDE>(a)
         : a.hd <= 128 ? launch_rows<T, 8, WIDE>(a)
                       : launch_rows<T, 16, WIDE>(a);
}
template <typename T>
cudaError_t launch_rows_of(const PagedArgs &a) {
  const bool wide = a.hd * sizeof(T) % 16 == 0 && a.page_stride * sizeof(T) % 16 == 0 &&
                    !(((uintptr_t)a.key | (uintptr_t)a.value) & 15);
  return wide ? launch_rows_of<T, true>(a) : launch_rows_of<T, false>(a);
}

int blocks_of(int n_heads, int n_kv, int rows, int block) {
  return (int)(((long long)rows * (n_heads / n_kv) + block - 1) / block);
}

// Tickets first, to a whole number of 16 bytes, then the slots. A ticket for every query vector: enough for the segments
// of any batch of as many rows, whatever its KV heads.
size_t ticket_bytes(int n_heads, int batch, int rows) {
  return ((size_t)batch * rows * n_heads * sizeof(unsigned) + 15) & ~(size_t)15;
}

// The slots of whichever kernel has more.
size_t slots_floats(int hd) {
  const int rows = 2 * kCtas * slot_size(kVecs, hd), tc = kc_paged_tc_slots_floats(hd);
  return rows > tc ? rows : tc;
}

}  // namespace

extern "C" {

void k_rope_kv_store_paged(float *q_out, size_t q_out_ld, const float *q, size_t q_ld, const float *k, const float *v,
                           size_t kv_ld, const PagedCache *cache, const float *rope, int seq_len, const int *starts,
                           const int *counts, int n_heads, int n_kv_heads, int head_dim, int batch, int rows) {
  const char *name = "k_rope_kv_store_paged";
  if (batch == 0 || rows == 0)
    return;
  constexpr long long most = 0x7fffffff;
  if (n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || head_dim % 2 || batch < 0 || rows < 0 || seq_len <= 0 ||
      (long long)batch * rows > most || ((long long)n_heads + 2 * (long long)n_kv_heads) * head_dim > most ||
      q_ld < (size_t)n_heads * head_dim || q_out_ld < (size_t)n_heads * head_dim ||
      kv_ld < (size_t)n_kv_heads * head_dim) {
    kc_fail("%s: invalid shape heads=%d/%d head_dim=%d batch=%d rows=%d seq_len=%d strides %zu, %zu, %zu", name, n_heads,
            n_kv_heads, head_dim, batch, rows, seq_len, q_out_ld, q_ld, kv_ld);
    return;
  }
  if (!q_out || !q || !k || !v || !rope || !starts) {
    kc_fail("%s: missing queries, keys, values, rotation table or starts", name);
    return;
  }
  if (const char *fault = cache_fault(cache, n_kv_heads, head_dim)) {
    kc_fail("%s: %s", name, fault);
    return;
  }
  if (q_out == q && q_out_ld != q_ld) {
    kc_fail("%s: queries rotated in place need one row stride, not %zu and %zu", name, q_out_ld, q_ld);
    return;
  }
  StoreArgs a;
  memset(&a, 0, sizeof(a));
  a.q_out = q_out, a.q = q, a.k = k, a.v = v, a.rope = rope, a.key = cache->key, a.value = cache->value;
  a.table = cache->table, a.starts = starts, a.counts = counts;
  a.q_out_ld = (long long)q_out_ld, a.q_ld = (long long)q_ld, a.kv_ld = (long long)kv_ld;
  a.page_stride = cache->page_stride, a.pages = cache->pages, a.page_size = cache->page_size;
  a.max_pages = cache->max_pages, a.n_heads = n_heads, a.n_kv = n_kv_heads, a.hd = head_dim;
  const int held = cache->max_pages * cache->page_size;
  a.positions = held < seq_len ? held : seq_len;
  a.batch = batch, a.rows = rows, a.per_row = (n_heads + 2 * n_kv_heads) * (head_dim / 2);
  const long long ctas = ((long long)batch * rows * a.per_row + 255) / 256;
  if (ctas > most) {
    kc_fail("%s: %d requests of %d rows are too many for one call", name, batch, rows);
    return;
  }
  a.by_rows = divisor(rows), a.by_page = divisor(a.page_size), a.by_units = divisor(head_dim < 4 ? 1 : head_dim / 4);
  const cudaError_t e = cache->type == K_F32    ? launch_store<float>(a)
                        : cache->type == K_BF16 ? launch_store<__nv_bfloat16>(a)
                                                : launch_store<__half>(a);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

size_t k_attention_paged_bytes(int n_heads, int n_kv_heads, int head_dim, int batch, int rows) {
  if (!heads_ok(n_heads, n_kv_heads, head_dim, batch, rows))
    return 0;
  return ticket_bytes(n_heads, batch, rows) + sizeof(float) * slots_floats(head_dim);
}

void k_attention_paged_init(AttentionWork *work, int n_heads, int n_kv_heads, int head_dim, int batch, int rows,
                            void *memory) {
  const char *name = "k_attention_paged_init";
  const size_t bytes = k_attention_paged_bytes(n_heads, n_kv_heads, head_dim, batch, rows);
  memset(work, 0, sizeof(*work));
  if (!bytes) {
    kc_fail("%s: invalid shape", name);
    return;
  }
  if ((uintptr_t)memory & 15) {
    kc_fail("%s: the memory must be 16-byte aligned", name);
    return;
  }
  void *base = memory;
  if (!base && cudaMalloc(&base, bytes) != cudaSuccess) {
    cudaGetLastError();
    kc_fail("%s: cannot allocate %zu bytes of attention work", name, bytes);
    return;
  }
  const cudaError_t e = cudaMemsetAsync(base, 0, ticket_bytes(n_heads, batch, rows), kc_stream());
  if (e != cudaSuccess) {
    cudaGetLastError();
    if (!memory)
      cudaFree(base);
    kc_fail("%s: %s", name, cudaGetErrorString(e));
    return;
  }
  work->partial = static_cast<float *>(base);
  work->max_chunks = -1;
  work->n_heads = n_heads;
  work->head_dim = head_dim;
  work->workers = batch * rows;
  work->external = memory != nullptr;
  work->capacity = bytes / sizeof(float);
}

void k_attention_paged_rows(float *out, int8_t *oq, float *os, const float *q, const PagedCache *cache, const int *starts,
                            const int *counts, AttentionWork *work, int n_heads, int n_kv_heads, int head_dim, int batch,
                            int rows, int gs) {
  const char *name = "k_attention_paged_rows";
  if (batch == 0 || rows == 0)
    return;
  if (!heads_ok(n_heads, n_kv_heads, head_dim, batch, rows)) {
    kc_fail("%s: invalid shape heads=%d/%d head_dim=%d batch=%d rows=%d", name, n_heads, n_kv_heads, head_dim, batch, rows);
    return;
  }
  if (!out || !q || !starts || (oq && !os)) {
    kc_fail("%s: missing output, queries or starts", name);
    return;
  }
  if (const char *fault = cache_fault(cache, n_kv_heads, head_dim)) {
    kc_fail("%s: %s", name, fault);
    return;
  }
  if (oq && (gs <= 0 || head_dim % gs)) {
    kc_fail("%s: group size %d does not divide the head's %d outputs", name, gs, head_dim);
    return;
  }
  if (!work || !work->partial || work->max_chunks != -1 || work->n_heads != n_heads || work->head_dim != head_dim ||
      (long long)batch * rows > work->workers ||
      k_attention_paged_bytes(n_heads, n_kv_heads, head_dim, batch, rows) > work->capacity * sizeof(float)) {
    kc_fail("%s: the attention work is missing or too small for this shape", name);
    return;
  }
  PagedArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q, a.key = cache->key, a.value = cache->value, a.table = cache->table, a.starts = starts, a.counts = counts;
  a.out = out, a.oq = oq, a.os = os;
  a.page_stride = cache->page_stride, a.pages = cache->pages, a.max_pages = cache->max_pages;
  a.page_size = cache->page_size, a.positions = cache->max_pages * cache->page_size;
  a.n_heads = n_heads, a.n_kv = n_kv_heads, a.group = n_heads / n_kv_heads, a.hd = head_dim;
  a.batch = batch, a.rows = rows, a.gs = gs;
  const bool tc = kc_paged_tc_ok(a, cache->type), f32 = kc_paged_f32_ok(a, cache->type);
  a.block = tc ? kc_paged_tc_block(a.group, rows) : f32 ? kPagedF32Block : kVecs;
  a.blocks = blocks_of(n_heads, n_kv_heads, rows, a.block);
  a.slot_floats = slot_size(a.block, head_dim);
  a.by_page = divisor(a.page_size), a.by_group = divisor(a.group);
  a.tickets = reinterpret_cast<unsigned *>(work->partial);
  // The tickets' room is the work's own, so that it does not move between calls of different batches.
  a.partial = work->partial + (work->capacity - slots_floats(head_dim));
  const cudaError_t e = tc                      ? kc_launch_paged_tc(a, cache->type)
                        : f32                   ? kc_launch_paged_f32(a)
                        : cache->type == K_F32  ? launch_rows_of<float>(a)
                        : cache->type == K_BF16 ? launch_rows_of<__nv_bfloat16>(a)
                                                : launch_rows_of<__half>(a);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
