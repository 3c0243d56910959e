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
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "divide.cuh"
#include "kernels_cuda_internal.h"
#include "tcgen05.cuh"

namespace {

constexpr int kMaxHd = 256;
constexpr int kPlanSms = 148;      // the plan is a function of the shape alone, so that the workspace's size is too
constexpr int kMaxSplits = 64;     // of the prefix, or of a request's own positions

constexpr float kLog2e = 1.44269504088896341f;

constexpr int kGenericThreads = 256, kGenericWarps = kGenericThreads / 32;
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
  // The items' turns: CTAs below `heavy` have per_cta + 1 of the prefix's, the others per_cta and `extra` before the rest.
  int per_cta, heavy, extra;
  Divisor by_prefix_splits, by_own_splits, by_kv, by_own_tiles, by_group, by_rows;
};

// Rows that request b uses and the positions it has stored before them; 0 rows where they are not sound. Both loads go
// out at once.
struct Request {
  int count, start;
  bool bad;
};
__device__ __forceinline__ Request request_of(const SharedArgs &a, int b) {
  const int count = a.counts ? a.counts[b] : a.rows, start = a.starts[b];
  const bool ok = count > 0 && count <= a.rows && start >= 0 && start <= a.seq - count;
  return Request{ok ? count : 0, start, !ok && count != 0};
}

// One work item: up to a tile of query vectors of one KV head against a range of one cache's positions.
struct Item {
  const float *k, *v;  // the KV head's rows
  int kv, split;       // split: index of the partial result
  int b;               // the request, or -1: the prefix
  int start;           // the request's positions before its rows
  int first, vecs;     // tile vectors: the flat (b, r, group member) index of the first, and how many
  int p0, p1;          // positions
};

// The items of CTA `cta` of `ctas`: the prefix's in turn, so that some CTAs get one more of them than the others; of the
// requests' own, `extra` to each of the others, then the rest in turn, the others first. -1 past the last.
__host__ __device__ __forceinline__ int item_id(const SharedArgs &a, int cta, int ctas, int n) {
  const int prefix = a.n_kv * a.tiles * a.prefix_splits, own = a.n_kv * a.batch * a.own_tiles * a.own_splits;
  const int heavy = a.heavy, light = ctas - heavy, mine = a.per_cta + (cta < heavy);
  if (n < mine)
    return cta + n * ctas;
  n -= mine;
  int id;
  if (cta >= heavy && n < a.extra) {
    id = cta - heavy + n * light;
  } else {
    n -= cta >= heavy ? a.extra : 0;
    const long long rest = (long long)(cta >= heavy ? cta - heavy : cta + light) + (long long)n * ctas;
    if (rest >= own - a.extra * light)
      return -1;
    id = a.extra * light + (int)rest;
  }
  return prefix + id;
}

// Vector i of KV head kv's flat list: index in the [batch][rows][n_heads] order.
__device__ __forceinline__ int vector_at(const SharedArgs &a, int kv, int i) {
  const int row = divide(i, a.by_group);
  return row * a.n_heads + kv * a.group + i;
}

// Index of the tile's vector i, -1 for one that is not in use.
__device__ __forceinline__ int vector_of(const SharedArgs &a, int first, int vecs, int kv, int i) {
  int member = first + min(i, vecs - 1);
  int row = divide(member, a.by_group);
  const int vec = row * a.n_heads + kv * a.group + member;
  const int b = divide(row, a.by_rows);
  return i < vecs && row < request_of(a, b).count ? vec : -1;
}

// The positions of one of the splits of `length`, which differ by one at most.
__device__ __forceinline__ void split_range(int length, int split, const Divisor &by_splits, Item *it) {
  int longer = length;
  const int each = divide(longer, by_splits);
  it->p0 = each * split + min(split, longer);
  it->p1 = it->p0 + each + (split < longer);
}

// Items 0 .. n_kv * tiles * prefix_splits - 1 are the prefix's, then one per (request, KV head, query tile, split).
// False: nothing to do; with `report`, a request that is not sound is an error.
__device__ __forceinline__ bool item_at(const SharedArgs &a, int id, int tile, bool report, Item *it) {
  const int prefix_items = a.n_kv * a.tiles * a.prefix_splits;
  if (id < prefix_items) {
    int kv = divide(id, a.by_prefix_splits);
    it->split = id;
    it->first = divide(kv, a.by_kv) * tile;
    it->kv = kv;
    it->b = -1;
    it->vecs = min(tile, a.batch * a.rows * a.group - it->first);
    it->k = a.pk + (size_t)it->kv * a.prefix_seq * a.hd;
    it->v = a.pv + (size_t)it->kv * a.prefix_seq * a.hd;
    split_range(a.prefix, id, a.by_prefix_splits, it);
    return true;
  }
  id -= prefix_items;
  int own_tile = divide(id, a.by_own_splits);
  const int split = id;
  it->split = a.prefix_splits + split;
  int kv = divide(own_tile, a.by_own_tiles);
  own_tile *= tile;
  it->b = divide(kv, a.by_kv);
  it->kv = kv;
  const Request r = request_of(a, it->b);
  if (!r.count) {
    if (r.bad && report)
      kc_raise(KC_ERR_BAD_ARGS);
    return false;
  }
  it->first = it->b * a.rows * a.group + own_tile;
  it->vecs = min(tile, r.count * a.group - own_tile);
  if (it->vecs <= 0)
    return false;
  const size_t head = ((size_t)it->b * a.n_kv + it->kv) * a.seq * a.hd;
  it->k = a.k + head;
  it->v = a.v + head;
  it->start = r.start;
  split_range(r.start + r.count, split, a.by_own_splits, it);
  return true;
}

// Positions of the item that its vector i (a flat index) sees: [p0, limit).
__device__ __forceinline__ int limit_of(const SharedArgs &a, const Item &it, int i) {
  if (it.b < 0)
    return it.p1;
  i -= it.b * a.rows * a.group;
  return min(it.p1, it.start + divide(i, a.by_group) + 1);
}

// Any head_dim up to 256 and any alignment, in fp32 FMAs: a warp takes a vector at a time, its lanes the 32 positions of
// a tile for the scores and the head's elements for the sums. The shared-memory reads, two to an FMA, bound it, so the
// positions are split finely (8 rows of 16 heads of 256 behind 2048 positions: 69 us; of 32 heads of 128 the tensor-core
// kernel takes 18).
__global__ void __launch_bounds__(kGenericThreads) shared_generic_kernel(const SharedArgs a) {
  extern __shared__ float smem[];
  pdl_wait();
  pdl_launch_dependents();
  Item it;
  if (!item_at(a, blockIdx.x, kGenericVecs, threadIdx.x == 0, &it))
    return;
  const int hd = a.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *ks = smem;                                 // [32][hd + 1]
  float *vs = ks + kGenericPos * (hd + 1);          // [32][hd]
  float *qs = vs + kGenericPos * hd;                // [8 warps][hd]
  const float scale = rsqrtf((float)hd) * kLog2e;
  const bool wide = hd % 4 == 0 && (((uintptr_t)it.k | (uintptr_t)it.v) & 15) == 0;
  for (int v0 = 0; v0 < it.vecs; v0 += kGenericWarps) {
    // One vector a warp at a time; the tiles come again from the cache for the next eight.
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
#pragma unroll
      for (int r = 0; r < kGenericPos / kGenericWarps; r++) {
        const int p = warp + r * kGenericWarps;
        if (p >= n)
          break;
        const float *kr = it.k + (size_t)(t0 + p) * hd, *vr = it.v + (size_t)(t0 + p) * hd;
        float *kd = ks + p * (hd + 1), *vd = vs + p * hd;
        if (wide) {
          for (int c = 4 * lane; c < hd; c += 128) {
            const float4 x = *reinterpret_cast<const float4 *>(kr + c);
            *reinterpret_cast<float4 *>(vd + c) = *reinterpret_cast<const float4 *>(vr + c);
            kd[c] = x.x, kd[c + 1] = x.y, kd[c + 2] = x.z, kd[c + 3] = x.w;
          }
        } else {
          for (int c = lane; c < hd; c += 32)
            kd[c] = kr[c], vd[c] = vr[c];
        }
      }
      __syncthreads();
      const bool seen = t0 + lane < limit;
      float s = 0.0f;
      if (seen) {
        const float *qw = qs + warp * hd, *kl = ks + lane * (hd + 1);
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        int e = 0;
#pragma unroll 4
        for (; e + 4 <= hd; e += 4)
#pragma unroll
          for (int j = 0; j < 4; j++)
            part[j] = fmaf(qw[e + j], kl[e + j], part[j]);
        for (; e < hd; e++)
          part[0] = fmaf(qw[e], kl[e], part[0]);
        s = (part[0] + part[1]) + (part[2] + part[3]);
      }
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

// head_dim <= 128 in whole 16-byte units. A CTA per SM takes its items one after another: up to 128 query vectors of a KV
// head against a range of positions in tiles of 64, S = Q K^T and P V on tcgen05 with accumulators in TMEM. The
// tiles of all items run through the same stages: the next item's keys and values are under way, and its queries laid
// out, before the last sums are done (a CTA per item took 8 % longer at 256 rows behind 8192 positions).
// What bounds it: two chains of dependent steps, 4.3 thousand clocks a tile of 64 positions and 128 vectors together. A
// group of softmax warps takes 7 thousand for its tile of two (1.2 for the maximum, 2.2 for the probabilities, 1.2 until
// the product is done, 1.3 to add it, 1.0 until the next scores), the converter warps 3.1 for a tile, the MMAs 1.8. 256
// rows of 32 heads of 128 behind 8192 positions: 213 us with 12 in the join, 103 TFLOP/s of fp32 products (310 of fp16),
// the tensor pipe 30 % busy, the shared-memory pipe 37 %, the issue slots 44 %; for more warps there are no registers.
//
// fp32 products on half-precision tensor cores: x = 2^-k (hi + lo) with hi and lo fp16, 22 bits of x, and
// x y = 2^-(k + k') (hi hi' + hi lo' + lo hi') up to 2^-22 of the product (what is dropped, lo lo', is below the
// rounding of lo). The two bits less than fp32's cost less than the roundings of a chain of fp32 sums (0.9 to 1.0e-6 off
// 64 bits at the sizes below, such chains 1.1 to 1.8e-6); a third part would double the MMAs, and its operands do not fit
// into two stages. The power 2^k puts the largest magnitude of one query, key or value vector just below 2^15, so no
// finite input overflows and an element 2^-17 of its vector's largest still keeps its 22 bits. k of a key goes into its
// scores' scale, k of a value into its probabilities (exact powers of two both). No power is shared between positions: a
// vector that a row does not see, or that has no weight in it, takes no bits of the others. For the same reason the
// probabilities' own power, one to a row and tile, follows the largest product of a seen probability and its value's
// power: what is added to a row's result is off by 2^-22 of itself, and by 2^-29 of the largest one of its tile at most.
//
// Warps: 0-3 the softmax of the even tiles and 4-7 that of the odd ones, a thread per query vector (TMEM lane), each
// group with a reference and a sum of its own (joined at the end), so that a group has two tiles' time; 8 issues
// the MMAs; 9-16 split eight keys and eight values of a tile each and store them as the MMAs' operands (keys K-major,
// values MN-major, so neither is transposed), two stages. The queries are the A operand in TMEM (from shared memory an
// MMA of 64 columns would wait for it), and the probabilities take the place of the scores they come from.
//
// The tensor cores' accumulators truncate, always towards zero. So P V of a tile is a product of its own (twelve MMAs,
// the small terms first: four cuts that count), which the tile's group adds to the item's sums in fp32, rounded to
// nearest, under the next tile's MMAs. Both lie in TMEM, each with a power of two per vector (powers are whole numbers,
// so references move without a rounding). Accumulated over the tiles by the MMAs themselves, 16 tiles would be
// 1.8e-6 off and a long run 15e-6, by an amount that depends on where the weight lies.
constexpr int kTcVecs = 128, kTcPos = 64;
constexpr int kSoftWarps = 8, kConvWarps = 8;
constexpr int kTcThreads = 32 * (kSoftWarps + 1 + kConvWarps);
constexpr uint32_t kTmemQ = 0, kTmemS = 128, kTmemCols = 512;  // S: two buffers
constexpr uint32_t kTmemSum = 256, kTmemProduct = 384;            // an item's sums so far, a tile's product
constexpr int kPShift = 14;  // a tile's probabilities with their values' powers are brought to 2^14 at most

constexpr int kMaxItems = 32;  // of a CTA: a lane of every warp finds one
constexpr int kTailBytes = 10240;
template <int HD>
struct TcSmem {
  static constexpr int kv_bytes = kTcPos * HD * 2;  // hi or lo of K or V
  static constexpr int stage = 4 * kv_bytes;
  static constexpr int raw_at = 2 * stage;          // the next tile's keys and values as they come, a slot per converter
  static constexpr int tail_at = raw_at + 2 * kTcPos * HD * 4;
  static constexpr int total = tail_at + kTailBytes + 1024;  // the tail, and room to align the start to 1 KiB
};

__device__ __forceinline__ int tiles_of(const Item &it) { return (it.p1 - it.p0 + kTcPos - 1) / kTcPos; }

__device__ __forceinline__ const float *shfl_ptr(const float *p, int from) {
  return reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)p, from));
}

// A whole warp's bounded wait, with one answer for all lanes: false once any wait of the CTA has given up.
__device__ __forceinline__ bool tc_wait(uint64_t *bar, unsigned parity, volatile int *abort_flag) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    ok = *abort_flag == 0;
    if (ok && !mbar_wait_sleep_bounded(bar, parity)) {
      *abort_flag = 1;
      ok = false;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// kind::f16 instruction descriptor: fp16 A and B, A K-major, B K-major or MN-major, fp32 accumulators, M x N.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// MN-major operand in the 128-byte swizzle: rows of 64 values along N, 8 rows (K) to an atom of 1 KiB; atoms 1 KiB apart
// along K, `n_bytes` apart along N.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(const void *smem_tile, uint32_t n_bytes) {
  uint64_t d = (smem_u32(smem_tile) >> 4) & 0x3FFFull;
  d |= (uint64_t)(n_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// A from TMEM (lane = row, a 32-bit column holds two neighbouring elements), B from shared memory.
__device__ __forceinline__ void umma_f16_ta(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// 16 lanes x 8 N consecutive columns, four registers to 8 columns: lane t has columns 2 (t % 4) and the next of row t / 4
// in the first two, of row t / 4 + 8 in the others.
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_rows(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Writes 32 lanes (this warp's quadrant) x 16 consecutive columns.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The power k for a largest magnitude (its bits): magnitudes times 2^k below 2^15. At most 100 (zeros, and maxima below
// 2^-86; those below 2^-97 keep fewer than 22 bits), so that a scale times 2^-k is a normal number.
__device__ __forceinline__ int shift_for(unsigned max_bits) {
  const int e = (int)(max_bits >> 23) - 127;
  return min(14 - e, 100);
}
// 2^k for k <= 127, 0 below the normal range.
__device__ __forceinline__ float pow2(int k) { return k < -126 ? 0.0f : __int_as_float((k + 127) << 23); }

// The power of two 2^(m + rest) of a vector's values, as two whole numbers: m is a reference of the softmax (-infinity
// where all values are zeros so far), which may be too large for the sum to be one, and rest is small.
struct Power {
  float m, rest;
};
__device__ __forceinline__ float minus(const Power &a, const Power &b) { return (a.m - b.m) + (a.rest - b.rest); }
// 2^(a - b), 0 below the normal range; a is not above b by more than 127.
__device__ __forceinline__ float pow2_ratio(const Power &a, const Power &b) {
  const float e = minus(a, b);
  return e >= -126.0f ? pow2((int)e) : 0.0f;
}

// Two values (packed) as packed fp16 high parts and the packed rest.
__device__ __forceinline__ void split2(uint64_t xy, uint32_t &hi, uint32_t &lo) {
  float x, y;
  f2_unpack(xy, x, y);
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  f2_unpack(f2_fma(f2_pack(f.x, f.y), f2_pack(-1.0f, -1.0f), xy), x, y);  // exact
  const __half2 l = __floats2half2_rn(x, y);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float abs_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float abs_max(float m, float4 v) { return abs_max3(abs_max3(m, v.x, v.y), v.z, v.w); }

struct TcTail {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pfull[2], pvdone[2], added, qfull;
  uint32_t tmem;
  int abort_flag;
  // Of each key 2^-k, of each value 2^-k and -k: a ring of tiles.
  __align__(16) float kscale[4][kTcPos], vscale[4][kTcPos], vlog[4][kTcPos];
  // A bit for each of eight positions whose keys or values hold a NaN or an infinity.
  __align__(8) uint8_t wrong[4][kConvWarps];
  int qshift[2][kTcVecs];  // of this item and the next
  float m[2][kTcVecs], l[2][kTcVecs];  // of a group's tiles
  Power sum[kTcVecs], last[kTcVecs];   // of the item's sums so far, and of its last tile's product where it has several
  Item items[kMaxItems];
};
static_assert(sizeof(TcTail) <= kTailBytes, "the tail's room");

// 16 bytes from global to shared memory, asynchronously; zeros without `in`.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Four elements of every 16 from src on, zeros from `left` elements on.
template <int HD>
__device__ __forceinline__ void load_row(float4 (&x)[HD / 16], const float *src, int left) {
  if (((uintptr_t)src & 15) == 0) {
#pragma unroll
    for (int c = 0; c < HD / 16; c++)
      x[c] = 16 * c < left ? *reinterpret_cast<const float4 *>(src + 16 * c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  } else {
#pragma unroll
    for (int c = 0; c < HD / 16; c++)
      x[c] = 16 * c < left ? make_float4(src[16 * c], src[16 * c + 1], src[16 * c + 2], src[16 * c + 3])
                           : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
}
// All but the newest group of this thread's copies are done.
__device__ __forceinline__ void copy_wait1() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// Eight rows of a tile in a warp's registers: HD / 4 lanes to a row. They come by way of a slot of shared memory, where
// every lane reads what it copied itself.
template <int HD>
struct Rows8 {
  static constexpr int kSteps = HD / 16;    // float4 a lane: 8 or 4
  static constexpr int kAt = 128 / HD;      // rows a step
  float4 x[kSteps];

  // Starts the copy of rows [row0, row0 + 8) of cache rows of hd floats; rows from `end` on and columns from hd on are
  // zeros.
  static __device__ __forceinline__ void copy(float4 *slot, const float *cache, int row0, int end, int hd, int lane) {
    const int col = lane * 4 % HD, r = lane * 4 / HD;
    const float *src = cache + (size_t)(row0 + r) * hd + col;
    const uint32_t dst = smem_u32(slot + lane);
    if (hd == HD && row0 + 8 <= end) {  // whole rows: addresses a constant apart
#pragma unroll
      for (int i = 0; i < kSteps; i++)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 512 * i), "l"(src + i * kAt * HD) : "memory");
      return;
    }
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const bool in = row0 + r + i * kAt < end && col < hd;
      copy16(dst + 512 * i, in ? src + (size_t)i * kAt * hd : cache, in);
    }
  }
  __device__ __forceinline__ void take(const float4 *slot, int lane) {
#pragma unroll
    for (int i = 0; i < kSteps; i++)
      x[i] = slot[32 * i + lane];
#pragma unroll
    for (int i = 0; i < kSteps; i++)  // the values are here before the slot's next copy starts
      asm volatile("" : "+f"(x[i].x), "+f"(x[i].y), "+f"(x[i].z), "+f"(x[i].w)::"memory");
  }
  // Splits the rows, with a power of two for each (2^k with k as shift_for gives it), and stores them as rows row .. row + 7
  // of the operand pair (64 rows of 128 swizzled bytes to 64 columns); returns the bits of 2^-k of row lane % 8. Rows with
  // a NaN or an infinity are stored as zeros and named in `wrong`: the queries that do not see them are not to notice.
  __device__ __forceinline__ int store(uint8_t *hi_at, uint8_t *lo_at, int row, int lane, unsigned *wrong) {
    const int col = lane * 4 % HD, r = lane * 4 / HD;
    const uint32_t base = (col >> 6) * (kTcPos * 128) + row * 128 + (col & 7) * 2;
    auto place = [&](int i) {
      const int rr = r + i * kAt;
      return base + rr * 128 + ((((col & 63) >> 3) ^ (rr & 7)) << 4);
    };
    unsigned own = 0;
    *wrong = 0;
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const unsigned top = __float_as_uint(abs_max(0.0f, x[i]));
      unsigned mine = 0;
#pragma unroll
      for (int a = 0; a < kAt; a++) {
        const unsigned bits = __reduce_max_sync(0xffffffffu, kAt == 1 || r == a ? top : 0u);
        *wrong |= (bits >= 0x7f800000u ? 1u : 0u) << (i * kAt + a);
        own = (lane & 7) == i * kAt + a ? bits : own;
        mine = kAt == 1 || r == a ? bits : mine;
      }
      const unsigned power = min((268u << 23) - (mine & 0x7f800000u), 227u << 23);
      const uint64_t f = f2_pack_bits(power, power);
      uint2 hi, lo;
      split2(f2_mul(f2_pack(x[i].x, x[i].y), f), hi.x, lo.x);
      split2(f2_mul(f2_pack(x[i].z, x[i].w), f), hi.y, lo.y);
      *reinterpret_cast<uint2 *>(hi_at + place(i)) = hi;
      *reinterpret_cast<uint2 *>(lo_at + place(i)) = lo;
    }
    if (*wrong) {
#pragma unroll
      for (int i = 0; i < kSteps; i++)
        if (*wrong >> (r + i * kAt) & 1) {
          *reinterpret_cast<uint2 *>(hi_at + place(i)) = make_uint2(0, 0);
          *reinterpret_cast<uint2 *>(lo_at + place(i)) = make_uint2(0, 0);
        }
      own = *wrong >> (lane & 7) & 1 ? 0 : own;
    }
    return max((int)(own & 0x7f800000u) - (14 << 23), 27 << 23);
  }
};

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
  // This CTA's items: every warp finds them all, a lane each, so that none has to wait for the first. Those with tiles
  // go into the list; a split that got no positions is an empty result.
  Item it;
  memset(&it, 0, sizeof(it));
  const int id = item_id(a, blockIdx.x, gridDim.x, lane);
  if (id >= 0 && !item_at(a, id, kTcVecs, warp == 0, &it))
    it.vecs = 0;
  const bool any = it.vecs > 0 && it.p1 > it.p0;
  const unsigned mask = __ballot_sync(0xffffffffu, any);
  const int items = __popc(mask);
  if (warp == 0) {
    if (any)
      t->items[__popc(mask & ((1u << lane) - 1))] = it;
    for (unsigned rest = __ballot_sync(0xffffffffu, it.vecs > 0 && !any); rest; rest &= rest - 1) {
      const int from = __ffs(rest) - 1;
      const int vecs = __shfl_sync(0xffffffffu, it.vecs, from), first = __shfl_sync(0xffffffffu, it.first, from);
      const int kv = __shfl_sync(0xffffffffu, it.kv, from), split = __shfl_sync(0xffffffffu, it.split, from);
      for (int i = lane; i < vecs; i += 32)
        a.ml[(size_t)split * a.vectors + vector_at(a, kv, first + i)] = make_float2(-INFINITY, 0.0f);
    }
  }
  if (!items)
    return;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&t->kfull[i], kConvWarps);
      mbar_init(&t->vfull[i], kConvWarps);
      mbar_init(&t->kempty[i], 1);
      mbar_init(&t->vempty[i], 1);
      mbar_init(&t->sfull[i], 1);
      mbar_init(&t->pfull[i], kSoftWarps / 2);
      mbar_init(&t->pvdone[i], 1);
    }
    mbar_init(&t->qfull, kSoftWarps);
    mbar_init(&t->added, kSoftWarps / 2);
    t->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kSoftWarps)
    tmem_alloc(&t->tmem, kTmemCols);
  const int hd = a.hd;
  const int cw = warp - kSoftWarps - 1;
  float4 *kslot = reinterpret_cast<float4 *>(smem + L::raw_at) + max(cw, 0) * (4 * HD), *vslot = kslot + 2 * HD;
  if (cw >= 0) {  // the first tile starts on its way
    const int from = __ffs(mask) - 1;
    const int p0 = __shfl_sync(0xffffffffu, it.p0, from) + 8 * cw, p1 = __shfl_sync(0xffffffffu, it.p1, from);
    Rows8<HD>::copy(kslot, shfl_ptr(it.k, from), p0, p1, hd, lane);
    copy_commit();
    Rows8<HD>::copy(vslot, shfl_ptr(it.v, from), p0, p1, hd, lane);
    copy_commit();
  }
  int vec_ahead = 0;  // softmax warps: the vector of the next item
  if (warp < kSoftWarps) {
    const int from = __ffs(mask) - 1;
    const int first = __shfl_sync(0xffffffffu, it.first, from), vecs = __shfl_sync(0xffffffffu, it.vecs, from);
    vec_ahead = vector_of(a, first, vecs, __shfl_sync(0xffffffffu, it.kv, from), 32 * (warp & 3) + lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = t->tmem;

  if (warp > kSoftWarps) {
    // ---- converters ----
    // The slots hold tile j; once its rows are in registers, the copies of tile j + 1 start. Every copy is a group of its
    // own, empty past the last. The tiles of all items are one sequence; `ahead` is the item of the tile fetched next.
    const float *ck = t->items[0].k, *cv = t->items[0].v;
    int ahead = 0, at = t->items[0].p0 + 8 * cw, end = t->items[0].p1;
    auto advance = [&]() {
      at += kTcPos;
      if (at - 8 * cw >= end && ahead < items && ++ahead < items) {
        const Item &it = t->items[ahead];
        ck = it.k, cv = it.v, at = it.p0 + 8 * cw, end = it.p1;
      }
    };
    Rows8<HD> x;
    auto next = [&](float4 *slot, const float *cache) {
      copy_wait1();
      x.take(slot, lane);
      if (ahead < items)
        Rows8<HD>::copy(slot, cache, at, end, hd, lane);
      copy_commit();
    };
    int tiles = 0;
    for (int n = 0; n < items; n++)
      tiles += tiles_of(t->items[n]);
    for (int j = 0; j < tiles; j++) {
      advance();
      const int s = j & 1, use = j >> 1;
      uint8_t *stage = smem + s * L::stage;
      next(kslot, ck);
      tc_wait(&t->kempty[s], (use & 1) ^ 1, abort_flag);
      unsigned wrong, wrong_v;
      const int ks = x.store(stage, stage + L::kv_bytes, 8 * cw, lane, &wrong);
      if (lane < 8)
        t->kscale[j & 3][8 * cw + lane] = __int_as_float(ks);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->kfull[s]);
      next(vslot, cv);
      tc_wait(&t->vempty[s], (use & 1) ^ 1, abort_flag);
      const int vs = x.store(stage + 2 * L::kv_bytes, stage + 3 * L::kv_bytes, 8 * cw, lane, &wrong_v);
      if (lane < 8)
        t->vscale[j & 3][8 * cw + lane] = __int_as_float(vs), t->vlog[j & 3][8 * cw + lane] = (float)((vs >> 23) - 127);
      if (lane == 0)
        t->wrong[j & 3][cw] = (uint8_t)(wrong | wrong_v);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->vfull[s]);
    }
  } else if (warp == kSoftWarps) {
    // ---- MMA issue. The scores of tile j + 1 go out before the sums of tile j, so that they run under its softmax, or
    // after them where they have to wait for the next item's queries. The MMAs run in the order of issue, so the scores
    // of tile j + 2 never overtake the sums that read their buffer. ----
    const bool leader = elect_one();
    const uint32_t idesc_s = umma_idesc_f16(kTcVecs, kTcPos, false), idesc_o = umma_idesc_f16(kTcVecs, HD, true);
    const uint64_t kdesc = umma_desc_sw128(smem), vdesc = umma_desc_sw128_mn(smem + 2 * L::kv_bytes, kTcPos * 128);
    auto scores = [&](int j) {
      const int s = j & 1, use = j >> 1;
      if (!tc_wait(&t->kfull[s], use & 1, abort_flag))
        return;
      tc_fence_after();
      if (leader) {
        const uint64_t kd = kdesc + (uint64_t)(s * (L::stage >> 4));
        const uint32_t d = tmem + kTmemS + 64 * s;
#pragma unroll
        for (int term = 0; term < 3; term++)  // lo hi, hi lo, hi hi: the small terms first
#pragma unroll
          for (int c = 0; c < HD / 16; c++)
            umma_f16_ta(d, tmem + kTmemQ + (term == 0 ? 64 : 0) + 8 * c,
                        kd + ((term == 1 ? L::kv_bytes : 0) + (c >> 2) * (kTcPos * 128) + 32 * (c & 3)) / 16, idesc_s,
                        term || c);
        umma_commit(&t->sfull[s]);
        umma_commit(&t->kempty[s]);
      }
      __syncwarp();
    };
    if (tc_wait(&t->qfull, 0, abort_flag))
      scores(0);
    int first = 0, last = tiles_of(t->items[0]) - 1;  // the item's tiles
    int adds = 0;
    for (int j = 0, n = 0;; j++) {
      if (j < last)
        scores(j + 1);
      const int s = j & 1, use = j >> 1;
      // An item's first product is its sums and its last one is taken at its end: those between are added to the sums
      // before the next one takes their place.
      if (!tc_wait(&t->vfull[s], use & 1, abort_flag) || !tc_wait(&t->pfull[s], use & 1, abort_flag) ||
          (j > first + 1 && !tc_wait(&t->added, adds++ & 1, abort_flag)))
        break;
      tc_fence_after();
      if (leader) {
        const uint64_t vd = vdesc + (uint64_t)(s * (L::stage >> 4));
        const uint32_t p = tmem + kTmemS + 64 * s, d = tmem + (j == first ? kTmemSum : kTmemProduct);
#pragma unroll
        for (int term = 0; term < 3; term++)
#pragma unroll
          for (int c = 0; c < kTcPos / 16; c++)  // 32 positions: 16 columns of hi, 16 of lo
            umma_f16_ta(d, p + 32 * (c >> 1) + 8 * (c & 1) + (term == 0 ? 16 : 0),
                        vd + ((term == 1 ? L::kv_bytes : 0) + 2048 * c) / 16, idesc_o, term || c);
        umma_commit(&t->pvdone[s]);
        umma_commit(&t->vempty[s]);
      }
      __syncwarp();
      if (j == last) {
        if (++n >= items || !tc_wait(&t->qfull, n & 1, abort_flag))
          break;
        scores(j + 1);
        first = j + 1, last = j + tiles_of(t->items[n]);
      }
    }
  } else {
    // ---- softmax: a thread per query vector, group g the tiles of its parity ----
    const int g = warp >> 2, vec_i = 32 * (warp & 3) + lane;
    const uint32_t quadrant = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t ts = quadrant + kTmemS + 64 * g;
    int vec = -1;
    for (int n = 0, j0 = 0, j1 = 0;; n++) {
      const int at = vec;
      const bool some = n < items;
      if (some) {
        // The queries become the A operand in TMEM once the scores of the tiles before are done. Group g's warps lay out
        // 16 of the quadrant's rows: lanes have four neighbouring elements of rows lane / 4 and lane / 4 + 8, whole
        // sectors of global memory and the layout in which they go to TMEM. Vectors not in use are zeros.
        vec = vec_ahead;
        constexpr int kParts = HD / 16;
        if (32 * (warp & 3) < t->items[n].vecs) {
          float4 x[2][kParts];
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const int from = __shfl_sync(0xffffffffu, vec, 16 * g + (lane >> 2) + 8 * r);
            load_row<HD>(x[r], a.q + (size_t)max(from, 0) * hd + 4 * (lane & 3), from < 0 ? 0 : hd - 4 * (lane & 3));
          }
          int k[2];
#pragma unroll
          for (int r = 0; r < 2; r++) {
            float mx = 0.0f;
#pragma unroll
            for (int c = 0; c < kParts; c++)
              mx = abs_max(mx, x[r][c]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            k[r] = shift_for(__float_as_uint(mx));
            if ((lane & 3) == 0)
              t->qshift[n & 1][32 * (warp & 3) + 16 * g + (lane >> 2) + 8 * r] = k[r];
          }
          if (n)
            tc_wait(&t->sfull[(j1 - 1) & 1], ((j1 - 1) >> 1) & 1, abort_flag);
          tc_fence_after();
          const uint32_t to_q = quadrant + ((uint32_t)(16 * g) << 16) + kTmemQ;
#pragma unroll
          for (int c0 = 0; c0 < kParts; c0 += 4) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int r = 0; r < 2; r++) {
              const uint64_t f = f2_pack(pow2(k[r]), pow2(k[r]));
#pragma unroll
              for (int c = 0; c < 4; c++) {
                const float4 y = x[r][c0 + c];
                split2(f2_mul(f2_pack(y.x, y.y), f), hi[4 * c + 2 * r], lo[4 * c + 2 * r]);
                split2(f2_mul(f2_pack(y.z, y.w), f), hi[4 * c + 2 * r + 1], lo[4 * c + 2 * r + 1]);
              }
            }
            tmem_st_rows(to_q + 8 * c0, hi);
            tmem_st_rows(to_q + 64 + 8 * c0, lo);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&t->qfull);
        if (n + 1 < items) {
          const Item &it = t->items[n + 1];
          vec_ahead = vector_of(a, it.first, it.vecs, it.kv, vec_i);
        }
      }
      if (n) {
        // Item n - 1: the sums, and the last tile's product with them, become the partial result, 16 rows of the quadrant
        // by each group, in the layout of the queries.
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftWarps) : "memory");
        const Item &from_it = t->items[n - 1];
        const bool several = j1 - j0 > 1;
        const bool done = tc_wait(&t->pvdone[(j1 - 1) & 1], ((j1 - 1) >> 1) & 1, abort_flag);
        if (done && 32 * (warp & 3) < from_it.vecs) {
          tc_fence_after();
          const float m0 = t->m[0][vec_i], m1 = t->m[1][vec_i], both = fmaxf(m0, m1);
          const float w0 = m0 == -INFINITY ? 0.0f : ex2(m0 - both), w1 = m1 == -INFINITY ? 0.0f : ex2(m1 - both);
          if (at >= 0 && g == 0)
            a.ml[(size_t)from_it.split * a.vectors + at] = make_float2(both, w0 * t->l[0][vec_i] + w1 * t->l[1][vec_i]);
          const Power result = {both, 0.0f};
          const float f0 = both == -INFINITY ? 0.0f : pow2_ratio(t->sum[vec_i], result);
          const float f1 = both == -INFINITY || !several ? 0.0f : pow2_ratio(t->last[vec_i], result);
          float *part = a.acc + (size_t)from_it.split * a.vectors * hd + 2 * (lane & 3);
          float *dst[2];
          uint64_t s0[2], s1[2];
          bool in[2];
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const int row = 16 * g + (lane >> 2) + 8 * r;
            const float x0 = __shfl_sync(0xffffffffu, f0, row), x1 = __shfl_sync(0xffffffffu, f1, row);
            s0[r] = f2_pack(x0, x0), s1[r] = f2_pack(x1, x1);
            const int to_vec = __shfl_sync(0xffffffffu, at, row);
            in[r] = to_vec >= 0;
            dst[r] = part + (size_t)max(to_vec, 0) * hd;
          }
          const uint32_t from = quadrant + ((uint32_t)(16 * g) << 16);
          if (32 * (warp & 3) + 16 * g < from_it.vecs)
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[16], p[16];
              tmem_ld_rows(from + kTmemSum + c, o);
              tmem_ld_rows(from + kTmemProduct + c, p);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const int r = e >> 1 & 1, col = c + 2 * (e & 12);
                uint64_t y = f2_mul(f2_pack_bits(o[e], o[e + 1]), s0[r]);
                if (several)
                  y = f2_fma(f2_pack_bits(p[e], p[e + 1]), s1[r], y);
                if (in[r] && col + 2 * (lane & 3) < hd) {
                  float2 z;
                  f2_unpack(y, z.x, z.y);
                  *reinterpret_cast<float2 *>(dst[r] + col) = z;
                }
              }
            }
          tc_fence_before();
        }
        if (!some)
          break;
        // Only now may the next item's first product overwrite the sums, and its results what the other group reads here.
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftWarps) : "memory");
      }
      tc_wait(&t->qfull, n & 1, abort_flag);
      const int qshift = t->qshift[n & 1][vec_i];
      const Item &it = t->items[n];
      j0 = j1, j1 += tiles_of(it);
      const bool have = vec_i < it.vecs, busy = 32 * (warp & 3) < it.vecs;
      const int limit = have ? limit_of(a, it, it.first + vec_i) : it.p0;
      const int lowest = __reduce_min_sync(0xffffffffu, have ? limit : 0x7fffffff);
      const float scale = rsqrtf((float)hd) * kLog2e * pow2(-qshift);
      const uint64_t scale2 = f2_pack(scale, scale);
      float m = -INFINITY, l = 0.0f;
      for (int j = j0 + ((j0 ^ g) & 1); j < j1; j += 2) {
        const int use = j >> 1;
        // The scores and the values' powers. (The group's previous product is done when the scores are; the wait keeps
        // step with the barrier's phases.)
        if (!tc_wait(&t->sfull[g], use & 1, abort_flag) || !tc_wait(&t->vfull[g], use & 1, abort_flag) ||
            (use > 0 && !tc_wait(&t->pvdone[g], (use - 1) & 1, abort_flag)))
          break;
        tc_fence_after();
        Power own = {-INFINITY, 0.0f};  // of the tile's product
        if (busy) {
          const int p0 = it.p0 + (j - j0) * kTcPos;
          const bool masked = p0 + kTcPos > lowest;
          const float *kscale = t->kscale[j & 3], *vscale = t->vscale[j & 3], *vlog = t->vlog[j & 3];
          // 32 scores from column c on, without the row's scale where `plain`, else in units of log 2 and -infinity where
          // they are not seen.
          auto scores = [&](auto plain, int c, uint64_t (&y)[16]) {
            tmem_ld32_pairs(ts + c, y);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float4 f = *reinterpret_cast<const float4 *>(kscale + c + 2 * e);
              uint64_t f0 = f2_pack(f.x, f.y), f1 = f2_pack(f.z, f.w);
              if (!decltype(plain)::value)
                f0 = f2_mul(f0, scale2), f1 = f2_mul(f1, scale2);
              y[e] = f2_mul(y[e], f0), y[e + 1] = f2_mul(y[e + 1], f1);
            }
            if (!decltype(plain)::value && masked)
#pragma unroll
              for (int e = 0; e < 16; e++) {
                float y0, y1;
                f2_unpack(y[e], y0, y1);
                y[e] = f2_pack(p0 + c + 2 * e < limit ? y0 : -INFINITY, p0 + c + 2 * e + 1 < limit ? y1 : -INFINITY);
              }
          };
          // Their maximum, and the maximum of score + log2 of the value's power, scores taken from `from` on.
          auto maxima = [&](float from, float &top, float &high) {
            top = high = -INFINITY;
            const uint64_t from2 = f2_pack(-from, -from);
#pragma unroll 1
            for (int c = 0; c < 64; c += 32) {
              uint64_t y[16];
              scores(std::false_type(), c, y);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const float4 v = *reinterpret_cast<const float4 *>(vlog + c + 2 * e);
                float y0, y1, y2, y3, z0, z1, z2, z3;
                y[e] = f2_add(y[e], from2), y[e + 1] = f2_add(y[e + 1], from2);
                f2_unpack(y[e], y0, y1);
                f2_unpack(y[e + 1], y2, y3);
                f2_unpack(f2_add(y[e], f2_pack(v.x, v.y)), z0, z1);
                f2_unpack(f2_add(y[e + 1], f2_pack(v.z, v.w)), z2, z3);
                top = max3(max3(top, y0, y1), y2, y3);
                high = max3(max3(high, z0, z1), z2, z3);
              }
            }
          };
          // The plain case: every row of the warp sees the whole tile, the values' powers lie within 2^10 of one another
          // (so that their largest will do for the row's own), no scale times a score overflows and no score is beyond
          // 2^15 (where powers added to it are rounded away). All tiles the general way: 222 us instead of 213 at 256 rows
          // behind 8192 positions.
          const int v0 = (int)vlog[lane], v1 = (int)vlog[lane + 32], vmax = __reduce_max_sync(0xffffffffu, max(v0, v1));
          bool plain = !masked && vmax - __reduce_min_sync(0xffffffffu, min(v0, v1)) <= 10 &&
                       __all_sync(0xffffffffu, fmaxf(kscale[lane], kscale[lane + 32]) < 0x1p80f);
          float top = -INFINITY, high = -INFINITY;
          if (plain) {
#pragma unroll 1
            for (int c = 0; c < 64; c += 32) {
              uint64_t y[16];
              scores(std::true_type(), c, y);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float y0, y1, y2, y3;
                f2_unpack(y[e], y0, y1);
                f2_unpack(y[e + 1], y2, y3);
                top = max3(max3(top, y0, y1), y2, y3);
              }
            }
            top *= scale;
            high = top + (float)vmax;
            plain = __all_sync(0xffffffffu, fabsf(top) <= 0x1p15f);
          }
          if (!plain)
            maxima(0.0f, top, high);
          const float m_new = fmaxf(m, ceilf(top)), base = m_new == -INFINITY ? 0.0f : m_new;
          l *= m == -INFINITY ? 0.0f : ex2(m - m_new);
          m = m_new;
          if (!plain && __any_sync(0xffffffffu, top > 0x1p15f || (top < -0x1p15f && top > -INFINITY)))
            maxima(base, top, high);  // the differences first
          else
            high -= base;
          const float rest = fmaxf(ceilf(high) - (float)kPShift, -120.0f);
          own = Power{m, rest};
          // Probabilities times 2^-rest and their values' powers, and their sum.
          auto probabilities = [&](auto plain) {
            const float raise = pow2(-(int)rest), from = decltype(plain)::value ? -base - rest : -base;
            const uint64_t from2 = f2_pack(from, from), raise2 = f2_pack(raise, raise);
#pragma unroll 1
            for (int c = 0; c < 64; c += 32) {
              uint64_t y[16], sum2 = 0;
              uint32_t hi[16], lo[16];
              scores(plain, c, y);
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const float2 v = *reinterpret_cast<const float2 *>(vscale + c + 2 * e);
                float x0, x1;
                f2_unpack(decltype(plain)::value ? f2_fma(y[e], scale2, from2) : f2_add(y[e], from2), x0, x1);
                uint64_t p = f2_pack(ex2(x0), ex2(x1));
                sum2 = f2_add(sum2, p);
                p = f2_mul(p, f2_pack(v.x, v.y));
                if (!decltype(plain)::value)
                  p = f2_mul(p, raise2);
                split2(p, hi[e], lo[e]);
              }
              float s0, s1;
              f2_unpack(sum2, s0, s1);
              l = fmaf(s0 + s1, decltype(plain)::value ? pow2((int)rest) : 1.0f, l);
              tmem_st16(ts + c, hi);
              tmem_st16(ts + c + 16, lo);
            }
          };
          if (plain)
            probabilities(std::true_type());
          else
            probabilities(std::false_type());
          tmem_wait_st();
          // A vector that sees a position which is not finite has no result.
          const unsigned long long wrong = *reinterpret_cast<const unsigned long long *>(t->wrong[j & 3]);
          if (wrong && limit > p0 && (limit - p0 >= 64 || wrong << (64 - (limit - p0))))
            l = NAN;
        }
        if (busy && j == j0)
          t->sum[vec_i] = own;
        if (busy && j == j1 - 1)
          t->last[vec_i] = own;
        tc_fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&t->pfull[g]);
        if (j > j0 && j < j1 - 1) {
          if (!tc_wait(&t->pvdone[g], use & 1, abort_flag))
            break;
          tc_fence_after();
          if (busy) {
            const Power before = t->sum[vec_i];
            const Power after = minus(own, before) > 0.0f ? own : before;
            const float keep = pow2_ratio(before, after), f = pow2_ratio(own, after);
            const uint64_t keep2 = f2_pack(keep, keep), f2 = f2_pack(f, f);
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint64_t o[16], p[16];
              tmem_ld32_pairs(quadrant + kTmemSum + c, o);
              tmem_ld32_pairs(quadrant + kTmemProduct + c, p);
              tmem_wait_ld();
#pragma unroll
              for (int h = 0; h < 2; h++) {
                uint32_t y[16];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                  float y0, y1;
                  f2_unpack(f2_fma(p[8 * h + e], f2, f2_mul(o[8 * h + e], keep2)), y0, y1);
                  y[2 * e] = __float_as_uint(y0), y[2 * e + 1] = __float_as_uint(y1);
                }
                tmem_st16(quadrant + kTmemSum + c + 16 * h, y);
              }
            }
            tmem_wait_st();
            t->sum[vec_i] = after;
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0)
            mbar_arrive(&t->added);
        }
      }
      t->m[g][vec_i] = m, t->l[g][vec_i] = l;
    }
  }
  __syncthreads();
  if (warp == kSoftWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int HD>
cudaError_t launch_tc(const SharedArgs &a, unsigned ctas) {
  const cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(shared_tc_kernel<HD>), TcSmem<HD>::total);
  return e != cudaSuccess ? e
                          : kc_launch_pdl(shared_tc_kernel<HD>, dim3(ctas), dim3(kTcThreads), TcSmem<HD>::total,
                                          kc_stream(), a);
}

// Heads of whole 16-byte units at 16-byte addresses.
bool tc_shape(const SharedArgs &a) {
  const uintptr_t at = (uintptr_t)a.k | (uintptr_t)a.v | (a.prefix ? (uintptr_t)a.pk | (uintptr_t)a.pv : 0);
  return a.hd <= 128 && a.hd % 4 == 0 && !(at & 15);
}

// A warp per output vector: the splits joined in their order, and optionally quantized in gs-groups as k_quantize does.
// 8192 vectors of 128 from 9 splits: 12 us, bounded by the partial results' way out of L2 (38 MB).
__global__ void __launch_bounds__(256) shared_merge_kernel(const SharedArgs a) {
  __shared__ float weights[8][2 * kMaxSplits];
  __shared__ __align__(16) float outs[8][kMaxHd];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vec = blockIdx.x * 8 + warp;
  if (vec >= a.vectors)
    return;
  const int row = vec / a.n_heads, b = row / a.rows, r = row - b * a.rows;
  const int splits = a.prefix_splits + a.own_splits, hd = a.hd;
  const Request request = request_of(a, b);
  constexpr int kPer = 2 * kMaxSplits / 32;
  float2 ml[kPer];  // read before the request is looked at: one round trip
#pragma unroll
  for (int i = 0; i < kPer; i++)
    ml[i] = lane + 32 * i < splits ? __ldcg(&a.ml[(size_t)(lane + 32 * i) * a.vectors + vec]) : make_float2(-INFINITY, 0.0f);
  if (r >= request.count)
    return;  // rows out of use stay as they were
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; i++)
    top = fmaxf(top, ml[i].x);
#pragma unroll
  for (int o = 16; o; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const float w = ml[i].x == -INFINITY ? 0.0f : exp2f(ml[i].x - top);
    weights[warp][lane + 32 * i] = w;
    sum += w * ml[i].y;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncwarp();
  const float inv = 1.0f / sum;
  const float *acc = a.acc + (size_t)vec * hd;
  const size_t step = (size_t)a.vectors * hd;
  if (hd % 4 == 0) {
    for (int e = 4 * lane; e < hd; e += 128) {
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int s = 0; s < splits; s += 8) {  // eight loads in flight; a split without weight was not written
        float4 x[8];
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          w[i] = s + i < splits ? weights[warp][s + i] : 0.0f;
          x[i] = w[i] != 0.0f ? __ldcg(reinterpret_cast<const float4 *>(acc + (s + i) * step + e))
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
          o.x = fmaf(w[i], x[i].x, o.x), o.y = fmaf(w[i], x[i].y, o.y), o.z = fmaf(w[i], x[i].z, o.z),
          o.w = fmaf(w[i], x[i].w, o.w);
      }
      o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
      if (((uintptr_t)a.out & 15) == 0)
        *reinterpret_cast<float4 *>(a.out + (size_t)vec * hd + e) = o;
      else
        a.out[(size_t)vec * hd + e] = o.x, a.out[(size_t)vec * hd + e + 1] = o.y, a.out[(size_t)vec * hd + e + 2] = o.z,
                               a.out[(size_t)vec * hd + e + 3] = o.w;
      *reinterpret_cast<float4 *>(&outs[warp][e]) = o;
    }
  } else {
    for (int e = lane; e < hd; e += 32) {
      float o = 0.0f;
      for (int s = 0; s < splits; s++)
        if (weights[warp][s] != 0.0f)
          o = fmaf(weights[warp][s], acc[s * step + e], o);
      o *= inv;
      a.out[(size_t)vec * hd + e] = o;
      outs[warp][e] = o;
    }
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
long long ceil_div64(long long a, long long b) { return (a + b - 1) / b; }

bool shape_ok(int n_heads, int n_kv, int hd, int batch, int rows) {
  constexpr long long most = 1 << 24;  // vectors; the product of two of the numbers does not wrap
  return n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && hd > 0 && hd <= kMaxHd && batch > 0 && rows > 0 &&
         (long long)batch * rows <= most && (long long)batch * rows * n_heads <= most;
}
constexpr int kMaxPositions = 0x7fffffff - 1024;  // tiles are numbered past the last one

// Floats of n (m, l) pairs, to a whole number of 16-byte units: the accumulators behind them stay aligned.
size_t pairs_floats(size_t n) { return (2 * n + 3) & ~(size_t)3; }

// Partial results of up to 2 * kMaxSplits splits as far as 96 MiB hold them, of two at least (one of the prefix, one of
// the requests' own positions).
size_t partial_floats(int n_heads, int hd, int batch, int rows) {
  const size_t vectors = (size_t)batch * rows * n_heads, each = vectors * (hd + 2);
  size_t splits = ((size_t)96 << 20) / (sizeof(float) * each);
  splits = splits < 2 ? 2 : splits > 2 * kMaxSplits ? 2 * kMaxSplits : splits;
  return splits * each + 4;
}

// How the positions are split, `most` splits at most, two at least: the lengths whose CTAs are estimated to end first.
// In units of a tile of 64 positions against a query tile (about 1.5 us): an item takes kItem units besides its tiles,
// and kItemFull more with a whole tile of queries to bring and of results to write; the requests' caches are taken to be
// half full; a split costs its partial results' way to memory and back. No more than kSplitTiles tiles to a split where the
// work's size allows it.
// Returns the CTAs, one per SM, or more where each would have more than kMaxItems items.
constexpr double kItem = 2.2, kItemFull = 1.2;
constexpr int kSplitTiles = 16;
int plan_splits(SharedArgs *a, int most, bool tc) {
  const int prefix_tiles = ceil_div(a->prefix, kTcPos), own_tiles = ceil_div(a->seq, kTcPos);
  const int columns = a->n_kv * a->tiles, own_columns = a->n_kv * a->batch * a->own_tiles;
  const int vecs = a->batch * a->rows * a->group, own_vecs = a->rows * a->group;
  double item = kItem + kItemFull * (vecs < kTcVecs ? vecs : kTcVecs) / kTcVecs;
  double own_item = kItem + kItemFull * (own_vecs < kTcVecs ? own_vecs : kTcVecs) / kTcVecs;
  double pass = (double)a->vectors * (a->hd + 2) * 8 / 5e12 / 1.5e-6;  // a split's partial results
  if (!tc)  // a tile of the generic kernel takes ten times as long, the rest as long
    item *= 0.1, own_item *= 0.1, pass *= 0.1;
  const int most_own = most / 2 < kMaxSplits ? most / 2 : kMaxSplits;
  double best = 0.0;
  int ctas = 1, tried_own = 0;
  for (int own_length = own_tiles < kSplitTiles ? own_tiles : kSplitTiles; own_length >= 1; own_length -= own_length > 4 ? 2 : 1) {
    const int own = ceil_div(own_tiles, own_length) < most_own ? ceil_div(own_tiles, own_length) : most_own;
    if (own == tried_own)
      continue;
    tried_own = own;
    const int rest = most - own < kMaxSplits ? most - own : kMaxSplits;
    int tried = -1;
    for (int length = prefix_tiles < kSplitTiles ? prefix_tiles : kSplitTiles; length >= (prefix_tiles ? 1 : 0); length--) {
      int n = prefix_tiles ? ceil_div(prefix_tiles, length) : 0;
      n = n < rest ? n : rest;
      if (n == tried)
        continue;
      tried = n;
      const double c = n ? item + (double)prefix_tiles / n : 0.0, c_own = own_item + 0.5 * own_tiles / own;
      const long long p = (long long)columns * n, o = (long long)own_columns * own;
      long long g = p + o < kPlanSms ? p + o : kPlanSms;
      if (ceil_div64(p + o, kMaxItems - 4) > g)  // fewer than kMaxItems with up to 3 extra ones
        g = ceil_div64(p + o, kMaxItems - 4);
      const long long heavy = p % g, light = g - heavy;
      const int want = (int)(c / c_own + 0.5);
      long long extra = heavy ? o / light : 0;
      extra = extra < want ? extra : want;
      extra = extra < 3 ? extra : 3;
      const long long turn = o - extra * light;
      const double end_heavy = (p / g + 1) * c + (turn / g + (turn % g > light)) * c_own;
      const double end_light = (p / g) * c + (extra + turn / g + (turn % g > 0)) * c_own;
      const double t = (heavy && end_heavy > end_light ? end_heavy : end_light) + pass * (n + own);
      if (best == 0.0 || t < best) {
        best = t;
        a->prefix_splits = n;
        a->own_splits = own;
        a->per_cta = (int)(p / g);
        a->heavy = (int)heavy;
        a->extra = (int)extra;
        ctas = (int)g;
      }
      if (!prefix_tiles)
        break;
    }
  }
  return ctas;
}

size_t generic_smem(int hd) { return sizeof(float) * ((size_t)kGenericPos * (2 * hd + 1) + kGenericWarps * (size_t)hd); }

}  // namespace

extern "C" {

size_t k_attention_shared_bytes(int n_heads, int n_kv_heads, int head_dim, int batch, int rows) {
  if (!shape_ok(n_heads, n_kv_heads, head_dim, batch, rows))
    return 0;
  return sizeof(float) * partial_floats(n_heads, head_dim, batch, rows);
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
  work->n_heads = n_heads;
  work->head_dim = head_dim;
  work->workers = batch * rows;
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
  if (!shape_ok(n_heads, n_kv_heads, head_dim, batch, rows) || seq_len <= 0 || rows > seq_len ||
      seq_len > kMaxPositions || prefix < 0 || prefix > prefix_seq_len || prefix > kMaxPositions) {
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
  if (!work || !work->partial || work->max_chunks != 0 || work->n_heads != n_heads || work->head_dim != head_dim ||
      (long long)batch * rows > work->workers) {
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
  const bool tc = tc_shape(a);
  const int tile = tc ? kTcVecs : kGenericVecs;
  a.tiles = ceil_div(batch * rows * a.group, tile);
  a.own_tiles = ceil_div(rows * a.group, tile);
  const int ctas = plan_splits(&a, (int)((work->capacity - 4) / ((size_t)a.vectors * (head_dim + 2))), tc);
  a.by_prefix_splits = divisor(a.prefix_splits ? a.prefix_splits : 1);
  a.by_own_splits = divisor(a.own_splits);
  a.by_kv = divisor(a.n_kv);
  a.by_own_tiles = divisor(a.own_tiles);
  a.by_group = divisor(a.group);
  a.by_rows = divisor(a.rows);
  const size_t splits = (size_t)a.prefix_splits + a.own_splits;
  a.ml = reinterpret_cast<float2 *>(work->partial);
  a.acc = work->partial + pairs_floats(splits * a.vectors);
  const long long items = (long long)n_kv_heads * ((long long)a.tiles * a.prefix_splits +
                                                   (long long)batch * a.own_tiles * a.own_splits);
  if (items > 0x7fffffff) {
    kc_fail("%s: batch %d of %d rows is too large", name, batch, rows);
    return;
  }
  cudaError_t e;
  if (tc) {
    e = head_dim > 64 ? launch_tc<128>(a, ctas) : launch_tc<64>(a, ctas);
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
