// Attention over a paged cache on the tensor cores: 16-bit keys and values, head_dim 64 or 128, 16-byte aligned pages.
//
// The positions are the rows of both products, so that a decode step's few query vectors cost no padding to 128 and the
// cache's bytes go from global memory to the tensor core as they are: for a tile of 128 positions
//   S^T [128 positions x N] = K [128 x hd] Q^T,    O^T [hd x N] = V^T [hd x 128 positions] P^T,
// K the K-major and V the MN-major operand A of the same row-major layout (128-byte swizzle), Q and P the operand B.
// The 16-bit types are widened by columns: a query vector takes three of the N columns, x = x0 + x1 + x2 in three 16-bit
// parts, and so does a vector of probabilities; the products of a 16-bit key or value with each part are exact, their sum
// is the fp32 product up to 2^-22 of it.
//   bf16: the parts are the leading, middle and last eight bits of the significand, cut off, not rounded: no part's
//         rounding carries into the one before, and they add up to x exactly. bf16 has fp32's exponents.
//   fp16: x 2^k with the largest magnitude of a query vector just below 2^15 (probabilities: 2^15 at most), then each part
//         rounded and the rest times 2^11 for the next, so that a part of a small x is not lost below fp16's exponents; the
//         columns are joined with 2^-11 and 2^-22. The last part is a multiple of 2^-24, so x is off by up to 2^-47: 2^-22 of
//         it down to 2^-25. A query's largest element is 2^14 at least, a row's largest probability 2^7: 2^-22 of elements
//         down to 2^-39 and of probabilities down to 2^-32 of the largest, below that 2^-61 and 2^-54 of the largest.
// A tile's sums are a product of their own, eight MMAs that start at zero; they join the running sums in fp32, in
// registers, rounded to nearest (the tensor cores' accumulators cut towards zero).
//
// A CTA per SM takes its share of the tiles of all segments without a pause between segments. Its warps: softmax, a thread
// per position of a tile and per element of the head of its sums, in groups of four warps that share out the query vectors
// (4 or 8 to a thread: with all 32 of the largest block in one group, a tile took 3.9 us); one that issues the MMAs; one to
// three that lay out the next segment's queries; four that copy the tiles, asynchronously, through a ring of stages. With up
// to eight vectors two more finish a segment (by the softmax warps themselves that takes 2 us of their time, and the shares
// of many short segments ended last: 8 requests of up to 2048 positions 19 us back to back with them against 22), but for a
// share's last, for which the softmax warps are faster; with more vectors those do it all (16 requests of up to five rows behind
// 4099, in blocks of 32: 58 us back to back against 64).
//
// What bounds it (32/8 heads of 128): for long requests memory, 64 of up to 8192 positions in bf16 205 us, 6.5 TB/s of the
// copy's 6.55, 1.5 us a tile; with 20 vectors, 16 requests of up to five rows behind 4099 48 us, nothing that is full (DRAM 41 %,
// issue slots 46 %, tensor pipe 9 % under a profiler): chains of dependent steps in the softmax and in the joins; for short ones
// the way to the first tile (5 us: the share, pages, copies) and the join of the pieces (4 us: results to memory, ticket, results
// back), which the code of those rare steps, fetched anew each time, makes longer: 8 requests of up to 2048 positions in fp16
// 16.4 us, 2.4 TB/s.
//
// A later draft's key or value of any kind must not reach the rows before it, not even with a weight of zero: a key gives
// scores in its own row of S^T only, which are masked; a value with an infinity or a NaN behind the block's first row is
// zeroed before its product, and the rows that see it get NaN for a weight there.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace {
using namespace paged;

constexpr int kTile = 128;  // positions
constexpr int kCopyWarps = 4;
constexpr int kCtas = 148;
constexpr int kMaxBlock = 32;
constexpr int kMaxStages = 10;
constexpr int kSmem = 227 * 1024;

template <int RESULTS>
struct Tail {
  uint64_t full[kMaxStages], empty[kMaxStages], sfull[2], pfull[2], ofull[2], qfull[2], qempty[2], rfull[2], rempty[2];
  uint64_t drained;
  uint32_t tmem;
  int abort_flag;
  __align__(16) float top[4][kMaxBlock];  // a tile's maxima by warp
  // A piece's results beside its sums: references, sums of weights by warp, a page that is none.
  struct {
    float m[kMaxBlock], l[4][kMaxBlock];
    int bad, last;
  } result[RESULTS];
  // Of the queries: four pieces, since the softmax may be two tiles behind the scores, and the queries two pieces ahead.
  float qscale[4][kMaxBlock];
};

template <int HD, int BLOCK>
struct Layout {
  static constexpr int groups = BLOCK == 4 ? 1 : BLOCK == 8 ? 2 : 4, vecs = BLOCK / groups;  // vectors to a thread
  static constexpr bool ends = groups < 4;  // warps that finish pieces
  static constexpr int query_warps = ends ? 1 : 3, end_warps = ends ? 2 : 0;  // (12, 16 or 24 warps in all)
  static constexpr int soft = 128 * groups;  // softmax threads
  static constexpr int threads = soft + 32 + 32 * (query_warps + end_warps) + 32 * kCopyWarps;
  static constexpr int n = (3 * BLOCK + 15) / 16 * 16;  // columns
  static constexpr int entry = kTile * HD * 2;
  static constexpr int q_bytes = n * HD * 2, p_bytes = n * kTile * 2;
  static constexpr int r_bytes = BLOCK * HD * 4, r_room = ends ? 2 * r_bytes : 0;  // without, over the probabilities
  static constexpr int results = ends ? 2 : 1;
  using End = Tail<results>;
  static constexpr int fit = (kSmem - 1024 - 2 * (q_bytes + p_bytes) - r_room - (int)sizeof(End)) / entry;
  static constexpr int stages = fit > kMaxStages ? kMaxStages : fit;
  static constexpr int q_at = stages * entry, p_at = q_at + 2 * q_bytes;
  static constexpr int r_at = ends ? p_at + 2 * p_bytes : p_at;
  static constexpr int tail_at = p_at + 2 * p_bytes + r_room;
  static_assert(ends || 2 * p_bytes >= r_bytes, "the results' room");
  static constexpr int total = tail_at + (int)sizeof(End) + 1024;
  static constexpr int tmem = 4 * n <= 64 ? 64 : 4 * n <= 128 ? 128 : 4 * n <= 256 ? 256 : 512;
  static_assert(stages >= 4 && total <= kSmem, "shared memory");
};

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

// kind::f16, fp32 accumulators, fp16 or bf16 operands, both K-major or both MN-major, M x N.
__host__ __device__ constexpr uint32_t umma_idesc(bool bf16, int m, int n, bool mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn ? (1u << 15) | (1u << 16) : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// MN-major operand in the 32-byte swizzle: rows of 16 values along N, 8 rows (K) to an atom of 256 bytes; atoms 256 bytes
// apart along K, `n_bytes` apart along N.
__device__ __forceinline__ uint64_t umma_desc_sw32_mn(const void *smem_tile, uint32_t n_bytes) {
  uint64_t d = (smem_u32(smem_tile) >> 4) & 0x3FFFull;
  d |= (uint64_t)(n_bytes >> 4) << 16;
  d |= (uint64_t)(256 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)6 << 61;
  return d;
}
// MN-major operand in the 128-byte swizzle: rows of 64 values along M, 8 rows (K) to an atom of 1 KiB; atoms 1 KiB apart
// along K, `m_bytes` apart along M.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(const void *smem_tile, uint32_t m_bytes) {
  uint64_t d = (smem_u32(smem_tile) >> 4) & 0x3FFFull;
  d |= (uint64_t)(m_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of the warp's numbers.
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// 2^k for -126 <= k <= 127.
__device__ __forceinline__ float pow2(int k) { return __int_as_float((k + 127) << 23); }

// The next part of two numbers (fp16: already brought to fp16's range), packed, and what is left of them, exactly.
__device__ __forceinline__ uint32_t next_part(float &x, float &y, __nv_bfloat16) {
  const unsigned a = __float_as_uint(x), b = __float_as_uint(y);
  x -= __uint_as_float(a & 0xffff0000u), y -= __uint_as_float(b & 0xffff0000u);
  return __byte_perm(a, b, 0x7632);
}
__device__ __forceinline__ uint32_t next_part(float &x, float &y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  x = (x - f.x) * 2048.0f, y = (y - f.y) * 2048.0f;
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ float join(float x0, float x1, float x2) {
  return __is_same(T, __half) ? fmaf(fmaf(x2, 0x1p-11f, x1), 0x1p-11f, x0) : (x2 + x1) + x0;
}

// 16 bytes from global to shared memory, asynchronously; zeros without `in`.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// Arrives once all copies that this thread has started are in memory.
__device__ __forceinline__ void copy_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// This thread's lane of 4 or 8 columns.
__device__ __forceinline__ void tmem_ld4(uint32_t at, float (&x)[4]) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
#pragma unroll
  for (int j = 0; j < 4; j++)
    x[j] = __uint_as_float(r[j]);
}
__device__ __forceinline__ void tmem_ld8(uint32_t at, float (&x)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at));
#pragma unroll
  for (int j = 0; j < 8; j++)
    x[j] = __uint_as_float(r[j]);
}
// The joined columns of this thread's lane: part p of vector v is column p * BLOCK + v. VECS (4 or 8) vectors, `at` the
// column of the first.
template <typename T, int BLOCK, int VECS>
__device__ __forceinline__ void tmem_joined(uint32_t at, float (&x)[VECS]) {
  float p[3][VECS];
#pragma unroll
  for (int i = 0; i < 3; i++) {
    if constexpr (VECS == 4)
      tmem_ld4(at + BLOCK * i, p[i]);
    else
      tmem_ld8(at + BLOCK * i, p[i]);
  }
  tmem_wait_ld();
#pragma unroll
  for (int v = 0; v < VECS; v++)
    x[v] = join<T>(p[0][v], p[1][v], p[2][v]);
}

// The four warps of a softmax group meet; meet_any: and learn whether any of their threads says so.
__device__ __forceinline__ void meet_group(int group) { asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory"); }
__device__ __forceinline__ bool meet_any(int group, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine), "r"(2 + group)
      : "memory");
  return any != 0;
}
// The reference before there is one: a number, so that the difference to a masked score (-infinity) is none.
constexpr float kFar = 3.402823466e+38f;
// How far a score, in powers of two, may lie above the reference before the reference moves.
constexpr float kRise = 8.0f;

// The first row of a piece's block, and how many rows it has beyond that.
struct Rows {
  int first, more;
};
__device__ __forceinline__ Rows rows_of(const PagedArgs &a, const Piece &p) {
  int lo = p.block * a.block, hi = lo + p.vecs - 1;
  Rows r;
  r.first = divide(lo, a.by_group);
  r.more = divide(hi, a.by_group) - r.first;
  return r;
}

// Row of the cache that holds a position, in elements, or -1 where its page is none.
__device__ __forceinline__ long long place_of(const PagedArgs &a, const Piece &p, int position, int hd) {
  int within = position;
  const int index = divide(within, a.by_page);
  const int page = a.table[(size_t)p.b * a.max_pages + index];
  return page < 0 || page >= a.pages
             ? -1
             : (long long)((size_t)page * a.page_stride + ((size_t)p.head * a.page_size + within) * hd);
}

template <typename T, int HD, int BLOCK>
__global__ void __launch_bounds__(Layout<HD, BLOCK>::threads, 1) paged_tc_kernel(const PagedArgs a) {
  using L = Layout<HD, BLOCK>;
  constexpr int kSoft = L::soft, kVecs = L::vecs, kMma = kSoft / 32, kQuery = kMma + 1,
                kEnd = kQuery + L::query_warps, kCopy = kEnd + L::end_warps;
  constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  auto *t = reinterpret_cast<typename L::End *>(smem + L::tail_at);
  volatile int *abort_flag = &t->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::stages; i++) {
      mbar_init(&t->full[i], 32 * kCopyWarps);
      mbar_init(&t->empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&t->sfull[i], 1);
      mbar_init(&t->pfull[i], kSoft / 32);
      mbar_init(&t->ofull[i], 1);
      mbar_init(&t->qfull[i], L::query_warps);
      mbar_init(&t->qempty[i], 1);
      mbar_init(&t->rfull[i], kSoft / 32);
      mbar_init(&t->rempty[i], 1);
      t->result[i % L::results].bad = 0;
    }
    mbar_init(&t->drained, 1);
    t->abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  Range here;
  if (!find_range(a, kTile, &here, reinterpret_cast<RangeRoom *>(t->top)))
    return;
  // The copies start without the tensor memory; the MMAs' warp and the softmax meet for it. Dependents start behind its
  // allocation: a kernel that waits for this one cannot hold what it still needs.
  if (warp <= kMma) {
    if (warp == kMma) {
      tmem_alloc(&t->tmem, L::tmem);
      pdl_launch_dependents();
    }
    tc_fence_before();
    meet<kSoft + 32, 7>();
    tc_fence_after();
  }
  const uint32_t tmem = t->tmem;  // for those two
  const Range *range = &here;
  const float scale = rsqrtf((float)HD) * kLog2e;
  Walk walk(range);
  Piece p;
  // Finishes the piece whose results are in a buffer: threads numbered tid, at a barrier of their own.
  auto end_piece = [&](int at, const Piece &p, int tid, auto threads, auto barrier) {
    auto &result = t->result[at];
    if (tid < p.vecs)
      result.l[0][tid] = (result.l[0][tid] + result.l[1][tid]) + (result.l[2][tid] + result.l[3][tid]);
    if (tid == 0 && *abort_flag)
      result.bad = 1;
    meet<threads(), barrier()>();
    finish<threads(), barrier(), HD>(a, range, p, result.m, result.l[0],
                                     reinterpret_cast<float *>(smem + L::r_at + at * L::r_bytes), &result.bad, &result.last,
                                     tid);
  };

  if (warp >= kCopy) {
    // ---- copies: warp w of them the rows 32 w .. 32 w + 31 of every tile, keys and values in turn ----
    constexpr int kChunks = HD / 8, kAt = 32 / kChunks;  // 16-byte units of a row, rows of a warp's instruction
    const int w = warp - kCopy;
    const int chunk = lane % kChunks, sub = lane / kChunks;
    const uint32_t base = smem_u32(smem) + (chunk >> 3) * (kTile * 128);
    int slot = 0;
    unsigned parity = 1;
    while (walk.next(a, range, kTile, &p)) {
      const Rows rows = rows_of(a, p);
      const int end = p.start + rows.first + rows.more + 1;  // seen by any row of the block
      int position = p.t0 * kTile + 32 * w + lane;
      long long next = position < end ? place_of(a, p, position, HD) : -1;
      for (int j = p.t0; j < p.t1; j++) {
        const long long place = next;
        position += kTile;
        next = j + 1 < p.t1 && position < end ? place_of(a, p, position, HD) : -1;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
          const T *from = static_cast<const T *>(kv ? a.value : a.key) + chunk * 8;
          tc_wait(&t->empty[slot], parity, abort_flag);
#pragma unroll
          for (int i = 0; i < 32 / kAt; i++) {
            const int r = i * kAt + sub;
            const long long at = __shfl_sync(0xffffffffu, place, r);
            const int row = 32 * w + r;
            copy16(base + slot * L::entry + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), from + max(at, 0ll), at >= 0);
          }
          copy_arrive(&t->full[slot]);
          slot++;
          if (slot == L::stages)
            slot = 0, parity ^= 1;
        }
      }
    }
    copy_wait_all();
  } else if (L::ends && warp >= kEnd) {
    // ---- the pieces' ends, but for the share's last ----
    const int tid = threadIdx.x - 32 * kEnd;
    for (int n = 0; walk.next(a, range, kTile, &p) && !Walk::last(range, p); n++) {
      const int at = n & 1;
      tc_wait(&t->rfull[at], (n >> 1) & 1, abort_flag);
      end_piece(at, p, tid, std::integral_constant<int, L::ends ? 32 * L::end_warps : 32>(), std::integral_constant<int, 1>());
      if (tid == 0) {
        t->result[at].bad = 0;
        mbar_arrive(&t->rempty[at]);
      }
    }
  } else if (warp >= kQuery) {
    // ---- queries: times the scores' scale, in three parts, row part * BLOCK + v of the operand ----
    constexpr int kEach = HD / 32, kAt = 4;
    for (int n = 0; walk.next(a, range, kTile, &p); n++) {
      uint8_t *to = smem + L::q_at + (n & 1) * L::q_bytes;
      tc_wait(&t->qempty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag);
#pragma unroll 1
      for (int v0 = kAt * (warp - kQuery); v0 < BLOCK; v0 += kAt * L::query_warps) {
        float x[kAt][kEach];
#pragma unroll
        for (int u = 0; u < kAt; u++) {
          int row;
          const float *q = a.q + (size_t)vector_at(a, p, min(v0 + u, p.vecs - 1), &row) * HD;
#pragma unroll
          for (int i = 0; i < kEach; i++)
            x[u][i] = v0 + u < p.vecs ? q[2 * lane + 32 * (i & ~1) + (i & 1)] * scale : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kAt; u++) {
          const int v = v0 + u;
          if (!kBf16) {
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < kEach; i++)
              mx = fmaxf(mx, fabsf(x[u][i]));
            const int e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)) >> 23) - 127;
            const int k = min(14 - e, 100);  // so that its inverse is a normal number
#pragma unroll
            for (int i = 0; i < kEach; i++)
              x[u][i] *= pow2(k);
            if (lane == 0)
              t->qscale[n & 3][v] = pow2(-k);
          }
#pragma unroll
          for (int i = 0; i < kEach; i += 2) {
            const int e = 2 * lane + 32 * i;
#pragma unroll
            for (int part = 0; part < 3; part++) {
              const int row = part * BLOCK + v;
              *reinterpret_cast<uint32_t *>(to + (e >> 6) * (L::n * 128) + row * 128 + ((((e & 63) >> 3) ^ (row & 7)) << 4) +
                                            (e & 7) * 2) = next_part(x[u][i], x[u][i + 1], T(0.0f));
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&t->qfull[n & 1]);
    }
  } else if (warp == kMma) {
    // ---- MMA issue: the scores of tile j + 1 before the sums of tile j, so that they run under its softmax. MMAs run in
    // the order of issue. S and O have two buffers each; that a buffer was read is known from the probabilities of a later
    // tile (the softmax reads the scores of a tile before it writes its probabilities, and the sums of the tile before the
    // last by then). The copies' writes come by the generic proxy, so a fence stands between their barrier and the MMAs. ----
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = umma_idesc(kBf16, kTile, L::n, false), idesc_o = umma_idesc(kBf16, HD, L::n, true);
    const uint64_t kdesc = umma_desc_sw128(smem), vdesc = umma_desc_sw128_mn(smem, kTile * 128);
    const uint64_t qdesc = umma_desc_sw128(smem + L::q_at), pdesc = umma_desc_sw32_mn(smem + L::p_at, kTile * 32);
    int piece = -1, left = 0;  // of the scores issued next: its piece, and tiles of it left
    int kslot = 0, vslot = 1;
    unsigned kpar = 0, vpar = 0;
    bool more = true;
    auto scores = [&](int j) {
      if (!left) {
        more = walk.next(a, range, kTile, &p);
        if (!more)
          return false;
        left = p.t1 - p.t0;
        piece++;
        if (!tc_wait(&t->qfull[piece & 1], (piece >> 1) & 1, abort_flag))
          return false;
      }
      left--;
      if (!tc_wait(&t->full[kslot], kpar, abort_flag))
        return false;
      fence_proxy_async_smem();
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int c = 0; c < HD / 16; c++)
          umma_f16(tmem + L::n * (j & 1), kdesc + (kslot * L::entry + (c >> 2) * (kTile * 128) + 32 * (c & 3)) / 16,
                   qdesc + ((piece & 1) * L::q_bytes + (c >> 2) * (L::n * 128) + 32 * (c & 3)) / 16, idesc_s, c);
        umma_commit(&t->sfull[j & 1]);
        umma_commit(&t->empty[kslot]);
        if (!left)
          umma_commit(&t->qempty[piece & 1]);
      }
      __syncwarp();
      kslot += 2;
      if (kslot >= L::stages)
        kslot -= L::stages, kpar ^= 1;
      return true;
    };
    bool now = scores(0);
    for (int j = 0; now; j++) {
      now = scores(j + 1);  // false behind the last tile, or where a wait has run out
      if (!now && more)
        break;
      if (!tc_wait(&t->full[vslot], vpar, abort_flag) || !tc_wait(&t->pfull[j & 1], (j >> 1) & 1, abort_flag))
        break;
      fence_proxy_async_smem();
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int c = 0; c < kTile / 16; c++)
          umma_f16(tmem + L::n * (2 + (j & 1)), vdesc + (vslot * L::entry + 2048 * c) / 16,
                   pdesc + ((j & 1) * L::p_bytes + 512 * c) / 16, idesc_o, c);
        umma_commit(&t->ofull[j & 1]);
        umma_commit(&t->empty[vslot]);
      }
      __syncwarp();
      vslot += 2;
      if (vslot >= L::stages)
        vslot -= L::stages, vpar ^= 1;
    }
    // No MMA is under way when the tensor memory is given back, whatever ended the loop.
    if (leader)
      umma_commit(&t->drained);
    __syncwarp();
    mbar_wait_sleep_bounded(&t->drained, 0);
  } else {
    // ---- softmax ----
    const int tid = threadIdx.x, group = warp >> 2, quad = warp & 3, v0 = group * kVecs;  // the group's first vector
    const int row = 32 * quad + lane;  // a position of the tile; of the sums, a row of the tensor memory
    const uint32_t quadrant = tmem + ((uint32_t)(32 * quad) << 16) + v0;
    // M = 64 keeps 16 rows in each quadrant of the tensor memory.
    const int element = HD == 128 ? row : 16 * quad + lane;
    const bool has_element = HD == 128 || lane < 16;
    // Its row of the probabilities, and where in a row's 32 bytes its unit of 16 lies.
    uint8_t *const prow = smem + L::p_at + row * 32;
    const int punit = (row >> 2) & 1;
    int j = 0, vslot = 1;
    unsigned vpar = 0;
    for (int n = 0; walk.next(a, range, kTile, &p); n++) {
      const Rows rows = rows_of(a, p);
      const int common = p.start + rows.first + 1, end = common + rows.more;
      float m[kVecs], l[kVecs], acc[kVecs];
#pragma unroll
      for (int v = 0; v < kVecs; v++)
        m[v] = -kFar, l[v] = 0.0f, acc[v] = 0.0f;
      const bool idle = v0 >= p.vecs;  // the group has none of the block's vectors
      // Weights are up to 2^kRise times this: bf16 as guard_of says, fp16 up to 2^15 (there is no value beyond 2^16).
      const float weight = kBf16 ? guard_of(p.start + p.count) * 0x1p-8f : 0x1p7f;
      // Every page of the piece's positions is one: asked for here, looked at behind the first tile.
      int from = p.t0 * kTile, to = min(p.t1 * kTile, p.start + p.count) - 1;
      from = divide(from, a.by_page) + tid, to = divide(to, a.by_page);
      const int *pages = a.table + (size_t)p.b * a.max_pages;
      const int first_page = from <= to ? pages[from] : 0;
      auto add = [&](int i) {  // the sums of tile i
        float o[kVecs];
        tc_wait(&t->ofull[i & 1], (i >> 1) & 1, abort_flag);
        if (idle)
          return;
        tc_fence_after();
        tmem_joined<T, BLOCK, kVecs>(quadrant + L::n * (2 + (i & 1)), o);
        tc_fence_before();
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          acc[v] += o[v];
      };
      for (int tile = p.t0; tile < p.t1; tile++, j++) {
        float s[kVecs], keep[kVecs];
        tc_wait(&t->sfull[j & 1], (j >> 1) & 1, abort_flag);
        tc_fence_after();
        if (!idle) {
          tmem_joined<T, BLOCK, kVecs>(quadrant + L::n * (j & 1), s);
          if (!kBf16)
#pragma unroll
            for (int v = 0; v < kVecs; v++)
              s[v] *= t->qscale[n & 3][v0 + v];
        }
        tc_fence_before();
        const int position = tile * kTile + row;
        if (tile * kTile + kTile > common) {
          // Not all of the tile, or not the same of it to all rows.
          unsigned seen = position < common ? (1u << kVecs) - 1 : 0;  // a bit a vector
          if (rows.more) {
            tc_wait(&t->full[vslot], vpar, abort_flag);
            const bool some = position >= common && position < end;
            uint8_t *const values = smem + vslot * L::entry + row * 128;
            bool wrong = false;
            if (some) {
              constexpr unsigned kExp = kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll 4
              for (int i = 0; i < HD / 8; i++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(values + (i >> 3) * (kTile * 128) + (i & 7) * 16);
                const unsigned u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 4; k++)
                  wrong |= (u[k] & kExp) == kExp || (u[k] >> 16 & kExp) == kExp;
              }
#pragma unroll
              for (int v = 0; v < kVecs; v++) {
                int member = p.block * BLOCK + v0 + v;
                if (v0 + v < p.vecs && position <= p.start + divide(member, a.by_group)) {
                  seen |= 1u << v;
                  s[v] = wrong ? NAN : s[v];
                }
              }
            }
            meet<kSoft, 6>();  // every group has looked
            if (wrong && group == 0)
              for (int i = 0; i < HD / 8; i++)
                *reinterpret_cast<uint4 *>(values + (i >> 3) * (kTile * 128) + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int v = 0; v < kVecs; v++)
            s[v] = seen >> v & 1 ? s[v] : -INFINITY;
        }
        vslot += 2;
        if (vslot >= L::stages)
          vslot -= L::stages, vpar ^= 1;
        bool moves = false;
        if (!idle) {
          float d[kVecs], high = -INFINITY;
#pragma unroll
          for (int v = 0; v < kVecs; v++) {
            d[v] = s[v] - m[v];
            high = fmaxf(high, d[v]);
          }
          // The reference stays while no score is far above it: one barrier that tells, instead of maxima over the tile.
          moves = meet_any(group, high > kRise);
          if (moves) {
            float (*top)[kMaxBlock] = t->top;
#pragma unroll
            for (int v = 0; v < kVecs; v++) {
              const float x = warp_max(s[v]);
              if (lane == 0)
                top[quad][v0 + v] = x;
            }
            meet_group(group);
#pragma unroll
            for (int v = 0; v < kVecs; v++) {
              const float x =
                  fmaxf(fmaxf(fmaxf(top[0][v0 + v], top[1][v0 + v]), fmaxf(top[2][v0 + v], top[3][v0 + v])), m[v]);
              keep[v] = ex2(m[v] - x);
              m[v] = x;
              d[v] = s[v] - x;
              l[v] *= keep[v];
            }
          }
          float w[kVecs];
#pragma unroll
          for (int v = 0; v < kVecs; v++) {
            w[v] = ex2(d[v]) * weight;
            l[v] += w[v];
          }
#pragma unroll
          for (int part = 0; part < 3; part++) {
            const int c = part * BLOCK + v0;  // the column of the first
            uint32_t packed[kVecs / 2];
#pragma unroll
            for (int v = 0; v < kVecs; v += 2)
              packed[v / 2] = next_part(w[v], w[v + 1], T(0.0f));
            uint8_t *at = prow + (j & 1) * L::p_bytes + (c >> 4) * (kTile * 32) + (((c >> 3 & 1) ^ punit) << 4) + (c & 7) * 2;
            if constexpr (kVecs == 4)
              *reinterpret_cast<uint2 *>(at) = make_uint2(packed[0], packed[1]);
            else
              *reinterpret_cast<uint4 *>(at) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&t->pfull[j & 1]);
        if (tile > p.t0)
          add(j - 1);
        if (moves)
#pragma unroll
          for (int v = 0; v < kVecs; v++)
            acc[v] *= keep[v];
      }
      add(j - 1);
      // The piece's result.
      bool bad = first_page < 0 || first_page >= a.pages;
      for (int i = from + kSoft; i <= to; i += kSoft) {
        const int page = pages[i];
        bad |= page < 0 || page >= a.pages;
      }
      const int at = L::ends ? n & 1 : 0;
      if (L::ends)
        tc_wait(&t->rempty[at], ((n >> 1) & 1) ^ 1, abort_flag);
      auto &result = t->result[at];
      float *sums = reinterpret_cast<float *>(smem + L::r_at + at * L::r_bytes);
#pragma unroll
      for (int v = 0; v < kVecs; v++) {
        if (has_element && v0 + v < p.vecs)
          sums[(v0 + v) * HD + element] = acc[v];
#pragma unroll
        for (int o = 16; o; o >>= 1)
          l[v] += __shfl_xor_sync(0xffffffffu, l[v], o);
        if (lane == 0)
          result.l[quad][v0 + v] = l[v];
        if (row == v)
          result.m[v0 + v] = m[v];
      }
      if (bad)
        result.bad = 1;
      if (L::ends && !Walk::last(range, p)) {
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&t->rfull[at]);
      } else {
        meet<kSoft, 6>();
        end_piece(at, p, tid, std::integral_constant<int, kSoft>(), std::integral_constant<int, 6>());
        if (tid == 0)
          result.bad = 0;
        if (!L::ends)
          meet<kSoft, 6>();
      }
    }
  }
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, L::tmem);
  }
}

template <typename T, int HD, int BLOCK>
cudaError_t launch(const PagedArgs &a) {
  const auto kernel = paged_tc_kernel<T, HD, BLOCK>;
  const cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(kernel), Layout<HD, BLOCK>::total);
  return e != cudaSuccess
             ? e
             : kc_launch_pdl(kernel, dim3(kCtas), dim3(Layout<HD, BLOCK>::threads), Layout<HD, BLOCK>::total, kc_stream(), a);
}
template <typename T, int HD>
cudaError_t launch_block(const PagedArgs &a) {
  return a.block == 4    ? launch<T, HD, 4>(a)
         : a.block == 8  ? launch<T, HD, 8>(a)
         : a.block == 16 ? launch<T, HD, 16>(a)
                         : launch<T, HD, kMaxBlock>(a);
}

}  // namespace

bool kc_paged_tc_ok(const PagedArgs &a, int type) {
  return (type == K_BF16 || type == K_F16) && (a.hd == 64 || a.hd == 128) && a.page_stride % 8 == 0 &&
         !(((uintptr_t)a.key | (uintptr_t)a.value) & 15);
}

// The smallest block that holds a KV head's vectors (of as many rows as the call's longest request may have) up to 16; blocks
// of 16 up to 64 vectors, and of 32, which fetch the keys and values half as often but keep four softmax groups with eight
// vectors to a thread and a ring of two tiles, beyond. Device time in a graph of calls, us, heads of 128 in bf16:
//   16 requests of 32/8 heads, up to 4099 positions   blocks of 4     8    16    32
//     4 vectors                                            39.0  38.8  38.1  50.1
//     8                                                    43.7  39.5  39.7  52.0
//     12                                                   54.9  45.3  41.7  54.6
//     20                                                   76.0  56.1  48.4  58.6
//     32                                                    105  73.7  54.9  62.2
//     48, 64, 128                                     of 16: 66.2, 89.1, 98.7  of 32: 74.4, 83.7, 89.1
//   4 requests of 8/8 heads, up to 1000 positions, 64, 96, 128 vectors  16.2, 20.8, 23.8    21.0, 21.0, 24.6
//   512 rows of 32/8 heads behind 2048 positions            217                     160
//   32 requests of 32/8 heads, up to 2048 positions: one of 8 rows, 31 of one  40.9  41.0  41.8  60.6
int kc_paged_tc_block(int group, int rows) {
  const long long vecs = (long long)group * rows;
  return vecs <= 4 ? 4 : vecs <= 8 ? 8 : vecs <= 64 ? 16 : kMaxBlock;
}

int kc_paged_tc_slots_floats(int hd) { return 2 * kCtas * slot_size(kMaxBlock, hd); }

cudaError_t kc_launch_paged_tc(const PagedArgs &a, int type) {
  if (type == K_BF16)
    return a.hd == 128 ? launch_block<__nv_bfloat16, 128>(a) : launch_block<__nv_bfloat16, 64>(a);
  return a.hd == 128 ? launch_block<__half, 128>(a) : launch_block<__half, 64>(a);
}
