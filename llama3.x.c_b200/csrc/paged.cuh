// What the kernels of attention over a paged cache share (paged.cu, paged_tc.cu): the requests, the shares of the work, and
// the end of a piece of it.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "divide.cuh"
#include "kernels_cuda_internal.h"

namespace paged {

constexpr int kMaxHd = 256;
constexpr float kLog2e = 1.44269504088896341f;

// A request's rows in use and the positions stored before them; 0 rows where they are not sound.
struct Request {
  int count, start;
  bool bad;
};
__device__ __forceinline__ Request request_of(const int *starts, const int *counts, int b, int rows, int positions) {
  const int count = counts ? counts[b] : rows, start = starts[b];
  const bool ok = count > 0 && count <= rows && start >= 0 && start <= positions - count;
  return Request{ok ? count : 0, start, !ok && count != 0};
}

struct PagedArgs {
  const float *q;
  const void *key, *value;
  const int *table, *starts, *counts;
  float *out;
  int8_t *oq;
  float *os;
  float *partial;        // [2 ctas] slots of slot_floats
  unsigned *tickets;     // one to a segment, zero between calls
  size_t page_stride;
  int pages, max_pages, positions, page_size;
  int n_heads, n_kv, group, hd, batch, rows, gs;
  int block, blocks;     // query vectors to a segment, and segments to a KV head of a request with all rows
  int slot_floats;
  Divisor by_page, by_group;
};

// Slots: a flag (4 floats), m and l of each vector, then their sums.
__host__ __device__ __forceinline__ int slot_size(int block, int hd) { return (4 + 2 * block + block * hd + 3) & ~3; }

// Tiles of a request's segments (of each one), and how many segments it has. The shares are cut in units: a segment's first
// stands for its beginning and end, which take about as long as a tile, the others are its tiles (64 requests of up to 1024
// positions: 46 us so, 51 with shares of as many tiles).
struct Shape {
  int tiles, segments, blocks;
  __device__ __forceinline__ long long units() const { return tiles ? (long long)(tiles + 1) * segments : 0; }
};
__device__ __forceinline__ Shape shape_of(const PagedArgs &a, const Request &r, int tile) {
  Shape s;
  s.blocks = (r.count * a.group + a.block - 1) / a.block;
  s.segments = a.n_kv * s.blocks;
  s.tiles = r.count ? (r.start + r.count + tile - 1) / tile : 0;
  return s;
}

// The shares of the units: `each` to a CTA, one more to the first `longer`. This CTA's are [lo, hi); request b, with
// `before` units before its own, holds the first of them.
struct Range {
  long long lo, hi, each, longer, before;
  Request request;
  Shape shape;
  int b;
};

// n / d where either is small more often than not.
__device__ __forceinline__ long long quotient(long long n, long long d) {
  return ((n | d) >> 32) == 0 ? (long long)((unsigned)n / (unsigned)d) : n / d;
}

// The CTA whose share holds unit x.
__device__ __forceinline__ int owner(const Range *range, long long x) {
  const long long edge = range->longer * (range->each + 1);
  return (int)(x < edge ? quotient(x, range->each + 1) : range->longer + quotient(x - edge, range->each));
}

// This CTA's share of `total` units: false where it has none.
__device__ __forceinline__ bool share(long long total, Range *range) {
  const long long ctas = total < gridDim.x ? total : gridDim.x, cta = blockIdx.x;
  if (cta >= ctas)
    return false;
  range->each = quotient(total, ctas), range->longer = total - range->each * ctas;
  range->lo = range->each * cta + min(cta, range->longer);
  range->hi = range->lo + range->each + (cta < range->longer);
  return true;
}

__device__ __forceinline__ long long scan(long long x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    x += lane >= o ? y : 0;
  }
  return x;
}

// This CTA's share, and the request in which it begins, in every thread's registers. All threads call it;
// `common` is shared memory. False: nothing to do. Up to kAlone requests, every warp finds it alone, a few requests to a
// lane: no barrier on the way to the first page (with two, a call of one request took 0.5 us longer).
constexpr int kEachAlone = 4, kAlone = 32 * kEachAlone;
struct RangeRoom {
  long long sums[32];
  Range range;
};
__device__ __forceinline__ bool find_range(const PagedArgs &a, int tile, Range *range, RangeRoom *common) {
  const int threads = blockDim.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  if (a.batch <= kAlone) {
    const int per = (a.batch + 31) / 32, b0 = lane * per;
    Request r[kEachAlone];
    Shape s[kEachAlone];
    long long own = 0;
#pragma unroll
    for (int i = 0; i < kEachAlone; i++)
      if (i < per && b0 + i < a.batch)
        r[i] = request_of(a.starts, a.counts, b0 + i, a.rows, a.positions);
      else
        r[i] = Request{0, 0, false};
#pragma unroll
    for (int i = 0; i < kEachAlone; i++) {
      if (r[i].bad && blockIdx.x == 0 && warp == 0)
        kc_raise(KC_ERR_BAD_ARGS);
      s[i] = shape_of(a, r[i], tile);
      own += s[i].units();
    }
    const long long upto = scan(own, lane);
    if (!share(__shfl_sync(0xffffffffu, upto, 31), range))
      return false;
    const int from = __ffs(__ballot_sync(0xffffffffu, range->lo < upto)) - 1;
    long long before = upto - own;
    Request at = r[0];
    Shape shape = s[0];
    int b = b0;
#pragma unroll
    for (int i = 0; i + 1 < kEachAlone; i++)
      if (b == b0 + i && lane == from && range->lo >= before + s[i].units())
        before += s[i].units(), b++, at = r[i + 1], shape = s[i + 1];
    range->before = __shfl_sync(0xffffffffu, before, from);
    range->b = __shfl_sync(0xffffffffu, b, from);
    range->request.count = __shfl_sync(0xffffffffu, at.count, from);
    range->request.start = __shfl_sync(0xffffffffu, at.start, from);
    range->request.bad = false;
    range->shape.tiles = __shfl_sync(0xffffffffu, shape.tiles, from);
    range->shape.segments = __shfl_sync(0xffffffffu, shape.segments, from);
    range->shape.blocks = __shfl_sync(0xffffffffu, shape.blocks, from);
    return true;
  }
  const int per = (a.batch + threads - 1) / threads;
  const int b0 = min(a.batch, t * per), b1 = min(a.batch, b0 + per);
  long long own = 0;
  for (int b = b0; b < b1; b++) {
    const Request r = request_of(a.starts, a.counts, b, a.rows, a.positions);
    if (r.bad && blockIdx.x == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    const Shape s = shape_of(a, r, tile);
    own += s.units();
  }
  long long upto = scan(own, lane);
  if (lane == 31)
    common->sums[warp] = upto;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < threads / 32; w++) {
    const long long x = common->sums[w];
    upto += w < warp ? x : 0;
    total += x;
  }
  if (!share(total, range))
    return false;
  long long before = upto - own;
  if (range->lo >= before && range->lo < upto) {
    for (int b = b0;; b++) {
      const Request r = request_of(a.starts, a.counts, b, a.rows, a.positions);
      const Shape s = shape_of(a, r, tile);
      const long long n = s.units();
      if (range->lo < before + n) {
        range->before = before, range->b = b, range->request = r, range->shape = s;
        common->range = *range;
        break;
      }
      before += n;
    }
  }
  __syncthreads();
  *range = common->range;
  __syncthreads();  // the room may be used again
  return true;
}

// Weights are held times 2^-guard, 2^guard above the positions that a row sees: so that the sum of as many values of the
// type's largest size, each with the largest weight, is a number.
__device__ __forceinline__ float guard_of(int positions) { return __int_as_float((127 - (32 - __clz(positions))) << 23); }

// One piece of work: tiles [t0, t1) of a segment.
struct Piece {
  int b, head, block;       // request, KV head, block of query vectors
  int start, count, vecs;   // the request's; vectors of this block
  int t0, t1, tiles;
  long long first;          // the segment's first unit
};

// Walks through a CTA's pieces; every thread that walks sees the same.
struct Walk {
  long long at, before;
  int b;
  Request request;
  Shape shape;
  __device__ __forceinline__ explicit Walk(const Range *range)
      : at(range->lo), before(range->before), b(range->b), request(range->request), shape(range->shape) {}
  __device__ __forceinline__ bool next(const PagedArgs &a, const Range *range, int tile, Piece *p) {
    for (;;) {
      if (at >= range->hi)
        return false;
      while (at - before >= shape.units()) {
        before += shape.units();
        b++;
        request = request_of(a.starts, a.counts, b, a.rows, a.positions);
        shape = shape_of(a, request, tile);
      }
      const int units = shape.tiles + 1;
      const long long local = at - before;
      const int segment = (int)quotient(local, units);
      p->first = before + (long long)segment * units;
      p->t0 = max((int)(at - p->first) - 1, 0);
      p->t1 = (int)min((long long)units, range->hi - p->first) - 1;
      at = p->first + p->t1 + 1;
      if (p->t1 == p->t0)  // the share ends with the segment's first unit
        continue;
      p->b = b;
      p->head = segment / shape.blocks;
      p->block = segment - p->head * shape.blocks;
      p->start = request.start, p->count = request.count;
      p->vecs = min(a.block, request.count * a.group - p->block * a.block);
      p->tiles = shape.tiles;
      return true;
    }
  }
  // Whether the piece is the share's last but for a segment's first unit.
  static __device__ __forceinline__ bool last(const Range *range, const Piece &p) {
    return p.first + 1 + p.t1 >= range->hi;
  }
};

// Vector v of a piece: index in the [batch][rows][n_heads] order.
__device__ __forceinline__ int vector_at(const PagedArgs &a, const Piece &p, int v, int *row) {
  int member = p.block * a.block + v;
  *row = divide(member, a.by_group);
  return (p.b * a.rows + *row) * a.n_heads + p.head * a.group + member;
}

template <int THREADS, int BARRIER>
__device__ __forceinline__ void meet() {
  asm volatile("bar.sync %0, %1;" ::"n"(BARRIER), "n"(THREADS) : "memory");
}

// The piece's vectors, with m and l of each and their sums o in shared memory, written to the output (a whole segment,
// or the last of its pieces to be done) or to a slot. All threads call it, after a barrier behind the last write to m, l,
// o and bad; it ends with one. THREADS threads, numbered t, meet at barrier BARRIER. HD:
// head_dim, or 0 where it is any.
template <int THREADS, int BARRIER, int HD>
__device__ __forceinline__ void finish(const PagedArgs &a, const Range *range, const Piece &p, float *m, float *l, float *o,
                       const int *bad, int *last, int t) {
  constexpr int threads = THREADS;
  const int hd = HD ? HD : a.hd;
  bool wrong = *bad != 0;
  if (p.t0 || p.t1 < p.tiles) {
    const int c0 = owner(range, p.first + 1), c1 = owner(range, p.first + p.tiles);
    const int cta = blockIdx.x, n = p.vecs * hd;
    const int l_at = 4 + a.block, o_at = 4 + 2 * a.block;
    auto slot_of = [&](int c) { return a.partial + (size_t)(2 * c + (c == c0)) * a.slot_floats; };
    float *slot = slot_of(cta);
    if (t == 0)
      slot[0] = wrong ? 1.0f : 0.0f;
    for (int i = t; i < p.vecs; i += threads)
      slot[4 + i] = m[i], slot[l_at + i] = l[i];
    if (hd % 4 == 0)
      for (int i = 4 * t; i < n; i += 4 * threads)
        *reinterpret_cast<float4 *>(slot + o_at + i) = *reinterpret_cast<const float4 *>(o + i);
    else
      for (int i = t; i < n; i += threads)
        slot[o_at + i] = o[i];
    meet<THREADS, BARRIER>();
    if (t == 0) {
      const size_t segment = ((size_t)p.b * a.n_kv + p.head) * a.blocks + p.block;
      __threadfence();  // the barrier's and this fence's order together: the slot is in memory before the ticket
      *last = atomicInc(&a.tickets[segment], (unsigned)(c1 - c0)) == (unsigned)(c1 - c0);
      __threadfence();
    }
    meet<THREADS, BARRIER>();
    if (!*last) {
      meet<THREADS, BARRIER>();
      return;
    }
    // Several slots at a time on their way; those past the last are the last again, without weight.
    constexpr int kAt = THREADS > 256 ? 4 : 8;
    wrong = false;
    const int step = hd % 4 == 0 ? 4 : 1;
    for (int i = step * t; i < n; i += step * threads) {
      const int v = i / hd;
      float top = -INFINITY, sum = 0.0f;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int c = c0; c <= c1; c += kAt) {
        float mc[kAt], lc[kAt], flag[kAt], high = top;
        float4 oc[kAt];
#pragma unroll
        for (int j = 0; j < kAt; j++) {
          const float *from = slot_of(min(c + j, c1));
          flag[j] = __ldcg(from), mc[j] = __ldcg(from + 4 + v), lc[j] = __ldcg(from + l_at + v);
          oc[j] = step == 4 ? __ldcg(reinterpret_cast<const float4 *>(from + o_at + i))
                            : make_float4(__ldcg(from + o_at + i), 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int j = 0; j < kAt; j++) {
          wrong |= flag[j] != 0.0f;
          high = fmaxf(high, mc[j]);
        }
        const float keep = top == -INFINITY ? 0.0f : exp2f(top - high);
        x.x *= keep, x.y *= keep, x.z *= keep, x.w *= keep, sum *= keep;
        top = high;
#pragma unroll
        for (int j = 0; j < kAt; j++) {
          if (c + j > c1)
            continue;
          const float w = mc[j] == -INFINITY ? 0.0f : exp2f(mc[j] - top);  // times NaN, where there is one, it is NaN
          sum = fmaf(w, lc[j], sum);
          x.x = fmaf(w, oc[j].x, x.x), x.y = fmaf(w, oc[j].y, x.y);
          x.z = fmaf(w, oc[j].z, x.z), x.w = fmaf(w, oc[j].w, x.w);
        }
      }
      if (step == 4)
        *reinterpret_cast<float4 *>(o + i) = x;
      else
        o[i] = x.x;
      if (i - v * hd < step)
        l[v] = sum;
    }
    if (wrong)
      *last = -1;
    meet<THREADS, BARRIER>();
    wrong = *last < 0;
  }
  if (wrong) {
    if (t == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    meet<THREADS, BARRIER>();
    return;
  }
  const bool wide = hd % 4 == 0 && ((uintptr_t)a.out & 15) == 0;
  const int unit = wide ? 4 : 1;
  for (int i = unit * t; i < p.vecs * hd; i += unit * threads) {
    const int v = i / hd;
    int row;
    float *to = a.out + (size_t)vector_at(a, p, v, &row) * hd + (i - v * hd);
    const float sum = l[v];
    // A mean of finite values may come out past the largest one by its rounding.
    auto mean = [&](float x) {
      const float y = x / sum;
      return fabsf(y) == INFINITY && fabsf(x) < INFINITY ? copysignf(3.402823466e+38f, y) : y;
    };
    if (wide) {
      float4 x = *reinterpret_cast<const float4 *>(o + i);
      x.x = mean(x.x), x.y = mean(x.y), x.z = mean(x.z), x.w = mean(x.w);
      *reinterpret_cast<float4 *>(to) = x;
      if (a.oq)
        *reinterpret_cast<float4 *>(o + i) = x;
    } else {
      o[i] = *to = mean(o[i]);
    }
  }
  meet<THREADS, BARRIER>();
  if (!a.oq)
    return;
  const int warp = t >> 5, lane = t & 31, groups = hd / a.gs;
  for (int i = warp; i < p.vecs * groups; i += threads / 32) {
    const int v = i / groups, g = (i - v * groups) * a.gs;
    int row;
    const size_t at = (size_t)vector_at(a, p, v, &row) * hd + g;
    const float *x = o + v * hd + g;
    float mx = 0.0f;
    bool infinite = false;
    for (int e = lane; e < a.gs; e += 32) {
      infinite |= !(fabsf(x[e]) < INFINITY);
      mx = fmaxf(mx, fabsf(x[e]));
    }
#pragma unroll
    for (int s = 16; s; s >>= 1)
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    if (infinite)
      kc_raise(KC_ERR_NONFINITE);
    const float scale = __fdiv_rn(mx, 127.0f);
    for (int e = lane; e < a.gs; e += 32)
      a.oq[at + e] = (int8_t)quantize_value(x[e], scale);
    if (lane == 0)
      a.os[at / a.gs] = scale;
  }
  meet<THREADS, BARRIER>();
}

}  // namespace paged

// The tensor-core kernel (paged_tc.cu): whether it takes the call, its query vectors to a segment, and its launch.
bool kc_paged_tc_ok(const paged::PagedArgs &a, int type);
int kc_paged_tc_block(int group, int rows);
int kc_paged_tc_slots_floats(int hd);
cudaError_t kc_launch_paged_tc(const paged::PagedArgs &a, int type);

// The tile kernel for fp32 (paged_f32.cu): whether it takes the call, and its launch; segments of kPagedF32Block vectors.
constexpr int kPagedF32Block = 8;
bool kc_paged_f32_ok(const paged::PagedArgs &a, int type);
cudaError_t kc_launch_paged_f32(const paged::PagedArgs &a);
