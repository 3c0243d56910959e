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

constexpr int kRangeThreads = 320;  // at most
struct Range {
  long long lo, hi, total, before;  // this CTA's tiles, all tiles, those before request b
  int b, ctas;
  long long sums[kRangeThreads / 32];
};

// Tiles of a request's segments (of each one), and how many segments it has.
struct Shape {
  int tiles, segments, blocks;
};
__device__ __forceinline__ Shape shape_of(const PagedArgs &a, const Request &r, int tile) {
  Shape s;
  s.blocks = (r.count * a.group + a.block - 1) / a.block;
  s.segments = a.n_kv * s.blocks;
  s.tiles = r.count ? (r.start + r.count + tile - 1) / tile : 0;
  return s;
}

// This CTA's share of the tiles, and the request in which it begins. All threads call it. False: nothing to do.
__device__ __forceinline__ bool find_range(const PagedArgs &a, int tile, Range *range) {
  const int threads = blockDim.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int per = (a.batch + threads - 1) / threads, b0 = t * per, b1 = min(a.batch, b0 + per);
  long long own = 0;
  for (int b = b0; b < b1; b++) {
    const Request r = request_of(a.starts, a.counts, b, a.rows, a.positions);
    if (r.bad && blockIdx.x == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    const Shape s = shape_of(a, r, tile);
    own += (long long)s.tiles * s.segments;
  }
  long long upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, o);
    upto += lane >= o ? x : 0;
  }
  if (lane == 31)
    range->sums[warp] = upto;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < threads / 32; w++) {
    upto += w < warp ? range->sums[w] : 0;
    total += range->sums[w];
  }
  const long long ctas = total < gridDim.x ? total : gridDim.x, cta = blockIdx.x;
  if (cta >= ctas)
    return false;
  const long long lo = total * cta / ctas, hi = total * (cta + 1) / ctas;
  if (lo >= upto - own && lo < upto) {
    long long before = upto - own;
    int b = b0;
    for (;; b++) {
      const Shape s = shape_of(a, request_of(a.starts, a.counts, b, a.rows, a.positions), tile);
      const long long n = (long long)s.tiles * s.segments;
      if (lo < before + n)
        break;
      before += n;
    }
    range->lo = lo, range->hi = hi, range->total = total, range->before = before, range->b = b, range->ctas = (int)ctas;
  }
  __syncthreads();
  return true;
}

// The CTA whose share holds tile x.
__device__ __forceinline__ int owner(const Range *range, long long x) {
  return (int)(((x + 1) * range->ctas - 1) / range->total);
}

// Weights are held times 2^-guard, 2^guard above the positions that a row sees: so that the sum of as many values of the
// type's largest size, each with the largest weight, is a number.
__device__ __forceinline__ float guard_of(int positions) { return __int_as_float((127 - (32 - __clz(positions))) << 23); }

// One piece of work: tiles [t0, t1) of a segment.
struct Piece {
  int b, head, block;       // request, KV head, block of query vectors
  int start, count, vecs;   // the request's; vectors of this block
  int t0, t1, tiles;
  long long first;          // the segment's first tile
};

// Walks through a CTA's pieces; every thread that walks sees the same.
struct Walk {
  long long at, before;
  int b;
  Request request;
  Shape shape;
  __device__ __forceinline__ Walk(const PagedArgs &a, const Range *range, int tile) {
    at = range->lo, before = range->before, b = range->b;
    request = request_of(a.starts, a.counts, b, a.rows, a.positions);
    shape = shape_of(a, request, tile);
  }
  __device__ __forceinline__ bool next(const PagedArgs &a, const Range *range, int tile, Piece *p) {
    if (at >= range->hi)
      return false;
    while (at - before >= (long long)shape.tiles * shape.segments) {
      before += (long long)shape.tiles * shape.segments;
      b++;
      request = request_of(a.starts, a.counts, b, a.rows, a.positions);
      shape = shape_of(a, request, tile);
    }
    const long long local = at - before;
    const int segment = (int)(local / shape.tiles);
    p->b = b;
    p->head = segment / shape.blocks;
    p->block = segment - p->head * shape.blocks;
    p->start = request.start, p->count = request.count;
    p->vecs = min(a.block, request.count * a.group - p->block * a.block);
    p->tiles = shape.tiles;
    p->first = before + (long long)segment * shape.tiles;
    p->t0 = (int)(at - p->first);
    p->t1 = (int)min((long long)shape.tiles, range->hi - p->first);
    at = p->first + p->t1;
    return true;
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
// o and bad; it ends with one. THREADS threads, numbered from 0, meet at barrier BARRIER.
template <int THREADS, int BARRIER>
__device__ __forceinline__ void finish(const PagedArgs &a, const Range *range, const Piece &p, float *m, float *l, float *o,
                       const int *bad, int *last) {
  constexpr int threads = THREADS;
  const int t = threadIdx.x, hd = a.hd;
  bool wrong = *bad != 0;
  if (p.t0 || p.t1 < p.tiles) {
    const int c0 = owner(range, p.first), c1 = owner(range, p.first + p.tiles - 1);
    const int cta = blockIdx.x;
    float *slot = a.partial + (size_t)(2 * cta + (cta == c0)) * a.slot_floats;
    float *slot_m = slot + 4, *slot_l = slot_m + a.block, *slot_o = slot_l + a.block;
    if (t == 0)
      slot[0] = wrong ? 1.0f : 0.0f;
    for (int i = t; i < p.vecs; i += threads)
      slot_m[i] = m[i], slot_l[i] = l[i];
    for (int i = t; i < p.vecs * hd; i += threads)
      slot_o[i] = o[i];
    __threadfence();
    meet<THREADS, BARRIER>();
    if (t == 0) {
      const size_t segment = ((size_t)p.b * a.n_kv + p.head) * a.blocks + p.block;
      *last = atomicInc(&a.tickets[segment], (unsigned)(c1 - c0)) == (unsigned)(c1 - c0);
    }
    meet<THREADS, BARRIER>();
    if (!*last) {
      meet<THREADS, BARRIER>();
      return;
    }
    __threadfence();
    auto slot_of = [&](int c) { return a.partial + (size_t)(2 * c + (c == c0)) * a.slot_floats; };
    wrong = false;
    for (int c = c0; c <= c1; c++)
      wrong |= __ldcg(slot_of(c)) != 0.0f;
    for (int i = t; i < p.vecs; i += threads) {
      float top = -INFINITY, sum = 0.0f;
      for (int c = c0; c <= c1; c++)
        top = fmaxf(top, __ldcg(slot_of(c) + 4 + i));
      for (int c = c0; c <= c1; c++) {
        const float mc = __ldcg(slot_of(c) + 4 + i);
        sum += mc == -INFINITY ? 0.0f : exp2f(mc - top) * __ldcg(slot_of(c) + 4 + a.block + i);
      }
      m[i] = top, l[i] = sum;
    }
    meet<THREADS, BARRIER>();
    for (int i = t; i < p.vecs * hd; i += threads) {
      const int v = i / hd;
      float x = 0.0f;
      for (int c = c0; c <= c1; c++) {
        const float mc = __ldcg(slot_of(c) + 4 + v);
        if (mc != -INFINITY)
          x = fmaf(exp2f(mc - m[v]), __ldcg(slot_of(c) + 4 + 2 * a.block + i), x);
      }
      o[i] = x;
    }
    meet<THREADS, BARRIER>();
  }
  if (wrong) {
    if (t == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    meet<THREADS, BARRIER>();
    return;
  }
  for (int i = t; i < p.vecs * hd; i += threads) {
    const int v = i / hd;
    int row;
    const size_t vec = vector_at(a, p, v, &row);
    float x = o[i] / l[v];
    if (fabsf(x) == INFINITY && fabsf(o[i]) < INFINITY)  // a mean of finite values, past the largest one by its rounding
      x = copysignf(3.402823466e+38f, x);
    o[i] = x;
    a.out[vec * hd + (i - v * hd)] = x;
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
