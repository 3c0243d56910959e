// Attention of a batch of requests that share a prefix (k_attention_shared_rows). Row r of request b attends to the
// prefix [0, prefix) of one cache that all requests read and to positions [0, starts[b] + r] of the request's own
// cache. The prefix is read once for all rows of the batch and not once a request: its query vectors are gathered over
// the whole batch per KV head.
//
// Both parts give partial results per query vector and split of the positions: the maximum m of the scores, the sum
// l of exp(score - m) and the vector sum of exp(score - m) v. A merge joins them: out = sum exp(m_i - M) o_i /
// sum exp(m_i - M) l_i with M the largest m_i. Statistics and accumulators are fp32.
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"

namespace {

constexpr int kMaxHd = 256;
constexpr int kPlanSms = 148;      // the plan is a function of the shape alone, so that the workspace's size is too
constexpr int kMaxSplits = 64;     // of the prefix, or of a request's own positions

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
  int prefix_splits, own_splits, tiles;  // splits of the positions; query tiles of the prefix part per KV head
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

// Items 0 .. n_kv * tiles * prefix_splits - 1 are the prefix's, then one per (request, KV head, split). False: nothing
// to do.
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
  it->kv = id % a.n_kv;
  it->b = id / a.n_kv;
  const int count = rows_of(a, it->b);
  if (!request_ok(a, it->b, count)) {
    if (count != 0 && threadIdx.x == 0)
      kc_raise(KC_ERR_BAD_ARGS);
    return false;
  }
  it->first = it->b * a.rows * a.group;
  it->vecs = count * a.group;
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
  return min(it.p1, a.starts[it.b] + (i - it.first) / a.group + 1);
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
  const float scale = rsqrtf((float)hd);
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
      const float keep = m == -INFINITY ? 0.0f : expf(m - m_new);
      const float p = seen ? expf(s - m_new) : 0.0f;
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
    const float w = ml.x == -INFINITY ? 0.0f : expf(ml.x - top);
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
  a.tiles = ceil_div(batch * rows * a.group, kGenericVecs);
  const long long items = (long long)n_kv_heads * ((long long)a.tiles * a.prefix_splits + (long long)batch * a.own_splits);
  if (items > 0x7fffffff) {
    kc_fail("%s: batch %d of %d rows is too large", name, batch, rows);
    return;
  }
  cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(shared_generic_kernel), (int)generic_smem(kMaxHd));
  if (e == cudaSuccess)
    e = kc_launch_pdl(shared_generic_kernel, dim3((unsigned)items), dim3(kGenericThreads), generic_smem(head_dim),
                      kc_stream(), a);
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
