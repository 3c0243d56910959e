// Verification of drafted tokens against the target model's probabilities (k_verify_draft): for each request the drafts
// are accepted in order while u_j q_j(x_j) < p_j(x_j), and the token after them is drawn from (p_a - q_a)+ at the first
// refused draft, or from p_a behind the last one, by inverting the running sum of the weights in vocabulary order.
//
// Every sum over the vocabulary and every weight is held in 64 bits: the sampled index is where a running sum of up to
// a vocabulary of terms passes u times the total, and with 128256 borders a relative error of 2^-24 in the sums would
// move the choice for about one u in a hundred.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kSumThreads = 256;
constexpr int kChunk = 16 * kSumThreads;  // logits of a row per CTA of the sums kernel
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kPickCtas = 8;  // a cluster per request
constexpr int kMaxRows = 64;
constexpr int kMaxSlots = 2 * kMaxRows + 1;

struct VerifyArgs {
  int *accepted, *tokens;
  const float *target, *draft;
  long long ldt, ldd;
  const int *drafted, *counts;
  const float *uniforms, *temperature;
  int vocab, batch, rows, chunks;
  double *sums;              // [batch][2 rows + 1][chunks]
  unsigned long long *keys;  // the same: order-preserving maximum and its first index
};

// 64-bit key whose unsigned maximum is the first maximum. NaN and +infinity have no place in a distribution: they get
// the largest key.
__device__ __forceinline__ unsigned long long row_key(float v, int i) {
  unsigned b = __float_as_uint(v);
  if (!(v < __int_as_float(0x7f800000)))
    return ~0ull;
  if (v == 0.0f)
    b = 0;  // the two zeros are one value: the first of them wins
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (0xFFFFFFFFu - (unsigned)i);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  unsigned b = (unsigned)(k >> 32);
  b = (b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b;
  return __uint_as_float(b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xFFFFFFFFu - (unsigned)k); }
// A maximum that gives a distribution: above -infinity, and no NaN or +infinity in the row.
__device__ __forceinline__ bool key_good(unsigned long long k) {
  return k != ~0ull && key_value(k) > __int_as_float(0xff800000);
}
__device__ __forceinline__ unsigned long long max64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v = max64(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// exp of a non-positive argument (or 0).
__device__ __forceinline__ double weight(float l, float m, double inv_t) { return exp(((double)l - (double)m) * inv_t); }

__device__ __forceinline__ int count_of(const VerifyArgs &a, int b) { return a.counts ? a.counts[b] : a.rows; }

// What a (request, slot) pair of the sums needs: slot j <= rows is row j of the target, rows + 1 + j row j of the draft.
// False when nothing reads the slot.
__device__ __forceinline__ bool slot_row(const VerifyArgs &a, int b, int slot, const float **row) {
  const int count = count_of(a, b);
  if (count < 0 || count > a.rows)
    return false;
  if (slot <= a.rows) {
    *row = a.target + ((long long)b * (a.rows + 1) + slot) * a.ldt;
    return slot <= count;
  }
  const int j = slot - a.rows - 1;
  *row = a.draft ? a.draft + ((long long)b * a.rows + j) * a.ldd : nullptr;
  return a.draft && j < count && a.temperature[b] != 0.0f;
}

// One chunk of one row: its first maximum, and the sum of exp((l - max) / T) over the chunk (T > 0).
__global__ void __launch_bounds__(kSumThreads) verify_sums_kernel(const VerifyArgs a) {
  __shared__ unsigned long long key_s[kSumThreads / 32];
  __shared__ double sum_s[kSumThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int chunk = blockIdx.x % a.chunks, id = blockIdx.x / a.chunks;
  const int b = id / (2 * a.rows + 1), slot = id - b * (2 * a.rows + 1);
  const float *row;
  if (!slot_row(a, b, slot, &row))
    return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = chunk * kChunk;
  float v[16];
  unsigned long long key = 0;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int e = first + i * kSumThreads + threadIdx.x;
    v[i] = e < a.vocab ? row[e] : __int_as_float(0xff800000);
  }
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int e = first + i * kSumThreads + threadIdx.x;
    if (e < a.vocab)
      key = max64(key, row_key(v[i], e));
  }
  key = warp_max(key);
  if (lane == 0)
    key_s[warp] = key;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSumThreads / 32; w++)
    key = max64(key, key_s[w]);
  const float t = a.temperature[b];
  double sum = 0.0;
  if (t > 0.0f && key_good(key)) {
    const float m = key_value(key);
    const double inv_t = 1.0 / (double)t;
#pragma unroll
    for (int i = 0; i < 16; i++)
      sum += weight(v[i], m, inv_t);
  }
  sum = warp_sum(sum);
  if (lane == 0)
    sum_s[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < kSumThreads / 32; w++)
      sum += sum_s[w];
    a.sums[(long long)id * a.chunks + chunk] = sum;
    a.keys[(long long)id * a.chunks + chunk] = key;
  }
}

// The weight of token i when the next token is drawn: p_a(i), less q_a(i) at a refused draft (the drafted token alone
// has q = 1 where there are no draft logits).
struct Residual {
  const float *p, *q;
  float pm, qm;
  double inv_t, p_norm, q_norm;
  int without;
  __device__ __forceinline__ double operator()(int i) const {
    // Both products are rounded (no fused multiply-add): where draft and target are the same row nothing is left.
    double w = __dmul_rn(weight(p[i], pm, inv_t), p_norm);
    if (q)
      w -= __dmul_rn(weight(q[i], qm, inv_t), q_norm);
    return i == without ? 0.0 : fmax(w, 0.0);
  }
};

// A cluster per request: every CTA decides which drafts are accepted, then sums its slice of the vocabulary's weights;
// the CTA whose slice holds the place of u inverts it.
__global__ void __launch_bounds__(kPickThreads) verify_pick_kernel(const VerifyArgs a) {
  __shared__ unsigned long long key_s[kMaxSlots];
  __shared__ double sum_s[kMaxSlots], warp_sums[kPickWarps], slices[kPickCtas];
  __shared__ int stop_s;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();  // every CTA has started before any writes into another's shared memory
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x / kPickCtas, rank = blockIdx.x % kPickCtas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = count_of(a, b);
  if (count < 0)
    return;  // the whole cluster: a slot of the batch that is not in use
  const float t = a.temperature[b];
  const bool greedy = t == 0.0f;
  int *tokens = a.tokens + (long long)b * (a.rows + 1);
  const bool valid = count <= a.rows && t >= 0.0f && t < __int_as_float(0x7f800000);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)t;
  if (threadIdx.x == 0)
    stop_s = valid ? count : 0;
  if (valid)
    for (int slot = warp; slot < 2 * a.rows + 1; slot += kPickWarps) {
      const float *row;
      if (!slot_row(a, b, slot, &row))
        continue;
      const long long at = ((long long)b * (2 * a.rows + 1) + slot) * a.chunks;
      unsigned long long key = 0;
      for (int c = lane; c < a.chunks; c += 32)
        key = max64(key, a.keys[at + c]);
      key = warp_max(key);
      double sum = 0.0;
      if (!greedy && key_good(key))
        for (int c = lane; c < a.chunks; c += 32) {
          const unsigned long long k = a.keys[at + c];
          if (key_good(k))
            sum += a.sums[at + c] * weight(key_value(k), key_value(key), inv_t);
        }
      sum = warp_sum(sum);
      if (lane == 0)
        key_s[slot] = key, sum_s[slot] = sum;
    }
  __syncthreads();
  // A draft is refused, or its rows have no distribution: the first such place ends the run.
  if (valid)
    for (int j = threadIdx.x; j < count; j += kPickThreads) {
      const int x = a.drafted[(long long)b * a.rows + j], dj = a.rows + 1 + j;
      const bool rows_good = key_good(key_s[j]) && (greedy || !a.draft || key_good(key_s[dj]));
      bool good = false;
      if (rows_good && x >= 0 && x < a.vocab) {
        if (greedy) {
          good = key_index(key_s[j]) == x;
        } else {
          const float *p = a.target + ((long long)b * (a.rows + 1) + j) * a.ldt;
          const double px = weight(p[x], key_value(key_s[j]), inv_t) / sum_s[j];
          double qx = 1.0;
          if (a.draft)
            qx = weight(a.draft[((long long)b * a.rows + j) * a.ldd + x], key_value(key_s[dj]), inv_t) / sum_s[dj];
          good = (double)a.uniforms[(long long)b * (a.rows + 1) + j] * qx < px;
        }
      }
      if (!good)
        atomicMin(&stop_s, j);
    }
  __syncthreads();
  const int stop = stop_s;
  const bool refused = stop < count;
  const int x = valid && refused ? a.drafted[(long long)b * a.rows + stop] : -1;
  // No distribution at the place where the run ends (or arguments that mean nothing): no answer.
  unsigned error = 0;
  if (!valid || (refused && (x < 0 || x >= a.vocab)))
    error = KC_ERR_BAD_ARGS;
  else if (!key_good(key_s[stop]) || (refused && !greedy && a.draft && !key_good(key_s[a.rows + 1 + stop])))
    error = KC_ERR_NONFINITE;
  if (rank == 0) {
    for (int j = threadIdx.x; j <= a.rows; j += kPickThreads)
      if (error || j > stop)
        tokens[j] = -1;
      else if (j < stop)
        tokens[j] = a.drafted[(long long)b * a.rows + j];
    if (threadIdx.x == 0) {
      a.accepted[b] = error ? -1 : stop;
      if (error)
        kc_raise(error);
      else if (greedy)
        tokens[stop] = key_index(key_s[stop]);
    }
  }
  if (error || greedy)
    return;  // the whole cluster

  Residual w;
  w.p = a.target + ((long long)b * (a.rows + 1) + stop) * a.ldt;
  w.pm = key_value(key_s[stop]), w.p_norm = 1.0 / sum_s[stop], w.inv_t = inv_t;
  w.q = refused && a.draft ? a.draft + ((long long)b * a.rows + stop) * a.ldd : nullptr;
  w.qm = w.q ? key_value(key_s[a.rows + 1 + stop]) : 0.0f, w.q_norm = w.q ? 1.0 / sum_s[a.rows + 1 + stop] : 0.0;
  w.without = refused && !a.draft ? x : -1;
  // Warp segments of equal length: segment s of kPickCtas * kPickWarps.
  const int segment = (a.vocab + kPickCtas * kPickWarps - 1) / (kPickCtas * kPickWarps);
  const int s0 = min((rank * kPickWarps + warp) * segment, a.vocab), s1 = min(s0 + segment, a.vocab);
  double sum = 0.0;
  for (int i = s0 + lane; i < s1; i += 32)
    sum += w(i);
  sum = warp_sum(sum);
  if (lane == 0)
    warp_sums[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double slice = 0.0;
    for (int i = 0; i < kPickWarps; i++)
      slice += warp_sums[i];
    for (int r = 0; r < kPickCtas; r++)
      *cluster.map_shared_rank(&slices[rank], r) = slice;
  }
  cluster.sync();
  double total = 0.0, before = 0.0;
  for (int r = 0; r < kPickCtas; r++) {
    if (r == rank)
      before = total;
    total += slices[r];
  }
  if (!(total > 0.0)) {  // nothing of the target is left but rounding: its first maximum
    if (rank == 0 && threadIdx.x == 0)
      tokens[stop] = key_index(key_s[stop]);
    return;
  }
  double place = (double)a.uniforms[(long long)b * (a.rows + 1) + a.rows] * total;
  if (!(place < total))
    place = total * (1.0 - 0x1p-52);
  place = fmax(place, 0.0);
  if (place < before || place >= before + slices[rank])  // the slices tile [0, total): one CTA goes on
    return;
  // The warp whose segment the place falls into; behind the last one with weight, that one.
  int seg = -1;
  double seg_before = before;
  for (int i = 0; i < kPickWarps; i++) {
    if (warp_sums[i] > 0.0 && (seg < 0 || place >= before)) {
      seg = i;
      seg_before = before;
    }
    before += warp_sums[i];
  }
  if (warp != seg)
    return;
  int last = -1;
  double run = seg_before;
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const double mine = i < s1 ? w(i) : 0.0;
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o)
        upto += other;
    }
    upto += run;
    const unsigned past = __ballot_sync(0xffffffffu, mine > 0.0 && upto > place);
    if (past) {
      last = i0 + __ffs(past) - 1;
      break;
    }
    const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
    if (some)
      last = i0 + 31 - __clz(some);
    run = __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0)
    tokens[stop] = last;
}

size_t verify_chunks(int vocab) { return ((size_t)vocab + kChunk - 1) / kChunk; }

}  // namespace

extern "C" {

size_t k_verify_bytes(int vocab, int batch, int rows) {
  if (vocab <= 0 || batch <= 0 || rows < 0 || rows > kMaxRows)
    return 0;
  return (size_t)batch * (2 * rows + 1) * verify_chunks(vocab) * (sizeof(double) + sizeof(unsigned long long));
}

void k_verify_draft(int *accepted, int *tokens, const float *target, size_t ldt, const float *draft, size_t ldd,
                    const int *drafted, const int *counts, const float *uniforms, const float *temperature, int vocab,
                    int batch, int rows, void *work) {
  const char *name = "k_verify_draft";
  if (vocab <= 0 || batch < 0 || rows < 0 || rows > kMaxRows || ldt < (size_t)vocab ||
      (draft && rows && ldd < (size_t)vocab)) {
    kc_fail("%s: invalid shape vocab=%d batch=%d rows=%d ldt=%zu ldd=%zu (at most %d rows)", name, vocab, batch, rows,
            ldt, ldd, kMaxRows);
    return;
  }
  if (!batch)
    return;
  if (!accepted || !tokens || !target || (rows && !drafted) || !uniforms || !temperature || !work ||
      ((uintptr_t)work & 15)) {
    kc_fail("%s: missing outputs, logits, drafts, numbers or 16-byte aligned work", name);
    return;
  }
  const size_t pairs = (size_t)batch * (2 * rows + 1) * verify_chunks(vocab);
  if (pairs > 0x7fffffffu || (size_t)batch * kPickCtas > 0x7fffffffu) {
    kc_fail("%s: batch %d of %d rows is too large", name, batch, rows);
    return;
  }
  VerifyArgs a;
  a.accepted = accepted, a.tokens = tokens, a.target = target, a.draft = rows ? draft : nullptr;
  a.ldt = (long long)ldt, a.ldd = (long long)ldd, a.drafted = drafted, a.counts = counts;
  a.uniforms = uniforms, a.temperature = temperature, a.vocab = vocab, a.batch = batch, a.rows = rows;
  a.chunks = (int)verify_chunks(vocab);
  a.sums = static_cast<double *>(work);
  a.keys = reinterpret_cast<unsigned long long *>(a.sums + pairs);
  cudaError_t e =
      kc_launch_pdl(verify_sums_kernel, dim3((unsigned)pairs), dim3(kSumThreads), 0, kc_stream(), a);
  if (e == cudaSuccess) {
    kc_count_launch();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)batch * kPickCtas);
    cfg.blockDim = dim3(kPickThreads);
    cfg.stream = kc_stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kc_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kPickCtas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, verify_pick_kernel, a);
    if (e == cudaSuccess)
      kc_count_launch();
  }
  if (e != cudaSuccess)
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
