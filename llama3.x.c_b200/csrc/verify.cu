// Verification of drafted tokens against the target model's probabilities (k_verify_draft): for each request the drafts
// are accepted in order while u_j q_j(x_j) < p_j(x_j), and the token after them is drawn from (p_a - q_a)+ at the first
// refused draft, or from p_a behind the last one, by inverting the running sum of the weights in vocabulary order.
//
// Every sum over the vocabulary and every weight is held in 64 bits: the sampled index is where a running sum of up to
// a vocabulary of terms passes u times the total, and with 128256 borders a relative error of 2^-24 in the sums would
// move the choice for about one u in a hundred.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kSumThreads = 256;
constexpr int kBlock = 16 * kSumThreads;  // logits that a CTA of the sums kernel takes at a time
constexpr int kLoops = 4;                 // and how often, where there is work enough for every SM all the same
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kMaxCtas = 16;  // a cluster per request, of 4 to 16 CTAs, or of one
constexpr int kMaxRows = 64;
constexpr int kMaxSlots = 2 * kMaxRows + 1;
constexpr float kMaxTemperature = 1e30f;  // 700 T is a number

struct VerifyArgs {
  int *accepted, *tokens;
  const float *target, *draft;
  long long ldt, ldd;
  const int *drafted, *counts;
  const float *uniforms, *temperature;
  int vocab, batch, rows, slots, loops, chunks;  // slots a request; chunks of loops * kBlock logits a row
  double *sums;              // [batch][slots][chunks]
  unsigned long long *keys;  // the same: order-preserving maximum and its first index
};

// 64-bit key whose unsigned maximum is the first maximum; kBad, the largest, where a value is NaN or +infinity, which
// have no place in a distribution.
constexpr unsigned long long kBad = ~0ull;
__device__ __forceinline__ unsigned long long row_key(float v, unsigned i) {
  unsigned b = v == 0.0f ? 0u : __float_as_uint(v);  // the two zeros are one value
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  unsigned b = (unsigned)(k >> 32);
  b = (b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b;
  return __uint_as_float(b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xFFFFFFFFu - (unsigned)k); }
// A maximum that gives a distribution: above -infinity, and no NaN or +infinity in the row.
__device__ __forceinline__ bool key_good(unsigned long long k) {
  return k != kBad && key_value(k) > __int_as_float(0xff800000);
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

// exp((l - m) / T) for l <= m, to about 2^-43 of itself: 2^(a / 32) with a = (l - m) 32 / (T ln 2) = k + r, |r| <= 1/2,
// as a table value 2^((k mod 32) / 32), the exponent k / 32, and a polynomial for 2^(r / 32) (Tang's table-driven scheme;
// the polynomial is the Taylor sum of degree 5 with its last term economized onto the lower ones by Chebyshev's T5,
// 8e-14 off at most). 0 below `floor`, some 700 T below m. Ten 64-bit operations.
struct Weights {
  const uint2 *table;  // kExpfTable in shared memory
  double k32;          // 32 / (T ln 2)
  // e^-700 of the largest instead of 0 below the floor: what a sum does not see.
  __device__ __forceinline__ double above(float l, float m, float floor) const {
    constexpr double c = 0.021660849392498290, a2 = c * c / 4;  // ln 2 / 32; the square of |r| c's largest value
    constexpr double c4 = c * c * c * c / 24, c3 = c * c * c * (1.0 / 6 + a2 * 5 / 4 / 120), c2 = c * c / 2,
                     c1 = c * (1 - a2 * a2 * 5 / 16 / 120), shift = 0x1.8p+52;
    const double d = (double)fmaxf(l, floor) - (double)m;
    const double t = __fma_rn(d, k32, shift), kd = t - shift, r = __fma_rn(d, k32, -kd);
    const int k = __double2loint(t);
    const uint2 e = table[k & 31];
    const double s = __hiloint2double((int)e.y + (k << 15), (int)e.x);
    const double y = __fma_rn(__fma_rn(__fma_rn(__fma_rn(c4, r, c3), r, c2), r, c1), r, 1.0);
    return y * s;
  }
  __device__ __forceinline__ double operator()(float l, float m, float floor) const {
    const double w = above(l, m, floor);
    return l < floor ? 0.0 : w;
  }
};
// The floor, the smallest float from m - 700 T on: (l - m) / T is in [-700, 0] above it, and finite. (Rounded to the
// nearest it may lie half a step of m lower, which at a small T is far more than the 708 that a 64-bit exponent has room
// for: at m = 20, T = 1e-8 it would be 763.)
__device__ __forceinline__ float floor_of(float m, float t) { return fmaxf(__fmaf_ru(-700.0f, t, m), -FLT_MAX); }
__device__ __forceinline__ double k32_of(float t) { return 46.166241308446829 / (double)t; }  // 32 / ln 2
__device__ __forceinline__ void load_table(uint2 *table) {
  if (threadIdx.x < 32) {
    const unsigned long long e = kExpfTable[threadIdx.x];
    table[threadIdx.x] = make_uint2((unsigned)e, (unsigned)(e >> 32));
  }
}

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

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// One chunk of one row (a.loops blocks of 4096): its maximum and the sum of exp((l - max) / T) over the chunk, or
// (T = 0) its first maximum. A warp keeps a maximum of its own from block to block, to which its lanes' sums refer.
// 64 requests of up to 5 drafts, 128256 tokens: 190 MB in 59 us, 3.3 TB/s; bounded by the weights' instructions, 25 for
// 32 logits with ten of 64 bits among them (issue slots 55 %, the FP64 pipe 45 % busy).
__global__ void __launch_bounds__(kSumThreads, 4) verify_sums_kernel(const VerifyArgs a) {
  __shared__ float max_s[kSumThreads / 32];
  __shared__ double sum_s[kSumThreads / 32];
  __shared__ unsigned first_s[kSumThreads / 32];
  __shared__ uint2 table[32];
  load_table(table);
  pdl_wait();
  pdl_launch_dependents();
  const int chunk = blockIdx.x % a.chunks, id = blockIdx.x / a.chunks;
  const int b = id / a.slots, slot = id - b * a.slots;
  const float t = a.temperature[b];
  const float *row;
  if (!slot_row(a, b, slot, &row))
    return;
  __syncthreads();
  constexpr float kInf = __builtin_inff();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Weights weight{table, t > 0.0f ? k32_of(t) : 0.0};
  float m = -kInf, floor = 0.0f;  // the warp's maximum (the lane's at T = 0)
  unsigned at = 0xFFFFFFFFu;
  double sum = 0.0;
  bool bad = false, deep = false;
  for (int loop = 0; loop < a.loops; loop++) {
    const int first = (chunk * a.loops + loop) * kBlock;
    if (first >= a.vocab)
      break;
    // Sixteen values a thread: four neighbouring ones of each quarter of the block where they lie at 16-byte addresses.
    const bool whole = first + kBlock <= a.vocab && ((uintptr_t)(row + first) & 15) == 0;
    float v[16];
    if (whole) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float4 x = reinterpret_cast<const float4 *>(row + first)[i * kSumThreads + threadIdx.x];
        v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int e = first + i * kSumThreads + threadIdx.x;
        v[i] = e < a.vocab ? row[e] : -kInf;
      }
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < 16; i++)
      top = max_nan(top, v[i]);
    if (!(t > 0.0f)) {
      bad |= !(top < kInf);
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (v[i] > m) {
          m = v[i];
          at = whole ? first + 4 * ((i >> 2) * kSumThreads + (int)threadIdx.x) + (i & 3)
                     : first + i * kSumThreads + (int)threadIdx.x;
        }
      continue;
    }
    top = warp_max_nan(top);
    if (!(top < kInf)) {
      bad = true;
      break;
    }
    if (top > m) {
      floor = floor_of(top, t);
      deep = (double)top - (double)floor >= 600.0 * (double)t;
      if (m > -kInf)
        sum *= weight(m, top, floor);
      m = top;
    }
    if (m == -kInf)
      continue;
    if (deep) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        sum += weight.above(v[i], m, floor);
    } else {  // the floor is rounded to the maximum, or ends at the lowest number
#pragma unroll
      for (int i = 0; i < 16; i++)
        sum += weight(v[i], m, floor);
    }
  }
  float top = bad ? kInf : m;
  top = warp_max_nan(top);
  if (lane == 0)
    max_s[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSumThreads / 32; w++)
    top = fmaxf(top, max_s[w]);
  if (t > 0.0f && top < kInf && m > -kInf)
    sum *= weight(m, top, floor_of(top, t));
  sum = warp_sum(sum);
  at = __reduce_min_sync(0xffffffffu, m == top ? at : 0xFFFFFFFFu);
  if (lane == 0)
    sum_s[warp] = sum, first_s[warp] = at;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < kSumThreads / 32; w++)
      sum += sum_s[w], at = min(at, first_s[w]);
    a.sums[(long long)id * a.chunks + chunk] = sum;
    a.keys[(long long)id * a.chunks + chunk] = top == kInf ? kBad : row_key(top, at);
  }
}

// The weight of token i when the next token is drawn: p_a(i), less q_a(i) at a refused draft (the drafted token alone
// has q = 1 where there are no draft logits).
struct Residual {
  Weights weight;
  const float *p, *q;
  float pm, qm, p_floor, q_floor;
  double p_norm, q_norm;
  int without;
  __device__ __forceinline__ double of(float pl, float ql) const {
    // Both products are rounded (no fused multiply-add): where draft and target are the same row nothing is left.
    double w = __dmul_rn(weight(pl, pm, p_floor), p_norm);
    if (q)
      w -= __dmul_rn(weight(ql, qm, q_floor), q_norm);
    return fmax(w, 0.0);
  }
  __device__ __forceinline__ double operator()(int i) const {
    return i == without ? 0.0 : of(p[i], q ? q[i] : 0.0f);
  }
};

// The whole CTA: the first token of [s0, s1) whose running sum, `run` before s0, passes `place`; the last one with
// weight where rounding leaves none. Every thread a run of neighbouring tokens.
struct Invert {
  double warp_sums[kPickWarps];
  int first, last;
};
__device__ int invert(const Residual &w, Invert *t, int s0, int s1, double run, double place) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (s1 - s0 + kPickThreads - 1) / kPickThreads;
  const int i0 = min(s0 + (int)threadIdx.x * per, s1), i1 = min(i0 + per, s1);
  double mine = 0.0;
#pragma unroll 4
  for (int i = i0; i < i1; i++)
    mine += w(i);
  double upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o)
      upto += other;
  }
  if (lane == 31)
    t->warp_sums[warp] = upto;
  if (threadIdx.x == 0)
    t->first = kPickThreads, t->last = -1;
  __syncthreads();
  for (int i = 0; i < warp; i++)
    run += t->warp_sums[i];
  upto += run;
  if (mine > 0.0) {
    if (upto > place)
      atomicMin(&t->first, (int)threadIdx.x);
    atomicMax(&t->last, (int)threadIdx.x);
  }
  __syncthreads();
  if ((int)threadIdx.x != (t->first < kPickThreads ? t->first : t->last))
    return -1;
  run = upto - mine;
  int at = -1;
  for (int i = i0; i < i1; i++) {
    const double x = w(i);
    if (x > 0.0) {
      at = i;
      run += x;
      if (run > place)
        break;
    }
  }
  return at;
}

// A cluster per request: every CTA decides which drafts are accepted. Where the weights are p alone the chunks' sums are
// known, and one CTA inverts one chunk; else every CTA sums its slice of the vocabulary's weights, and the CTA whose
// slice holds the place of u inverts the part of it that a warp summed. Eight round trips to memory or the cluster one
// after another bound it (8.7 us for one request), at large batches the residuals' weights too (64 requests: 30 us).
__global__ void __launch_bounds__(kPickThreads, 2) verify_pick_kernel(const VerifyArgs a) {
  __shared__ unsigned long long key_s[kMaxSlots];
  __shared__ uint2 table[32];
  __shared__ double sum_s[kMaxSlots], warp_sums[kPickWarps], slices[kMaxCtas];
  __shared__ Invert inv;
  __shared__ int stop_s, found_s, drafted_s[kMaxRows];
  cg::cluster_group cluster = cg::this_cluster();
  load_table(table);
  pdl_wait();
  pdl_launch_dependents();
  const int ctas = cluster.num_blocks(), b = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // What does not depend on one another is on its way at once: the drafts, the first chunks of this warp's first slot
  // (whether they count shows later), the request's numbers.
  const int j = threadIdx.x;
  const int drafted = j < a.rows ? a.drafted[(long long)b * a.rows + j] : -1;
  const long long base = (long long)b * a.slots * a.chunks;
  const long long first_at = base + (long long)warp * a.chunks + lane;
  const bool have_first = warp < a.slots && lane < a.chunks;
  const unsigned long long first_key = have_first ? a.keys[first_at] : 0;
  const double first_sum = have_first ? a.sums[first_at] : 0.0;
  const int count = count_of(a, b);
  const float t = a.temperature[b];
  const bool greedy = t == 0.0f;
  const bool valid = count >= 0 && count <= a.rows && t >= 0.0f && t <= kMaxTemperature;
  // This thread's draft, and its logits.
  const bool drafts = valid && j < count;
  const int x = drafts ? drafted : -1;
  const bool x_good = x >= 0 && x < a.vocab;
  float px = 0.0f, qx = 0.0f, u = 0.0f;
  if (drafts && x_good && !greedy) {
    px = a.target[((long long)b * (a.rows + 1) + j) * a.ldt + x];
    qx = a.draft ? a.draft[((long long)b * a.rows + j) * a.ldd + x] : 0.0f;
    u = a.uniforms[(long long)b * (a.rows + 1) + j];
  }
  const float u_last = a.uniforms[(long long)b * (a.rows + 1) + a.rows];
  if (threadIdx.x == 0)
    stop_s = valid ? count : 0;
  if (j < a.rows)
    drafted_s[j] = drafted;
  cluster.sync();  // every CTA has started before any writes into another's shared memory; the table is there
  if (count == -1)
    return;  // the whole cluster: a slot of the batch that is not in use
  const Weights weight{table, greedy ? 0.0 : k32_of(t)};
  int *tokens = a.tokens + (long long)b * (a.rows + 1);
  if (valid)
    for (int slot = warp; slot < a.slots; slot += kPickWarps) {
      const float *row;
      if (!slot_row(a, b, slot, &row))
        continue;
      const long long at = base + (long long)slot * a.chunks;
      const bool ahead = slot == warp;
      unsigned long long key = ahead ? first_key : lane < a.chunks ? a.keys[at + lane] : 0;
      const unsigned long long key0 = key;
      for (int c = lane + 32; c < a.chunks; c += 32)
        key = max64(key, a.keys[at + c]);
      key = warp_max(key);
      double sum = 0.0;
      if (!greedy && key_good(key))
        for (int c = lane; c < a.chunks; c += 32) {
          const unsigned long long k = c == lane ? key0 : a.keys[at + c];
          if (key_good(k))
            sum += (ahead && c == lane ? first_sum : a.sums[at + c]) *
                   weight(key_value(k), key_value(key), floor_of(key_value(key), t));
        }
      sum = warp_sum(sum);
      if (lane == 0)
        key_s[slot] = key, sum_s[slot] = sum;
    }
  __syncthreads();
  // A draft is refused, or its rows have no distribution: the first such place ends the run.
  if (drafts) {
    const int dj = a.rows + 1 + j;
    bool good = false;
    if (x_good && key_good(key_s[j]) && (greedy || !a.draft || key_good(key_s[dj]))) {
      if (greedy) {
        good = key_index(key_s[j]) == x;
      } else {
        const float pm = key_value(key_s[j]), qm = a.draft ? key_value(key_s[dj]) : 0.0f;
        const double p = weight(px, pm, floor_of(pm, t)) / sum_s[j];
        const double q = a.draft ? weight(qx, qm, floor_of(qm, t)) / sum_s[dj] : 1.0;
        good = (double)u * q < p;
      }
    }
    if (!good)
      atomicMin(&stop_s, j);
  }
  __syncthreads();
  const int stop = stop_s;
  const bool refused = stop < count;
  const int at_stop = valid && refused ? drafted_s[stop] : -1;
  // No distribution at the place where the run ends (or arguments that mean nothing): no answer.
  unsigned error = 0;
  if (!valid || (refused && (at_stop < 0 || at_stop >= a.vocab)))
    error = KC_ERR_BAD_ARGS;
  else if (!key_good(key_s[stop]) || (refused && !greedy && a.draft && !key_good(key_s[a.rows + 1 + stop])))
    error = KC_ERR_NONFINITE;
  if (rank == 0) {
    if (j <= a.rows) {
      if (error || j > stop)
        tokens[j] = -1;
      else if (j < stop)
        tokens[j] = x;
    }
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
  w.weight = weight;
  w.p = a.target + ((long long)b * (a.rows + 1) + stop) * a.ldt;
  w.pm = key_value(key_s[stop]), w.p_norm = 1.0 / sum_s[stop];
  w.q = refused && a.draft ? a.draft + ((long long)b * a.rows + stop) * a.ldd : nullptr;
  w.qm = w.q ? key_value(key_s[a.rows + 1 + stop]) : 0.0f, w.q_norm = w.q ? 1.0 / sum_s[a.rows + 1 + stop] : 0.0;
  w.p_floor = floor_of(w.pm, t), w.q_floor = floor_of(w.qm, t);
  w.without = refused && !a.draft ? at_stop : -1;
  int s0 = 0, s1 = 0;
  double before = 0.0, total = 0.0, place = 0.0;
  // The weights of the warps' segments (of `segment` tokens) of [first, last), eight reads of both rows under way a lane.
  auto segments = [&](int first, int last, int segment) {
    const int w0 = min(first + warp * segment, last), w1 = min(w0 + segment, last);
    double sum = 0.0;
    for (int i0 = w0 + lane; i0 < w1; i0 += 256) {
      float p[8], q[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int i = i0 + 32 * k;
        p[k] = i < w1 && i != w.without ? w.p[i] : __int_as_float(0xff800000);
        q[k] = i < w1 && w.q ? w.q[i] : __int_as_float(0xff800000);
      }
#pragma unroll
      for (int k = 0; k < 8; k++)
        sum += w.of(p[k], q[k]);
    }
    sum = warp_sum(sum);
    if (lane == 0)
      warp_sums[warp] = sum;
    __syncthreads();
  };
  // The segment that the place falls into; behind the last one with weight, that one.
  auto narrow = [&](int first, int last, int segment) {
    int seg = 0;
    bool some = false;
    double run = before;
    for (int i = 0; i < kPickWarps; i++) {
      if (warp_sums[i] > 0.0 && (!some || place >= run)) {
        seg = i;
        before = run;
        some = true;
      }
      run += warp_sums[i];
    }
    s0 = min(first + seg * segment, last), s1 = min(s0 + segment, last);
  };
  auto place_in = [&]() {
    place = (double)u_last * total;
    if (!(place < total))
      place = total * (1.0 - 0x1p-52);
    place = fmax(place, 0.0);
  };
  if (!w.q) {
    if (rank)
      return;
    // p alone: the chunks' sums; the refused token's chunk is summed again without it (a difference would leave rounding
    // where nothing is left).
    const long long at = base + (long long)stop * a.chunks;
    const int length = a.loops * kBlock, again = w.without >= 0 ? w.without / length : -1;
    if (again >= 0) {
      const int first = again * length;
      segments(first, min(first + length, a.vocab), length / kPickWarps);
    }
    auto chunk = [&](int c) {
      if (c == again) {
        double sum = 0.0;
        for (int i = 0; i < kPickWarps; i++)
          sum += warp_sums[i];
        return sum;
      }
      const unsigned long long k = a.keys[at + c];
      return key_good(k) ? a.sums[at + c] * weight(key_value(k), w.pm, w.p_floor) * w.p_norm : 0.0;
    };
    if (warp == 0) {
      double upto = 0.0;
      for (int c0 = 0; c0 < a.chunks; c0 += 32)
        upto += warp_sum(c0 + lane < a.chunks ? chunk(c0 + lane) : 0.0);
      total = upto;
      place_in();
      // The chunk whose running sum passes the place; behind the last one with weight, that one.
      int found = -1;
      double run = 0.0, at_found = 0.0;
      for (int c0 = 0; c0 < a.chunks; c0 += 32) {
        const double mine = c0 + lane < a.chunks ? chunk(c0 + lane) : 0.0;
        double sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double other = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o)
            sum += other;
        }
        const unsigned past = __ballot_sync(0xffffffffu, mine > 0.0 && run + sum > place);
        const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
        if (past || some) {
          const int l = past ? __ffs(past) - 1 : 31 - __clz(some);
          found = c0 + l;
          at_found = run + __shfl_sync(0xffffffffu, sum - mine, l);
        }
        if (past)
          break;
        run += __shfl_sync(0xffffffffu, sum, 31);
      }
      if (lane == 0)
        slices[0] = total, slices[1] = place, slices[2] = at_found, found_s = found;
    }
    __syncthreads();
    total = slices[0], place = slices[1], before = slices[2];
    const int first = max(found_s, 0) * length, last = min(first + length, a.vocab);
    segments(first, last, length / kPickWarps);
    narrow(first, last, length / kPickWarps);
  } else {
    const int segment = (a.vocab + ctas * kPickWarps - 1) / (ctas * kPickWarps);
    const int first = min(rank * kPickWarps * segment, a.vocab), last = min(first + kPickWarps * segment, a.vocab);
    segments(first, last, segment);
    if ((int)threadIdx.x < ctas) {
      double slice = 0.0;
      for (int i = 0; i < kPickWarps; i++)
        slice += warp_sums[i];
      *cluster.map_shared_rank(&slices[rank], threadIdx.x) = slice;
    }
    cluster.sync();
    for (int r = 0; r < ctas; r++) {
      if (r == rank)
        before = total;
      total += slices[r];
    }
    place_in();
    if (total > 0.0 && (place < before || place >= before + slices[rank]))  // the slices tile [0, total): one CTA goes on
      return;
    narrow(first, last, segment);
  }
  if (!(total > 0.0)) {  // nothing of the target is left but rounding: its first maximum
    if (rank)
      return;
    __syncthreads();
    if (threadIdx.x == 0)
      found_s = a.vocab;
    __syncthreads();
    for (int i = threadIdx.x; i < a.vocab; i += kPickThreads)
      if (w.p[i] == w.pm) {
        atomicMin(&found_s, i);
        break;
      }
    __syncthreads();
    if (threadIdx.x == 0)
      tokens[stop] = found_s;
    return;
  }
  const int token = invert(w, &inv, s0, s1, before, place);
  if (token >= 0)
    tokens[stop] = token;
}

size_t verify_blocks(int vocab) { return ((size_t)vocab + kBlock - 1) / kBlock; }

}  // namespace

extern "C" {

size_t k_verify_bytes(int vocab, int batch, int rows) {
  if (vocab <= 0 || batch <= 0 || rows < 0 || rows > kMaxRows)
    return 0;
  return (size_t)batch * (2 * rows + 1) * verify_blocks(vocab) * (sizeof(double) + sizeof(unsigned long long));
}

void k_verify_draft(int *accepted, int *tokens, const float *target, size_t ldt, const float *draft, size_t ldd,
                    const int *drafted, const int *counts, const float *uniforms, const float *temperature, int vocab,
                    int batch, int rows, void *work) {
  const char *name = "k_verify_draft";
  if (vocab <= 0 || vocab > (1 << 30) || batch < 0 || rows < 0 || rows > kMaxRows || ldt < (size_t)vocab ||
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
  const int slots = draft && rows ? 2 * rows + 1 : rows + 1;
  size_t blocks = verify_blocks(vocab), pairs = (size_t)batch * slots * blocks;
  if (pairs > 0x7fffffffu || (size_t)batch * kMaxCtas > 0x7fffffffu) {
    kc_fail("%s: batch %d of %d rows is too large", name, batch, rows);
    return;
  }
  VerifyArgs a;
  a.accepted = accepted, a.tokens = tokens, a.target = target, a.draft = rows ? draft : nullptr;
  a.ldt = (long long)ldt, a.ldd = (long long)ldd, a.drafted = drafted, a.counts = counts;
  a.uniforms = uniforms, a.temperature = temperature, a.vocab = vocab, a.batch = batch, a.rows = rows;
  // Longer chunks amortize a CTA's start and end, as long as those that find work (half of the drafts, say) fill the SMs
  // four times over at four CTAs each: 64 requests of 5 drafts, 128256 tokens, 92 us with one block and 59 with four.
  const size_t busy = (size_t)batch * (rows / 2 + 1 + (slots > rows + 1 ? rows / 2 : 0)) * blocks;
  a.loops = 1;
  while (a.loops < kLoops && busy / (2 * a.loops) >= (size_t)16 * kc_device_sms())
    a.loops *= 2;
  a.slots = slots;
  a.chunks = (int)((blocks + a.loops - 1) / a.loops);
  pairs = (size_t)batch * slots * a.chunks;
  a.sums = static_cast<double *>(work);
  a.keys = reinterpret_cast<unsigned long long *>(a.sums + pairs);
  cudaError_t e =
      kc_launch_pdl(verify_sums_kernel, dim3((unsigned)pairs), dim3(kSumThreads), 0, kc_stream(), a);
  if (e == cudaSuccess) {
    kc_count_launch();
    // With draft logits the largest clusters that run in about two waves of two CTAs per SM (greedy requests and accepted
    // drafts leave early): a request's rows are read by more SMs at once. Without, one CTA inverts one chunk (24 requests
    // of 7 drafts: 13 us with one CTA a request, 16 with sixteen).
    int ctas = a.draft ? kMaxCtas : 1;
    while (ctas > 4 && (long long)ctas * batch > 4 * kc_device_sms())
      ctas /= 2;
    e = kc_allow_clusters(reinterpret_cast<const void *>(verify_pick_kernel));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)batch * ctas);
    cfg.blockDim = dim3(kPickThreads);
    cfg.stream = kc_stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = kc_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (e == cudaSuccess)
      e = cudaLaunchKernelEx(&cfg, verify_pick_kernel, a);
    if (e == cudaSuccess)
      kc_count_launch();
  }
  if (e != cudaSuccess)
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
