// Log probabilities of tokens, the entropy of their distribution and its likeliest tokens, from rows of logits
// (k_token_logprobs). With M the row's maximum, taken once out of the sums, S = sum e^(x - M) and T = sum e^(x - M) (M - x)
// over the rest: log p_i = (x_i - M) - log(1 + S), entropy = log(1 + S) + T / (1 + S). Both sums have terms of one sign and
// neither is rounded against the 1, so that the small logarithm of a nearly certain token keeps its digits.
//
// The logits are read once. A CTA takes a row, or with few rows a part of one (a cluster joins them), as a stream of 16 KiB
// stages by bulk copies, through a ring that runs on into the next row; the ends of a row that does not begin and end at 16
// bytes come by their elements, so that nothing outside it is read. Each thread keeps the sums of its elements relative to
// a reference near their maximum, and that maximum with its place. At the end of the row the likeliest tokens are found by
// way of the threads' maxima: with the threads in 64 classes, every one of the top k elements is at or above the k-th largest
// class maximum, which about as many threads reach as there are tokens to find; only their elements, at a fixed stride,
// are read again (from L2).
// What bounds it: many rows, memory: 2048 rows of 128256 180 us in a graph of calls, 5.8 TB/s, with 10 us for the last rows'
// ends (193 call by call from Python); few rows the chain of a row's end, 6 us, a part's stream (12 us for 128256 logits
// by one CTA) and a cluster's two barriers, 2 us: 64 rows of 128256 with 20 alternatives 18.1 us in a graph, 18.7 call by call.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"
#include "tcgen05.cuh"
#include "units.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;  // that take logits; one more warp issues the copies
constexpr int kCtas = 3;               // to an SM: one's end of a row runs under the others' streams
constexpr int kMaxTop = 32;
constexpr int kHalf = 2 * kThreads;    // 16-byte units to a step: two neighbouring ones to a thread
constexpr int kUnits = 2 * kHalf;      // and to a stage
constexpr int kStages = 4;
constexpr int kClasses = 64;
constexpr int kCandidates = 512;
constexpr int kLooks = 2;  // (four at once took 0.4 us longer a row, eight 2: instructions that run once a row come from far)
constexpr int kMaxParts = 8;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kRise = 3.0f;   // how far a logit may lie above a thread's reference before the reference moves
constexpr float kLeast = -150.0f;  // e^-150 is 0 in fp32: a difference below it (-infinity) is taken for it

struct LogprobArgs {
  float *logprobs, *entropy;
  int *top_tokens;
  float *top_logprobs;
  const float *logits;
  size_t ld;
  const int *tokens;
  int vocab, rows, top;
};

// Order-preserving bits of a logit, then the inverted index: the larger key is the likelier token, the lower of equals.
// -0 and +0 are equal numbers.
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  unsigned b = __float_as_uint(x + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (unsigned)(0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float logit_of(unsigned long long key) {
  const unsigned b = (unsigned)(key >> 32);
  return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}

// What a part of a row gives: its maximum, the sums of the rest relative to it, and its top tokens in order (0: none).
struct Part {
  float max, s, t;
  int wrong;
  unsigned long long top[kMaxTop];
};

struct State {
  uint64_t full[kStages], empty[kStages];
  Part part;
  unsigned long long keys[kThreads], least, best;  // the threads' maxima; the k-th largest class maximum, the largest
  unsigned long long candidates[kCandidates];
  unsigned long long merged[kMaxParts * kMaxTop];
  __align__(16) float edges[8];  // the elements of a part's first and last unit
  float sums[2][kWarps], again[2];  // the warps' sums; the sums of the thread that has the maximum, without it
  int marked, found, wrong, verdict, owner;
  unsigned short who[kThreads];  // threads whose maximum may be a top one
};
constexpr int kRing = kStages * kUnits * 16;
constexpr int kSmem = kRing + (int)sizeof(State);

// The larger of numbers and the first of equals: order of values, then of pairs of units.
__device__ __forceinline__ unsigned long long pair_key(float x, unsigned pair) { return key_of(x, (int)pair); }

// Element i of a unit that is not whole, -infinity where it is not the row's.
__device__ __forceinline__ float edge_element(const UnitRow &r, int unit, int i) {
  const int at = element_of(r, unit, i);
  return at >= 0 ? __ldcg(r.data + at) : -INFINITY;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

// The weight e^d of a difference and its product with it.
__device__ __forceinline__ void weigh(float d, float &s, float &t) {
  d = fmaxf(d, kLeast);
  const float w = ex2(d * kLog2e);
  s += w;
  t = fmaf(w, d, t);
}

// A thread's running results: the maximum and the pair of units it first came in, and the sums s of e^(x - ref) and t of
// e^(x - ref) (x - ref) over its elements, in four chains.
struct Running {
  float max, ref;
  unsigned pair;
  uint64_t s[2], t[2];
};
// Two steps' elements: of the pairs `pair` and `pair` + kThreads.
__device__ __forceinline__ void take(Running &r, const float (&x)[2][8], unsigned pair, bool *wrong) {
  float top[2];
#pragma unroll
  for (int h = 0; h < 2; h++)
    top[h] = max3(max3(x[h][0], x[h][1], x[h][2]), max3(x[h][3], x[h][4], x[h][5]), fmax_nan(x[h][6], x[h][7]));
  const float high = fmax_nan(top[0], top[1]);
  *wrong |= !(high < INFINITY);
  if (high > r.max) {
    r.pair = top[0] == high ? pair : pair + kThreads;
    r.max = high;
  }
  if (high > r.ref + kRise) {
    const float by = fmaxf(r.ref - high, kLeast), f = ex2(by * kLog2e);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      r.t[i] = f2_mul(f2_fma(f2_pack(by, by), r.s[i], r.t[i]), f2_pack(f, f));
      r.s[i] = f2_mul(r.s[i], f2_pack(f, f));
    }
    r.ref = high;
  }
  const uint64_t ref = f2_pack(-r.ref, -r.ref), scale = f2_pack(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float *at = &x[i >> 2][2 * (i & 3)];
    float d0, d1;
    f2_unpack(f2_add(f2_pack(at[0], at[1]), ref), d0, d1);
    const uint64_t d = f2_pack(fmaxf(d0, kLeast), fmaxf(d1, kLeast));
    float e0, e1;
    f2_unpack(f2_mul(d, scale), e0, e1);
    const uint64_t w = f2_pack(ex2(e0), ex2(e1));
    r.s[i & 1] = f2_add(r.s[i & 1], w);
    r.t[i & 1] = f2_fma(w, d, r.t[i & 1]);
  }
}

// x - max - log_s, rounded once.
__device__ __forceinline__ float log_p(float x, float max, float log_s) {
  return (float)(((double)x - (double)max) - (double)log_s);
}

// A CTA per row, or a cluster of `parts`; each takes rows in turn.
__global__ void __launch_bounds__(kThreads + 32, kCtas) logprobs_kernel(const LogprobArgs a, int parts) {
  extern __shared__ __align__(128) uint8_t smem[];
  State *t = reinterpret_cast<State *>(smem + kRing);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = blockIdx.x % parts, stride = gridDim.x / parts;  // parts > 1: a row to a cluster, and no more
  cg::cluster_group cluster = cg::this_cluster();
  if (tid == 0) {
    for (int i = 0; i < kStages; i++) {
      mbar_init(&t->full[i], 1);
      mbar_init(&t->empty[i], kWarps);
    }
    t->marked = t->found = t->wrong = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  if (parts > 1 && a.tokens && a.tokens[blockIdx.x / parts] == -1)
    return;  // the whole cluster
  int stage = 0;
  unsigned parity = 0;

  if (warp == kWarps) {
    // ---- copies ----
    bool ok = true;
    unsigned fills = 0;  // of the ring's stages
    for (int row = blockIdx.x / parts; ok && row < a.rows; row += stride) {
      if (a.tokens && a.tokens[row] == -1)
        continue;
      const UnitRow r = unit_row(a.logits + (size_t)row * a.ld, a.vocab);
      int first, end, whole0, whole1;
      part_of(r, part, parts, &first, &end);
      whole_of(r, first, end, &whole0, &whole1);
      // The part's first and last unit where not all of them are the row's: an element each of lanes 0 to 3 and 4 to 7.
      const float edge = lane < 8 ? edge_element(r, lane < 4 ? first : end - 1, lane & 3) : 0.0f;
      for (int u = first; ok && u < end; u += kUnits) {
        const int upto = min(u + kUnits, end), from = max(u, whole0), to = min(upto, whole1);
        float4 *const slot = reinterpret_cast<float4 *>(smem + stage * kUnits * 16);
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&t->empty[stage], parity ^ 1));
        if (!ok)
          break;
        if (lane == 0 && from < to) {
          mbar_expect_tx(&t->full[stage], 16u * (unsigned)(to - from));
          bulk_g2s(slot + (from - u), unit_at(r, from), 16u * (unsigned)(to - from), &t->full[stage]);
        }
        if (to - from < upto - u) {
          if (lane < 4 ? from > u : lane < 8 && to < upto)
            reinterpret_cast<float *>(slot + (lane < 4 ? 0 : to - u))[lane & 3] = edge;
          fence_proxy_async_smem();  // before a later copy's writes
          __syncwarp();
        }
        if (lane == 0)
          mbar_arrive(&t->full[stage]);
        fills++;
        if (++stage == kStages)
          stage = 0, parity ^= 1;
      }
    }
    // No copy is under way when the CTA ends, also where a wait, here or of those who take the logits, has run out.
#pragma unroll 1
    for (unsigned i = fills > kStages ? fills - kStages : 0; i < fills; i++)
      mbar_wait_sleep_bounded(&t->full[i % kStages], (i / kStages) & 1);
    __syncwarp();
  } else {
    bool ok = true;  // no wait has run out
    for (int row = blockIdx.x / parts; row < a.rows; row += stride) {
      const int token = a.tokens ? a.tokens[row] : 0;
      if (token == -1)
        continue;
      const UnitRow r = unit_row(a.logits + (size_t)row * a.ld, a.vocab);
      int first, end;
      part_of(r, part, parts, &first, &end);
      Running mine;
      mine.max = -INFINITY, mine.ref = -3.402823466e+38f, mine.pair = tid;
      mine.s[0] = mine.s[1] = mine.t[0] = mine.t[1] = 0;
      bool wrong = token < 0 || token >= a.vocab;
      const float given = tid == 0 && part == 0 && !wrong ? __ldcg(a.logits + (size_t)row * a.ld + token) : 0.0f;
      // The part's first and last unit once more, for the second look: an element a thread.
      const float edge_value = tid < 8 ? edge_element(r, tid < 4 ? first : end - 1, tid & 3) : 0.0f;
      for (int u = first; u < end; u += kUnits) {
        ok = ok && mbar_wait_bounded(&t->full[stage], parity);
        // The two units in an order that keeps eight lanes in different banks.
        const int swap = tid >> 2 & 1;
        const float4 *from = reinterpret_cast<const float4 *>(smem + stage * kUnits * 16) + 2 * tid;
        float x[2][8];
#pragma unroll
        for (int h = 0; h < 4; h++) {
          const float4 y = from[(h >> 1) * kHalf + ((h & 1) ^ swap)];
          float *to = &x[h >> 1][4 * (h & 1)];
          to[0] = y.x, to[1] = y.y, to[2] = y.z, to[3] = y.w;
        }
        if (u + kUnits > end)  // the part's last stage, which others' units follow
#pragma unroll
          for (int h = 0; h < 4; h++)
            if (u + 2 * tid + (h >> 1) * kHalf + ((h & 1) ^ swap) >= end)
#pragma unroll
              for (int i = 0; i < 4; i++)
                x[h >> 1][4 * (h & 1) + i] = -INFINITY;
        take(mine, x, (unsigned)((u - first) / 2 + tid), &wrong);
        // The stage is given back only now, behind the fence between this warp's reads and the next copy's writes: before it,
        // loads still under way read what the copy brought (one row in a hundred wrong at 2048 rows of 128256).
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&t->empty[stage]);
        if (++stage == kStages)
          stage = 0, parity ^= 1;
      }
      wrong |= !ok;
      // ---- the end of the part: the maximum, and the class maximum that holds the top ones ----
      const unsigned long long key = first + 2 * tid < end ? pair_key(mine.max, mine.pair) : 0;
      t->keys[tid] = key;
      if (tid < 8)
        t->edges[tid] = edge_value;
      if (wrong)
        t->wrong = 1;
      meet();
      const int wanted = a.top > 1 ? a.top : 1;
      if (warp < 2) {
        unsigned long long k = t->keys[tid];
        for (int i = 1; i < kThreads / kClasses; i++)
          k = max_key(k, t->keys[tid + i * kClasses]);
        t->merged[tid] = k;
        asm volatile("bar.sync 2, 64;" ::: "memory");
        int before = 0;
        for (int i = 0; i < kClasses; i++)
          before += t->merged[i] > k || (t->merged[i] == k && i < tid);
        if (before == 0)
          t->best = k;
        if (before == wanted - 1)
          t->least = k;  // 0 where fewer classes have any
      }
      meet();
      const unsigned long long best = t->best, least = t->least;
      const float top = logit_of(best);
      const bool bad = t->wrong != 0;
      if (key != 0 && key >= least)
        t->who[atomicAdd(&t->marked, 1)] = (unsigned short)tid;
      if (key == best)
        t->owner = tid;  // the one of them that has the maximum (or any, where there is none)
      // ---- the sums, relative to the maximum; the thread that has it leaves its own to the second look ----
      float s, e;
      {
        float s0, s1, s2, s3, t0, t1, t2, t3;
        f2_unpack(mine.s[0], s0, s1), f2_unpack(mine.s[1], s2, s3);
        f2_unpack(mine.t[0], t0, t1), f2_unpack(mine.t[1], t2, t3);
        const float by = fmaxf(mine.ref - top, kLeast), f = ex2(by * kLog2e);
        s = (s0 + s1) + (s2 + s3);
        e = fmaf(by, s, (t0 + t1) + (t2 + t3)) * f;
        s *= f;
        if (key == best || key == 0 || top == -INFINITY)
          s = e = 0.0f;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, o), e += __shfl_xor_sync(0xffffffffu, e, o);
      if (lane == 0)
        t->sums[0][warp] = s, t->sums[1][warp] = e;
      meet();
      // ---- the second look at the marked threads' units: 16 of a thread's pairs, a unit a lane, kLooks times at once. The
      // first warp looks at the thread that has the maximum, and sums the rest of it up again. ----
      const int marked = bad ? 0 : t->marked;
      const int each = (end - first + 2 * 16 * kThreads - 1) / (2 * 16 * kThreads);  // looks at a thread's pairs
      const int looks = warp == 0 ? (marked ? each : 0) : marked * each;
      int whole0, whole1;  // the part's whole units
      whole_of(r, first, end, &whole0, &whole1);
      const unsigned best_pair = 0xffffffffu - (unsigned)best;
      const float edge = least ? logit_of(least) : -INFINITY;
      float s2 = 0.0f, e2 = 0.0f;
      for (int i0 = warp == 0 ? 0 : warp - 1; i0 < looks; i0 += warp == 0 ? kLooks : kLooks * (kWarps - 1)) {
        float4 y[kLooks];
        int pair[kLooks];
        bool in[kLooks];
#pragma unroll
        for (int k = 0; k < kLooks; k++) {
          const int i = i0 + k * (warp == 0 ? 1 : kWarps - 1), who = warp == 0 ? t->owner : t->who[min(i, looks - 1) / each];
          const int look = warp == 0 ? i : i % each;
          pair[k] = look * 16 * kThreads + who + (lane >> 1) * kThreads;
          const int unit = first + 2 * pair[k] + (lane & 1);
          in[k] = i < looks && unit >= whole0 && unit < whole1 && (warp == 0 || who != t->owner);
          y[k] = in[k] ? __ldcg(reinterpret_cast<const float4 *>(unit_at(r, unit))) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < kLooks; k++) {
          const int unit = first + 2 * pair[k] + (lane & 1);
          float x[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
          if (in[k] && fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= edge) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int at = element_of(r, unit, j);
              if (at >= 0 && pair_key(x[j], (unsigned)pair[k]) >= least) {
                const int n = atomicAdd(&t->found, 1);
                if (n < kCandidates)
                  t->candidates[n] = key_of(x[j], at);
              }
            }
          }
          if (warp == 0) {
            // The maximum is left out once: in the pair that it first came in, the first of it. (What is not the row's is
            // -infinity, and adds nothing.)
            if (!in[k]) {
              x[0] = x[1] = x[2] = x[3] = -INFINITY;
              if (i0 + k < looks && unit < end)  // an edge
#pragma unroll
                for (int j = 0; j < 4; j++)
                  x[j] = t->edges[(unit < whole0 ? 0 : 4) + j];
            }
            const bool has = (unsigned)pair[k] == best_pair && fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) == top;
            const unsigned holders = __ballot_sync(0xffffffffu, has);
            bool out = has && lane == __ffs(holders) - 1;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              if (out && x[j] == top)
                x[j] = -INFINITY, out = false;
              weigh(x[j] - top, s2, e2);
            }
          }
        }
      }
      // The edges' elements, which threads 0 to 7 have.
      if (!bad && (tid < 4 ? first < whole0 : tid < 8 && whole1 < end)) {
        const int unit = tid < 4 ? first : end - 1, at = element_of(r, unit, tid & 3);
        if (at >= 0 && pair_key(edge_value, (unsigned)(unit - first) / 2) >= least) {
          const int n = atomicAdd(&t->found, 1);
          if (n < kCandidates)
            t->candidates[n] = key_of(edge_value, at);
        }
      }
      if (warp == 0) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
          s2 += __shfl_xor_sync(0xffffffffu, s2, o), e2 += __shfl_xor_sync(0xffffffffu, e2, o);
        if (lane == 0)
          t->again[0] = s2, t->again[1] = e2;
      }
      meet();
      // ---- the top ones in order ----
      const int found = t->found;
      if (tid < kMaxTop)
        t->part.top[tid] = 0;
      if (tid == 0) {
        const bool some = top > -INFINITY;
        float s2 = some && !bad ? t->again[0] : 0.0f, e2 = some && !bad ? t->again[1] : 0.0f;
        for (int w = 0; w < kWarps; w++)
          s2 += t->sums[0][w], e2 += t->sums[1][w];
        t->part.max = some ? top : -INFINITY, t->part.s = s2, t->part.t = -e2;
        t->part.wrong = bad;
      }
      meet();
      if (tid == 0)
        t->marked = t->found = t->wrong = 0;  // everybody has read them
      if (!bad && found <= kCandidates) {
        for (int i = tid; i < found; i += kThreads) {
          const unsigned long long k = t->candidates[i];
          int before = 0;
          for (int j = 0; j < found; j++)
            before += t->candidates[j] > k;
          if (before < wanted)
            t->part.top[before] = k;
        }
      } else if (!bad) {
        // More elements above the classes' maximum than there is room for: one token after another, from the logits.
        unsigned long long last = ~0ull;
        for (int n = 0; n < wanted; n++) {
          unsigned long long k = 0;
          for (int unit = first + tid; unit < end; unit += kThreads) {
            const float4 y = unit >= whole0 && unit < whole1
                                 ? __ldcg(reinterpret_cast<const float4 *>(unit_at(r, unit)))
                                 : *reinterpret_cast<const float4 *>(t->edges + (unit < whole0 ? 0 : 4));
            const float x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int at = element_of(r, unit, i);
              if (at >= 0) {
                const unsigned long long other = key_of(x[i], at);
                k = other < last ? max_key(k, other) : k;
              }
            }
          }
#pragma unroll
          for (int o = 16; o; o >>= 1)
            k = max_key(k, __shfl_xor_sync(0xffffffffu, k, o));
          meet();
          if (lane == 0)
            t->merged[warp] = k;
          meet();
          for (int w = 0; w < kWarps; w++)
            k = max_key(k, t->merged[w]);
          if (tid == 0)
            t->part.top[n] = k;
          last = k;
        }
      }
      // ---- the parts' results joined by the first of them ----
      if (parts > 1)
        cluster.sync();
      else
        meet();
      if (part == 0) {
        const int keys = parts * kMaxTop;
        if (parts > 1 && tid < keys)
          t->merged[tid] = cluster.map_shared_rank(&t->part, tid / kMaxTop)->top[tid % kMaxTop];
        if (tid == 0) {
          float max = -INFINITY, s3 = 0.0f, e3 = 0.0f, m[kMaxParts], n[kMaxParts], e2[kMaxParts];
          bool any_wrong = false;
          int of = 0;
#pragma unroll
          for (int i = 0; i < kMaxParts; i++) {
            const Part *from = i == 0 || i >= parts ? &t->part : cluster.map_shared_rank(&t->part, i);
            m[i] = i < parts ? from->max : -INFINITY, n[i] = from->s, e2[i] = from->t;
            any_wrong |= from->wrong != 0;
            if (m[i] > max)
              max = m[i], of = i;
          }
#pragma unroll
          for (int i = 0; i < kMaxParts; i++) {
            if (m[i] == -INFINITY)
              continue;
            const float by = m[i] - max, f = ex2(fmaxf(by, kLeast) * kLog2e);
            if (i != of)
              n[i] += 1.0f;  // another part's maximum is one of the rest
            if (f > 0.0f)
              s3 = fmaf(n[i], f, s3), e3 = fmaf(fmaf(-by, n[i], e2[i]), f, e3);
          }
          const bool w = any_wrong || !(max > -INFINITY);
          const float log_s = log1pf(s3);
          if (w)
            kc_raise(KC_ERR_BAD_ARGS);
          if (a.logprobs)
            a.logprobs[row] = w ? NAN : log_p(given, max, log_s);
          if (a.entropy)
            a.entropy[row] = w ? NAN : log_s + e3 / (1.0f + s3);
          t->sums[0][0] = max, t->sums[0][1] = log_s, t->verdict = w;
        }
        meet();
        const bool w = t->verdict != 0;
        const float max = t->sums[0][0], log_s = t->sums[0][1];
        int at = -1;
        unsigned long long k = 0;
        if (parts == 1) {
          at = tid, k = tid < kMaxTop ? t->part.top[tid] : 0;
        } else if (tid < keys && (k = t->merged[tid]) != 0) {
          at = 0;
          for (int i = 0; i < keys; i++)
            at += t->merged[i] > k;
        }
        if (w)
          at = tid;
        if (at >= 0 && at < a.top) {
          a.top_tokens[(size_t)row * a.top + at] = w ? -1 : (int)(0xffffffffu - (unsigned)k);
          a.top_logprobs[(size_t)row * a.top + at] = w ? NAN : log_p(logit_of(k), max, log_s);
        }
        meet();
      }
    }
  }
  if (parts > 1) {
    if (warp == kWarps)
      cluster.sync();  // with the consumers' above
    cluster.sync();    // the first part has read
  }
}

}  // namespace

extern "C" void k_token_logprobs(float *logprobs, float *entropy, int *top_tokens, float *top_logprobs,
                                 const float *logits, size_t ld, const int *tokens, int vocab, int rows, int top) {
  const char *name = "k_token_logprobs";
  if (rows == 0)
    return;
  if (vocab <= 0 || rows < 0 || top < 0 || top > kMaxTop || top > vocab || ld < (size_t)vocab) {
    kc_fail("%s: invalid shape vocab=%d rows=%d top=%d stride %zu", name, vocab, rows, top, ld);
    return;
  }
  if (!logits || !logprobs != !tokens || (top && (!top_tokens || !top_logprobs))) {
    kc_fail("%s: missing logits, log probabilities or tokens, or room for the top ones", name);
    return;
  }
  LogprobArgs a;
  memset(&a, 0, sizeof(a));
  a.logprobs = logprobs, a.entropy = entropy, a.top_tokens = top_tokens, a.top_logprobs = top_logprobs;
  a.logits = logits, a.ld = ld, a.tokens = tokens, a.vocab = vocab, a.rows = rows, a.top = top;
  // A cluster of CTAs to a row while their parts are long enough to pay for its two barriers, which cost more where CTAs share
  // their SMs; and one CTA where the rows have an SM each with few left over. Device time in a graph, us, by parts (rows x
  // vocabulary: in 1, 2, 4, 8): 1 x 32000: 8.8, 8.4, 8.2, 9.0; 8 x 32000: 9.0, 8.7, 8.5, 9.4; 64 x 32000: 9.2, 9.4, 11.0;
  // 8 x 128256: 18.8, 13.4, 11.0, 10.7; 30 x 50001: 11.2, 10.2, 10.2, 13.8; 37 x 128256: 19.0, 13.8, 12.5, 15.3; 64 x 128256:
  // 19.2, 15.2, 15.5; 32 x 262144: 32.7, 20.7, 16.6, 17.8; 74 x 65000: 12.4, 12.0, 12.7; 100 x 128256: 19.2, 16.9, 15.9;
  // 110: 19.3, 16.8; 120: 19.4, 21.1; 148: 19.3, 21.3; 160: 24.8, 21.6; 200: 26.6, 23.4; 129 x 50001: 11.5, 14.2.
  const int sms = kc_device_sms();
  int parts = 1;
  for (; parts < kMaxParts; parts *= 2) {
    const long long ctas = (long long)rows * parts * 2;
    if (ctas > kCtas * sms || vocab / (2 * parts) < (ctas <= sms ? 16384 : 49152))
      break;
    if (parts == 1 && rows <= sms && 2 * ctas > 3 * sms)
      break;
  }
  cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(logprobs_kernel), kSmem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(parts > 1 || rows < kCtas * sms ? rows * parts : kCtas * sms));
  cfg.blockDim = dim3(kThreads + 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = kc_stream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = kc_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (e == cudaSuccess)
    e = cudaLaunchKernelEx(&cfg, logprobs_kernel, a, parts);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}
