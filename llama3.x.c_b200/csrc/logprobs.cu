// Log probabilities of tokens, the entropy of their distribution and its likeliest tokens, from rows of logits
// (k_token_logprobs). With M the row's maximum, S = sum e^(x - M) and T = sum e^(x - M) (M - x):
// log p_i = (x_i - M) - log S, entropy = log S + T / S (two sums of terms of one sign: nothing cancels).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxTop = 32;

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

__device__ __forceinline__ unsigned long long block_max(unsigned long long k, unsigned long long *shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0)
    shared[threadIdx.x >> 5] = k;
  __syncthreads();
  for (int w = 0; w < kWarps; w++)
    k = max(k, shared[w]);
  return k;
}

// A CTA per row.
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobArgs a) {
  __shared__ unsigned long long keys[kWarps];
  __shared__ double sums[2][kWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int token = a.tokens ? a.tokens[row] : 0;
  if (token == -1)
    return;
  const float *x = a.logits + (size_t)row * a.ld;
  bool wrong = token < 0 || token >= a.vocab;
  unsigned long long best = 0;
  for (int i = t; i < a.vocab; i += kThreads) {
    wrong |= !(x[i] < INFINITY);
    best = max(best, key_of(x[i], i));
  }
  best = block_max(best, keys);
  const float top = logit_of(best);
  wrong = __syncthreads_or(wrong || !(top > -INFINITY));
  double s = 0.0, e = 0.0;
  if (!wrong)
    for (int i = t; i < a.vocab; i += kThreads) {
      const float d = x[i] - top, w = expf(d);
      s += w;
      e -= w > 0.0f ? (double)w * d : 0.0;
    }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    s += __shfl_xor_sync(0xffffffffu, s, o), e += __shfl_xor_sync(0xffffffffu, e, o);
  if (lane == 0)
    sums[0][warp] = s, sums[1][warp] = e;
  __syncthreads();
  s = e = 0.0;
  for (int w = 0; w < kWarps; w++)
    s += sums[0][w], e += sums[1][w];
  const double log_s = log(s);
  if (t == 0) {
    if (wrong)
      kc_raise(KC_ERR_BAD_ARGS);
    if (a.logprobs)
      a.logprobs[row] = wrong ? NAN : (float)((double)x[token] - top - log_s);
    if (a.entropy)
      a.entropy[row] = wrong ? NAN : (float)(log_s + e / s);
  }
  for (int k = 0; k < a.top; k++) {
    if (t == 0) {
      a.top_tokens[(size_t)row * a.top + k] = wrong ? -1 : (int)(0xffffffffu - (unsigned)best);
      a.top_logprobs[(size_t)row * a.top + k] = wrong ? NAN : (float)((double)logit_of(best) - top - log_s);
    }
    if (wrong || k + 1 == a.top)
      continue;
    unsigned long long next = 0;
    for (int i = t; i < a.vocab; i += kThreads) {
      const unsigned long long key = key_of(x[i], i);
      next = key < best ? max(next, key) : next;
    }
    best = block_max(next, keys);
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
  const cudaError_t e = kc_launch_pdl(logprobs_kernel, dim3((unsigned)rows), dim3(kThreads), 0, kc_stream(), a);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}
