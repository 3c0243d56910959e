// Low-rank adapters of many requests beside a shared projection (k_lora_rows): out[r] = base[r] + scale B (A x[r]) with
// the adapter that row r names, A [rank][n] and B [d][rank] in fp32, bf16 or fp16. Products and sums are fp32.
//
// One launch: a cluster of CTAs per row. Each CTA takes a slice of n for A x, the cluster sums the slices' partial
// vectors through distributed shared memory in CTA order (no atomics: the same bits on every call), and each CTA then
// takes a slice of d for B. The rank-long vector between the two products never leaves the SMs.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/kernels_cuda.h"
#include "common.cuh"
#include "kernels_cuda_internal.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRank = 256;

struct LoraArgs {
  float *out;
  const float *base, *x;
  long long ldo, ldb, ldx;
  const int *index;
  const LoraAdapter *adapters;
  int count, max_rank, n, d, rows;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// Eight neighbouring weights from a 16-byte aligned address.
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename H2>
__device__ __forceinline__ void halves(const void *p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    H2 h;
    *reinterpret_cast<unsigned *>(&h) = w[i];
    v[2 * i] = to_float(h.x), v[2 * i + 1] = to_float(h.y);
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) { halves<__nv_bfloat162>(p, v); }
__device__ __forceinline__ void load8(const __half *p, float (&v)[8]) { halves<__half2>(p, v); }

__device__ __forceinline__ bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename W>
__global__ void __launch_bounds__(kThreads) lora_row_kernel(const LoraArgs a) {
  __shared__ float part[kMaxRank], h[kMaxRank];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int id = a.index[row];
  LoraAdapter w = {nullptr, nullptr, 0, 0.0f};
  bool bad = id < -1 || id >= a.count;
  if (!bad && id >= 0) {
    w = a.adapters[id];
    bad = w.rank < 0 || w.rank > a.max_rank || (w.rank > 0 && (!w.a || !w.b));
  }
  if (bad) {
    w.rank = 0;
    if (rank == 0 && threadIdx.x == 0)
      kc_raise(KC_ERR_BAD_ARGS);
  }
  // A x over this CTA's slice of n, a warp per row of A.
  const W *A = static_cast<const W *>(w.a), *B = static_cast<const W *>(w.b);
  const float *x = a.x + (long long)row * a.ldx;
  const int n_slice = ((a.n + ctas - 1) / ctas + 7) & ~7;
  const int n0 = min(rank * n_slice, a.n), n1 = min(n0 + n_slice, a.n);
  const bool wide = aligned16(A) && aligned16(x) && a.n % 8 == 0;
  for (int k = warp; k < w.rank; k += kWarps) {
    const W *ak = A + (long long)k * a.n;
    float s = 0.0f;
    if (wide) {
      for (int i = n0 + 8 * lane; i < n1; i += 256) {
        float wv[8], xv[8];
        load8(ak + i, wv);
        load8(x + i, xv);
#pragma unroll
        for (int j = 0; j < 8; j++)
          s = fmaf(wv[j], xv[j], s);
      }
    } else {
      for (int i = n0 + lane; i < n1; i += 32)
        s = fmaf(to_float(ak[i]), x[i], s);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
      s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0)
      part[k] = s;
  }
  cluster.sync();
  for (int k = threadIdx.x; k < w.rank; k += kThreads) {
    float s = 0.0f;
    for (int c = 0; c < ctas; c++)
      s += *cluster.map_shared_rank(&part[k], c);
    h[k] = s * w.scale;
  }
  cluster.sync();  // the slices are read: a CTA may leave, and h is whole
  const int d_slice = (a.d + ctas - 1) / ctas;
  const int d0 = min(rank * d_slice, a.d), d1 = min(d0 + d_slice, a.d);
  const bool wide_b = aligned16(B) && w.rank % 8 == 0;
  for (int i = d0 + threadIdx.x; i < d1; i += kThreads) {
    const W *bi = B + (long long)i * w.rank;
    float s = 0.0f;
    if (wide_b) {
      for (int k = 0; k < w.rank; k += 8) {
        float wv[8];
        load8(bi + k, wv);
#pragma unroll
        for (int j = 0; j < 8; j++)
          s = fmaf(wv[j], h[k + j], s);
      }
    } else {
      for (int k = 0; k < w.rank; k++)
        s = fmaf(to_float(bi[k]), h[k], s);
    }
    const float before = a.base ? a.base[(long long)row * a.ldb + i] : 0.0f;
    a.out[(long long)row * a.ldo + i] = before + s;
  }
}

template <typename W>
cudaError_t launch(const LoraArgs &a) {
  cudaLaunchConfig_t cfg = {};
  const int ctas = 8;
  cfg.gridDim = dim3((unsigned)a.rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = kc_stream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = kc_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, lora_row_kernel<W>, a);
}

}  // namespace

extern "C" {

void k_lora_rows(float *out, size_t ldo, const float *base, size_t ldb, const float *x, size_t ldx, const int *index,
                 const LoraAdapter *adapters, int count, int type, int max_rank, int n, int d, int rows) {
  const char *name = "k_lora_rows";
  if (type != K_F32 && type != K_BF16 && type != K_F16) {
    kc_fail("%s: invalid weight type %d", name, type);
    return;
  }
  if (rows < 0 || rows > (1 << 24) || n <= 0 || d <= 0 || count < 0 || max_rank <= 0 || max_rank > kMaxRank ||
      ldx < (size_t)n || ldo < (size_t)d || (base && ldb < (size_t)d)) {
    kc_fail("%s: invalid shape rows=%d n=%d d=%d count=%d max_rank=%d (at most %d)", name, rows, n, d, count, max_rank,
            kMaxRank);
    return;
  }
  if (!rows)
    return;
  if (!out || !x || !index || (count && !adapters)) {
    kc_fail("%s: missing output, activations, row indices or adapters", name);
    return;
  }
  const LoraArgs a = {out, base, x, (long long)ldo, (long long)ldb, (long long)ldx, index, adapters, count, max_rank,
                      n, d, rows};
  const cudaError_t e = type == K_F32 ? launch<float>(a) : type == K_BF16 ? launch<__nv_bfloat16>(a) : launch<__half>(a);
  if (e == cudaSuccess)
    kc_count_launch();
  else
    kc_fail("%s: CUDA launch failed: %s", name, cudaGetErrorString(cudaGetLastError()));
}

}  // extern "C"
