// Attention over a paged cache in fp32, by tiles in shared memory: head_dim up to 128 in whole 16-byte units, aligned pages.
//
// Eight query vectors of a KV head against tiles of 64 positions, which four warps copy, asynchronously, through a ring that
// runs on into the next segment. Eight warps take a tile in three steps with a barrier behind each; what a key or value costs
// there besides its products is reads of shared memory, so each is read once:
//   scores: warp w takes the w-th eighth of the head, a lane two positions, all eight vectors: a key's unit of 16 bytes
//     meets eight vectors' (broadcasts), and two positions share each of those. No shuffles; the eighths' sums meet in
//     shared memory;
//   softmax: warp v takes vector v: its reference and its sum of weights are that warp's own;
//   sums: a warp takes eight positions, a lane four elements of the head, with all vectors' sums in registers.
// The 16-byte units of a row lie in an order that spreads eight rows over the banks.
// What bounds it: a tile's three steps take 3.0 thousand clocks (1.2 scores, 0.5 softmax, 1.2 sums; FMAs alone 1.0), its
// copies 2.9; with eight vectors where a KV head has fewer, some of that is for nothing. 24 requests of 28/4 heads of 128 up to
// 3001 positions: 50 us, 3.6 TB/s, of which 28 are for the tiles' bytes, 9 until the first tile is there and 5 for the joins; the
// other 8 have not been told apart.
#include "paged.cuh"
#include "tcgen05.cuh"

namespace {
using namespace paged;

constexpr int kTile = 64, kVecs = 8;
constexpr int kWarps = 8, kSoft = 32 * kWarps;  // that compute
constexpr int kCopyWarps = 4, kThreads = kSoft + 32 * kCopyWarps;
constexpr int kCtas = 148;
constexpr float kRise = 8.0f;            // how far a score may lie above the reference before the reference moves
constexpr float kFar = 3.402823466e+38f;  // the reference before there is one, negative

template <int HD>
struct Smem {
  static constexpr int kStages = HD == 128 ? 3 : 5;
  float kv[kStages][2][kTile][HD];
  union {
    float part[kWarps][kVecs][kTile];     // scores by eighths of the head
    float join[kWarps / 2][kVecs][HD];    // the warps' sums at the end of a piece
  };
  float q[kVecs][HD], weight[kVecs][kTile], keep[kVecs], m[kVecs], l[kVecs];
  uint64_t full[kStages], empty[kStages];
  RangeRoom room;
  int bad, last, abort_flag;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(void *dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}
// Arrives once all copies that this thread has started are in memory.
__device__ __forceinline__ void copy_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A wait that gives up at once when another one of the CTA has.
__device__ __forceinline__ void wait(uint64_t *bar, unsigned parity, volatile int *abort_flag) {
  if (!mbar_try_wait(bar, parity) && *abort_flag == 0 && !mbar_wait_sleep_bounded(bar, parity))
    *abort_flag = 1;
  __syncwarp();
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) paged_f32_kernel(const PagedArgs a) {
  using S = Smem<HD>;
  constexpr int kStages = S::kStages, kUnits = HD / 4;  // 16-byte units of a row
  extern __shared__ __align__(16) uint8_t raw[];
  S *s = reinterpret_cast<S *>(raw);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, hd = a.hd;
  if (t == 0) {
    for (int i = 0; i < kStages; i++) {
      mbar_init(&s->full[i], 32 * kCopyWarps);
      mbar_init(&s->empty[i], kWarps);
    }
    s->bad = s->abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  Range here;
  if (!find_range(a, kTile, &here, &s->room))
    return;
  const Range *range = &here;
  const float scale = rsqrtf((float)hd) * kLog2e;
  volatile int *abort_flag = &s->abort_flag;
  Walk walk(range);
  Piece p;

  if (warp >= kWarps) {
    // ---- copies: warp w of them rows 16 w .. 16 w + 15 of every tile ----
    constexpr int kRows = kTile / kCopyWarps, kAt = 32 / kUnits;  // rows of a warp, and of its instruction
    const int w = warp - kWarps, unit = lane % kUnits;
    int stage = 0;
    unsigned parity = 1;
    while (walk.next(a, range, kTile, &p)) {
      const int end = p.start + p.count;
      const int *pages = a.table + (size_t)p.b * a.max_pages;
      // Lane r of the first 16: the page of row r, asked for a tile before it is used; -1 where there is none.
      auto page_of = [&](int tile) -> int {
        int within = tile * kTile + kRows * w + lane;
        return tile < p.t1 && lane < kRows && within < end ? pages[divide(within, a.by_page)] : -1;
      };
      int page = page_of(p.t0);
      for (int tile = p.t0; tile < p.t1; tile++) {
        int within = tile * kTile + kRows * w + lane;
        divide(within, a.by_page);
        const long long place =
            page < 0 || page >= a.pages
                ? -1
                : (long long)((size_t)page * a.page_stride + ((size_t)p.head * a.page_size + within) * hd);
        page = page_of(tile + 1);
        wait(&s->empty[stage], parity, abort_flag);
#pragma unroll
        for (int i = 0; i < kRows / kAt; i++) {
          const int r = i * kAt + lane / kUnits, row = kRows * w + r;
          const long long at = __shfl_sync(0xffffffffu, place, r);
          const bool in = at >= 0 && 4 * unit < hd;
          const size_t src = in ? (size_t)at + 4 * unit : 0;
          const int to = (unit ^ (row & 7)) * 4;
          copy16(&s->kv[stage][0][row][to], static_cast<const float *>(a.key) + src, in);
          copy16(&s->kv[stage][1][row][to], static_cast<const float *>(a.value) + src, in);
        }
        copy_arrive(&s->full[stage]);
        if (++stage == kStages)
          stage = 0, parity ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ---- the computing warps ----
  int stage = 0;
  unsigned parity = 0;
  while (walk.next(a, range, kTile, &p)) {
    // The piece's queries, and whether every page of its positions is one.
    for (int i = t; i < kVecs * HD; i += kSoft) {
      const int v = i / HD, e = i % HD;
      int row;
      s->q[v][e] = v < p.vecs && e < hd ? a.q[(size_t)vector_at(a, p, v, &row) * hd + e] * scale : 0.0f;
    }
    {
      int from = p.t0 * kTile, to = min(p.t1 * kTile, p.start + p.count) - 1;
      from = divide(from, a.by_page), to = divide(to, a.by_page);
      bool bad = false;
      for (int i = from + t; i <= to; i += kSoft) {
        const int page = a.table[(size_t)p.b * a.max_pages + i];
        bad |= page < 0 || page >= a.pages;
      }
      if (bad)
        s->bad = 1;
    }
    const float guard = guard_of(p.start + p.count);
    int limit = 0;  // positions that this warp's vector sees
    if (warp < p.vecs) {
      int row;
      vector_at(a, p, warp, &row);
      limit = p.start + row + 1;
    }
    float m = -kFar, l = 0.0f;
    uint64_t acc[kVecs][2];
#pragma unroll
    for (int v = 0; v < kVecs; v++)
      acc[v][0] = acc[v][1] = 0;
    meet<kSoft, 1>();  // the queries are there
    for (int tile = p.t0; tile < p.t1; tile++) {
      wait(&s->full[stage], parity, abort_flag);
      // ---- scores ----
      {
        constexpr int kEach = HD / kWarps / 4;  // units of a row to a warp
        uint64_t x[2][kVecs];
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          x[0][v] = x[1][v] = 0;
#pragma unroll
        for (int u = 0; u < kEach; u++) {
          const int unit = warp * kEach + u, at = (unit ^ (lane & 7)) * 4;
          const ulonglong2 k0 = *reinterpret_cast<const ulonglong2 *>(&s->kv[stage][0][lane][at]);
          const ulonglong2 k1 = *reinterpret_cast<const ulonglong2 *>(&s->kv[stage][0][lane + 32][at]);
#pragma unroll
          for (int v = 0; v < kVecs; v++) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(&s->q[v][4 * unit]);
            x[0][v] = f2_fma(q.y, k0.y, f2_fma(q.x, k0.x, x[0][v]));
            x[1][v] = f2_fma(q.y, k1.y, f2_fma(q.x, k1.x, x[1][v]));
          }
        }
#pragma unroll
        for (int v = 0; v < kVecs; v++) {
          float lo, hi;
          f2_unpack(x[0][v], lo, hi);
          s->part[warp][v][lane] = lo + hi;
          f2_unpack(x[1][v], lo, hi);
          s->part[warp][v][lane + 32] = lo + hi;
        }
      }
      meet<kSoft, 1>();
      // ---- softmax of vector `warp` ----
      {
        float y[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int at = lane + 32 * i;
          y[i] = ((s->part[0][warp][at] + s->part[1][warp][at]) + (s->part[2][warp][at] + s->part[3][warp][at])) +
                 ((s->part[4][warp][at] + s->part[5][warp][at]) + (s->part[6][warp][at] + s->part[7][warp][at]));
          y[i] = tile * kTile + at < limit ? y[i] : -INFINITY;
        }
        float keep = 1.0f;
        if (__any_sync(0xffffffffu, y[0] > m + kRise || y[1] > m + kRise)) {
          const float top = fmaxf(warp_max(fmaxf(y[0], y[1])), m);
          keep = ex2(m - top);
          m = top;
          l *= keep;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float w = ex2(y[i] - m) * (guard * 0x1p-8f);
          l += w;
          s->weight[warp][lane + 32 * i] = w;
        }
        if (lane == 0)
          s->keep[warp] = keep;
      }
      meet<kSoft, 1>();
      // ---- sums: positions 8 warp .. 8 warp + 7 ----
      {
        const float4 keep[2] = {*reinterpret_cast<const float4 *>(&s->keep[0]), *reinterpret_cast<const float4 *>(&s->keep[4])};
        const float f[kVecs] = {keep[0].x, keep[0].y, keep[0].z, keep[0].w, keep[1].x, keep[1].y, keep[1].z, keep[1].w};
        bool moved = false;
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          moved |= f[v] != 1.0f;
        if (moved)
#pragma unroll
          for (int v = 0; v < kVecs; v++) {
            acc[v][0] = f2_mul(acc[v][0], f2_pack(f[v], f[v]));
            acc[v][1] = f2_mul(acc[v][1], f2_pack(f[v], f[v]));
          }
        // HD 128: all lanes a row; HD 64: half a warp a row, four of the eight positions each.
        constexpr int kSets = HD == 128 ? 2 : 1;
        const int unit = lane % kUnits, first = 8 * warp + (HD == 128 ? 0 : 4 * (lane / kUnits));
#pragma unroll
        for (int g = 0; g < kSets; g++) {
          const int p0 = first + 4 * g;
          float4 w[kVecs];
          ulonglong2 x[4];
#pragma unroll
          for (int i = 0; i < 4; i++)
            x[i] = *reinterpret_cast<const ulonglong2 *>(&s->kv[stage][1][p0 + i][(unit ^ ((p0 + i) & 7)) * 4]);
#pragma unroll
          for (int v = 0; v < kVecs; v++)
            w[v] = *reinterpret_cast<const float4 *>(&s->weight[v][p0]);
          auto add = [&](int v, int i) {
            const float y = i == 0 ? w[v].x : i == 1 ? w[v].y : i == 2 ? w[v].z : w[v].w;
            acc[v][0] = f2_fma(f2_pack(y, y), x[i].x, acc[v][0]);
            acc[v][1] = f2_fma(f2_pack(y, y), x[i].y, acc[v][1]);
          };
          if (tile * kTile + kTile <= p.start + 1) {  // every row sees all of the tile
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
              for (int v = 0; v < kVecs; v++)
                add(v, i);
          } else {
            // What a row does not see may be anything: its product is left out, not made with a weight of zero.
#pragma unroll
            for (int v = 0; v < kVecs; v++) {
              int member = p.block * kVecs + v;
              const int sees = p.start + divide(member, a.by_group) - (tile * kTile + p0);
#pragma unroll
              for (int i = 0; i < 4; i++)
                if (i <= sees && v < p.vecs)
                  add(v, i);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&s->empty[stage]);  // behind the products, which have waited for all that was read
      if (++stage == kStages)
        stage = 0, parity ^= 1;
    }
    // ---- the end of the piece: the warps' sums joined two by two ----
#pragma unroll
    for (int o = 16; o; o >>= 1)
      l += __shfl_xor_sync(0xffffffffu, l, o);
    float y[kVecs][4];
#pragma unroll
    for (int v = 0; v < kVecs; v++) {
      f2_unpack(acc[v][0], y[v][0], y[v][1]);
      f2_unpack(acc[v][1], y[v][2], y[v][3]);
      if (HD == 64)
#pragma unroll
        for (int i = 0; i < 4; i++)
          y[v][i] += __shfl_xor_sync(0xffffffffu, y[v][i], 16);
    }
    meet<kSoft, 1>();  // the scores' room is free
    if (lane == 0)
      s->m[warp] = m, s->l[warp] = l;
    if (*abort_flag)
      s->bad = 1;
#pragma unroll
    for (int half = kWarps / 2; half; half >>= 1) {
      if (warp >= half && warp < 2 * half && lane < kUnits)
#pragma unroll
        for (int v = 0; v < kVecs; v++)
          *reinterpret_cast<float4 *>(&s->join[warp - half][v][4 * lane]) = make_float4(y[v][0], y[v][1], y[v][2], y[v][3]);
      meet<kSoft, 1>();
      if (warp < half && lane < kUnits)
#pragma unroll
        for (int v = 0; v < kVecs; v++) {
          const float4 x = *reinterpret_cast<const float4 *>(&s->join[warp][v][4 * lane]);
          y[v][0] += x.x, y[v][1] += x.y, y[v][2] += x.z, y[v][3] += x.w;
        }
      meet<kSoft, 1>();
    }
    float *sums = &s->join[0][0][0];  // [vecs][hd]
    if (warp == 0 && 4 * lane < hd)
#pragma unroll
      for (int v = 0; v < kVecs; v++)
        if (v < p.vecs)
          *reinterpret_cast<float4 *>(sums + v * hd + 4 * lane) = make_float4(y[v][0], y[v][1], y[v][2], y[v][3]);
    meet<kSoft, 1>();
    finish<kSoft, 1, 0>(a, range, p, s->m, s->l, sums, &s->bad, &s->last, t);
    if (t == 0)
      s->bad = 0;
    meet<kSoft, 1>();
  }
}

template <int HD>
cudaError_t launch(const PagedArgs &a) {
  const auto kernel = paged_f32_kernel<HD>;
  const cudaError_t e = kc_allow_smem(reinterpret_cast<const void *>(kernel), (int)sizeof(Smem<HD>));
  return e != cudaSuccess ? e : kc_launch_pdl(kernel, dim3(kCtas), dim3(kThreads), sizeof(Smem<HD>), kc_stream(), a);
}

}  // namespace

// Everything that its copies can bring goes here: the kernel on the CUDA cores in paged.cu is slower at all of it. us here and
// there: 24 requests of one row, up to 3001 positions, heads of 32, 64, 96, 128:
//   28/4 heads   33.9, 34.6, 48.6, 50.1    69.1, 86.4, 139, 151      32/8   57.2, 58.0, 79.0, 80.0    77.4, 98.5, 150, 160
//   16/16        104, 104, 142, 142        140, 167, 269, 287        8/2    22.7, 22.6, 28.4, 28.8    31.5, 36.6, 48.1, 56.9
//   48/1         46.7, 46.5, 62.8, 62.1    96.4, 112, 173, 181
// 1 request of 512 positions, 32/8 heads of 4, 16, 128: 9.7, 9.7, 10.4    15.1, 15.3, 22.0. 2 requests of up to 64 rows, 512
// positions, 32/8 heads of 64: 31.0    71.9.
bool kc_paged_f32_ok(const PagedArgs &a, int type) {
  return type == K_F32 && a.hd % 4 == 0 && a.hd <= 128 && a.page_stride % 4 == 0 &&
         !(((uintptr_t)a.key | (uintptr_t)a.value) & 15);
}

cudaError_t kc_launch_paged_f32(const PagedArgs &a) { return a.hd > 64 ? launch<128>(a) : launch<64>(a); }
