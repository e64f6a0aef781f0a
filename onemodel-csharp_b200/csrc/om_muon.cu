// The Muon update: momentum, orthogonalisation of the update by Newton-Schulz steps, weight decay and the weights.
//
// A matrix is worked on as X [m, n] with m <= n (transposed where it is taller). One step is
//   G = X X^T,  Y = -4.7750 G + 2.0315 G G,  X' = 3.4445 X + Y X,
// three products; G and Y are symmetric, so their blocks above the diagonal are mirrored instead of computed. All matrices of a
// call go through each launch together: a launch covers the tiles of one product of up to MU_TENSORS matrices, whatever their
// shapes, so a step costs three launches for a whole model.
//
// The products run on the tensor pipe: a value v is kept as two half-precision numbers, h = half(v) and l = half(v - h), 22 significant
// bits together, and a product is h h' + h l' + l h' (what is left out is 2^-22 of it). Five steps raise an error in the direction of a small
// singular value up to 3.4445^5 = 485 times, which is why plain half or bfloat16 operands (2^-11, 2^-8) would leave few digits of the
// update. The tensor core cuts off what a sum cannot hold at every addition, always towards zero: an error that grows with the length of
// the sum (X off by 1.2e-5 for a long side of 1536 and 7.6e-5 for 16384, where fp32 products leave 2e-6). So its sums are of 256 terms
// and are added up in fp32 (6e-6 and 2e-6), and h h' has an accumulator of its own, the two small products another. Sums of 128 terms: 4e-6, and
// 24 matrices of 384 x 384 to 1536 368 us instead of 355. Every matrix of a step is bounded (|X| <= 1.2, |G| <= 1.5, |Y| <= 3 in the
// spectral norm, so element by element), and is stored times a power of two that puts its usual elements in the middle of the
// half's range. Three products at the 16-bit rate bound it: 3/1664 s a TFLOP; two planes of 2 bytes are what fp32 would read.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <vector>

#include "om_tc.cuh"

namespace om {

constexpr int MU_TENSORS = 32;
constexpr float MU_A = 3.4445f, MU_B = -4.7750f, MU_C = 2.0315f;   // the quintic's coefficients
constexpr int MU_CHUNK = 8192;                                     // elements of one partial sum of squares
constexpr int MU_BM = 128, MU_BK = 64;                             // rows of a tile of a product, terms of a stage
constexpr int MU_SUM = 4;                                          // stages that one sum of the tensor core runs over
constexpr float MU_SX = 1024.f, MU_SG = 4096.f;                    // X is stored times the first, G and Y times the second
constexpr int MU_EPI = 8;                                          // warps 0-7: results, half of a tile's columns each four; warp 8: MMA issue; warp 9: TMA
constexpr int MU_THREADS = 32 * (MU_EPI + 2);

// A matrix as two planes of halves, the second `plane` elements behind the first, rows `ld` apart.
struct MuonPlanes {
  __half* p;
  long long plane;
  int ld;
};
struct MuonTensor {
  float *p, *m;
  const float* g;
  uint16_t* p16;
  int rows, cols;        // as the caller has them
  int mm, nn;            // sides of X, mm <= nn
  int quads;             // rows of p, m and g start where four elements move at once
  double* partial;       // [ceil(rows * cols / MU_CHUNK)]
  MuonPlanes x, x2, gram, poly;   // [mm, nn], [mm, nn], [mm, mm], [mm, mm]
};
struct MuonList {
  om_muon_hyper hyper;
  const om_muon_hyper* hyper_dev;
  int32_t* status;
  int count;
  long long end[MU_TENSORS];      // work items of this launch up to and with tensor i
  MuonTensor t[MU_TENSORS];
};
// The operands of one launch's products: A's tiles, and B's.
struct MuonMaps {
  CUtensorMap a[MU_TENSORS], b[MU_TENSORS];
};
__device__ __forceinline__ om_muon_hyper mu_hyper(const MuonList& l) { return l.hyper_dev ? *l.hyper_dev : l.hyper; }
__device__ __forceinline__ int mu_find(const MuonList& l, long long item, long long* local) {
  int i = 0;
  while (item >= l.end[i]) i++;
  *local = item - (i ? l.end[i - 1] : 0);
  return i;
}

// m = momentum m + (1 - momentum) g, and the sum of squares of u over this chunk (in double: the chunks of a large matrix
// differ by orders of magnitude in what they add, and squares of u beyond 2^64 or below 2^-64 leave fp32).
__global__ void __launch_bounds__(256) muon_momentum_kernel(const __grid_constant__ MuonList l) {
  pdl_enter();
  long long chunk;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &chunk)];
  const om_muon_hyper h = mu_hyper(l);
  const long long n = (long long)t.rows * t.cols, e0 = chunk * MU_CHUNK, e1 = min(e0 + MU_CHUNK, n);
  double sum = 0.0;
  auto one = [&](float g, float& m) {
    g = g * h.grad_scale * (1.f - h.momentum);
    m = fmaf(m, h.momentum, g);
    const double u = h.nesterov ? fmaf(m, h.momentum, g) : m;
    return u * u;
  };
  // What a thread needs comes in front of what it writes: between a store and a load behind it the compiler keeps the order.
  if (t.quads) {
    for (long long e = e0 + 4 * threadIdx.x; e < e1; e += 4096) {
      float4 g[4], m[4];
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (e + 1024 * u < e1) {
          g[u] = *reinterpret_cast<const float4*>(t.g + e + 1024 * u);
          m[u] = *reinterpret_cast<const float4*>(t.m + e + 1024 * u);
        }
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (e + 1024 * u < e1) {
          const double a = one(g[u].x, m[u].x), b = one(g[u].y, m[u].y), c = one(g[u].z, m[u].z), d = one(g[u].w, m[u].w);
          *reinterpret_cast<float4*>(t.m + e + 1024 * u) = m[u];
          sum += (a + b) + (c + d);
        }
    }
  } else {
    for (long long e = e0 + threadIdx.x; e < e1; e += 2048) {
      float g[8], m[8];
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (e + 256 * u < e1) {
          g[u] = t.g[e + 256 * u];
          m[u] = t.m[e + 256 * u];
        }
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (e + 256 * u < e1) {
          sum += one(g[u], m[u]);
          t.m[e + 256 * u] = m[u];
        }
    }
  }
  __shared__ double s[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < 8; w++) all += s[w];
    t.partial[chunk] = all;
  }
}

__device__ __forceinline__ void mu_split(float v, __half* h, __half* l) {
  *h = __float2half_rn(v);
  *l = __float2half_rn(v - __half2float(*h));
}
// Tile (row block, column block) of 64 x 64 of the caller's matrix.
__device__ __forceinline__ void mu_block(const MuonTensor& t, long long tile, int* r0, int* c0) {
  const int across = (t.cols + 63) / 64;
  *r0 = (int)(tile / across) * 64;
  *c0 = (int)(tile % across) * 64;
}

// X = u / max(|u|, eps) as two planes, transposed where the matrix is taller than wide.
__global__ void __launch_bounds__(256) muon_start_kernel(const __grid_constant__ MuonList l) {
  pdl_enter();
  long long tile;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &tile)];
  const om_muon_hyper h = mu_hyper(l);
  const long long chunks = ((long long)t.rows * t.cols + MU_CHUNK - 1) / MU_CHUNK;
  __shared__ double s[8];
  __shared__ float block[64][65];
  double sum = 0.0;
  for (long long c = threadIdx.x; c < chunks; c += 256) sum += t.partial[c];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < 8; w++) sum += s[w];
  // A norm near fp32's end, or past it, is divided out 2^-64 of u at a time.
  const double full = fmax(sqrt(sum), (double)h.eps);
  const float part = full > 1e30 ? 0x1p-64f : 1.f, norm = full > 0.0 ? (float)(full * part) : 1.f;   // nothing over nothing: nothing
  int r0, c0;
  mu_block(t, tile, &r0, &c0);
  const bool turn = t.rows > t.cols;
  auto one = [&](float m, float g) { return (h.nesterov ? fmaf(m, h.momentum, g * h.grad_scale * (1.f - h.momentum)) : m) * part / norm * MU_SX; };
  if (t.quads) {
#pragma unroll
    for (int e = threadIdx.x; e < 64 * 16; e += 256) {
      const int a = e / 16, b = e % 16 * 4;
      if (r0 + a >= t.rows || c0 + b >= t.cols) continue;
      const long long at = (long long)(r0 + a) * t.cols + c0 + b;
      const float4 m = *reinterpret_cast<const float4*>(t.m + at), g = h.nesterov ? *reinterpret_cast<const float4*>(t.g + at) : m;
      block[a][b] = one(m.x, g.x);
      block[a][b + 1] = one(m.y, g.y);
      block[a][b + 2] = one(m.z, g.z);
      block[a][b + 3] = one(m.w, g.w);
    }
  } else {
#pragma unroll 16
    for (int e = threadIdx.x; e < 64 * 64; e += 256) {
      const int r = r0 + e / 64, c = c0 + e % 64;
      if (r >= t.rows || c >= t.cols) continue;
      const long long at = (long long)r * t.cols + c;
      block[e / 64][e % 64] = one(t.m[at], t.g[at]);
    }
  }
  __syncthreads();
  // Eight values of a row of X at a time: the pitch holds whole groups of 8.
#pragma unroll
  for (int e = threadIdx.x; e < 64 * 8; e += 256) {
    const int a = e / 8, b = e % 8 * 8;
    const int xr = (turn ? c0 : r0) + a, xc = (turn ? r0 : c0) + b;
    if (xr >= t.mm || xc >= t.nn) continue;
    uint4 hi, lo;
    __half *hp = reinterpret_cast<__half*>(&hi), *lp = reinterpret_cast<__half*>(&lo);
#pragma unroll
    for (int u = 0; u < 8; u++) mu_split(xc + u < t.nn ? (turn ? block[b + u][a] : block[a][b + u]) : 0.f, hp + u, lp + u);
    const long long at = (long long)xr * t.x.ld + xc;
    *reinterpret_cast<uint4*>(t.x.p + at) = hi;
    *reinterpret_cast<uint4*>(t.x.p + t.x.plane + at) = lo;
  }
}

// p = (1 - lr weight_decay) p - lr s X, with the bfloat16 copy where it is wanted.
__global__ void __launch_bounds__(256) muon_finish_kernel(const __grid_constant__ MuonList l) {
  pdl_enter();
  long long tile;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &tile)];
  const om_muon_hyper h = mu_hyper(l);
  const float s = h.match_rms ? 0.2f * sqrtf((float)max(t.rows, t.cols)) : sqrtf(fmaxf(1.f, (float)t.rows / (float)t.cols));
  const float keep = 1.f - h.lr * h.weight_decay, rate = h.lr * s;
  __shared__ float block[64][65];
  int r0, c0;
  mu_block(t, tile, &r0, &c0);
  const bool turn = t.rows > t.cols;
#pragma unroll
  for (int e = threadIdx.x; e < 64 * 8; e += 256) {
    const int a = e / 8, b = e % 8 * 8;
    const int xr = (turn ? c0 : r0) + a, xc = (turn ? r0 : c0) + b;
    if (xr >= t.mm || xc >= t.nn) continue;
    const long long at = (long long)xr * t.x.ld + xc;
    const uint4 hi = *reinterpret_cast<const uint4*>(t.x.p + at), lo = *reinterpret_cast<const uint4*>(t.x.p + t.x.plane + at);
    const __half *hp = reinterpret_cast<const __half*>(&hi), *lp = reinterpret_cast<const __half*>(&lo);
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const float v = (__half2float(hp[u]) + __half2float(lp[u])) * (1.f / MU_SX);
      if (turn) block[b + u][a] = v;
      else block[a][b + u] = v;
    }
  }
  __syncthreads();
  auto half16 = [](float v) {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    return *reinterpret_cast<const uint16_t*>(&b);
  };
  if (t.quads) {
    float4 p[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int a = (int)threadIdx.x / 16 + 16 * u, b = threadIdx.x % 16 * 4;
      if (r0 + a < t.rows && c0 + b < t.cols) p[u] = *reinterpret_cast<const float4*>(t.p + (long long)(r0 + a) * t.cols + c0 + b);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int a = (int)threadIdx.x / 16 + 16 * u, b = threadIdx.x % 16 * 4;
      if (r0 + a >= t.rows || c0 + b >= t.cols) continue;
      const long long at = (long long)(r0 + a) * t.cols + c0 + b;
      const float4 q = make_float4(fmaf(-rate, block[a][b], p[u].x * keep), fmaf(-rate, block[a][b + 1], p[u].y * keep), fmaf(-rate, block[a][b + 2], p[u].z * keep),
                                   fmaf(-rate, block[a][b + 3], p[u].w * keep));
      *reinterpret_cast<float4*>(t.p + at) = q;
      if (t.p16)
        *reinterpret_cast<uint2*>(t.p16 + at) = make_uint2((uint32_t)half16(q.x) | (uint32_t)half16(q.y) << 16, (uint32_t)half16(q.z) | (uint32_t)half16(q.w) << 16);
    }
  } else {
    float p[16];
    const int b = threadIdx.x % 64;
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const int a = (int)threadIdx.x / 64 + 4 * u;
      if (r0 + a < t.rows && c0 + b < t.cols) p[u] = t.p[(long long)(r0 + a) * t.cols + c0 + b];
    }
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const int a = (int)threadIdx.x / 64 + 4 * u;
      if (r0 + a >= t.rows || c0 + b >= t.cols) continue;
      const long long at = (long long)(r0 + a) * t.cols + c0 + b;
      const float q = fmaf(-rate, block[a][b], p[u] * keep);
      t.p[at] = q;
      if (t.p16) t.p16[at] = half16(q);
    }
  }
}

// ---- products ---------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void mu_load(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)), "l"(map),
               "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
               : "memory");
}
// A warp moves blocks of 32 rows by 32 columns of planes with four lanes a row (64 bytes; a lane a row would touch 32 lines with each
// access), and turns them to a row a lane through shared memory. Columns start at multiples of 8 and the pitch is one too, so whole
// groups of 8 lie within it. `e` of the four: row 8 e + lane / 4, columns 8 (lane & 3) ...
struct MuonBlock {
  uint4 h[4], l[4];
};
__device__ __forceinline__ void mu_fetch(const MuonPlanes& x, int row0, int rows, int col, int cols, int lane, MuonBlock& v) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int r = row0 + 8 * e + (lane >> 2), c = col + 8 * (lane & 3);
    v.h[e] = v.l[e] = make_uint4(0, 0, 0, 0);
    if (r < rows && c < cols) {
      const __half* at = x.p + (long long)r * x.ld + c;
      v.h[e] = *reinterpret_cast<const uint4*>(at);
      v.l[e] = *reinterpret_cast<const uint4*>(at + x.plane);
    }
  }
}
constexpr int MU_PITCH = 5;                              // uint4 a row of 32 halves: four and a gap
__device__ __forceinline__ void mu_to_rows(uint4* stage, int lane, const uint4 (&block)[4], uint4 (&row)[4]) {
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 4; e++) stage[(8 * e + (lane >> 2)) * MU_PITCH + (lane & 3)] = block[e];
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 4; e++) row[e] = stage[lane * MU_PITCH + e];
}
__device__ __forceinline__ void mu_put(uint4* stage, int lane, const uint32_t (&row)[16], __half* p, int ld, int row0, int rows, int col, int cols) {
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 4; e++) stage[lane * MU_PITCH + e] = make_uint4(row[4 * e], row[4 * e + 1], row[4 * e + 2], row[4 * e + 3]);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int r = row0 + 8 * e + (lane >> 2), c = col + 8 * (lane & 3);
    if (r < rows && c < cols) *reinterpret_cast<uint4*>(p + (long long)r * ld + c) = stage[(8 * e + (lane >> 2)) * MU_PITCH + (lane & 3)];
  }
}
__device__ __forceinline__ float mu_value(const uint4 (&h)[4], const uint4 (&l)[4], int u) {
  return __half2float(reinterpret_cast<const __half*>(h)[u]) + __half2float(reinterpret_cast<const __half*>(l)[u]);
}

// Shared memory of a product's CTA. Tensor memory: two accumulators of the large products, which take the sums in turn, and two of the
// small ones, which take the tiles in turn: what one holds is read back under the products of the other.
constexpr int MU_PLANE = MU_BM * MU_BK * 2, MU_STAGE = 4 * MU_PLANE, MU_STAGES = 3;
constexpr int MU_TURN = MU_STAGES * MU_STAGE, MU_BARS = MU_TURN + MU_EPI * 32 * MU_PITCH * 16, MU_SMEM = MU_BARS + 256;

// Where item `tile` of a launch lies.
struct MuonTile {
  int which, r0, c0;
};
template <int KIND>
__device__ __forceinline__ MuonTile mu_tile(const MuonList& l, long long tile) {
  MuonTile m;
  m.which = mu_find(l, tile, &tile);
  if (KIND == 2) {
    const int down = (l.t[m.which].mm + MU_BM - 1) / MU_BM;      // down the rows first: the CTAs of a round share columns of X
    m.c0 = (int)(tile / down) * MU_BM;
    m.r0 = (int)(tile % down) * MU_BM;
  } else {
    int rb = 0;
    for (; tile > rb; rb++) tile -= rb + 1;
    m.r0 = rb * MU_BM;
    m.c0 = (int)tile * MU_BM;
  }
  return m;
}

// Blocks of 128 rows by 128 columns of one product over every matrix; a CTA takes every gridDim.x-th. KIND 0: gram = x x^T; 1: poly = B gram +
// C gram gram (both symmetric: only the blocks on and below the diagonal, the others mirrored from there); 2: x2 = A x + poly x.
template <int KIND>
__global__ void __launch_bounds__(MU_THREADS, 1) muon_product_kernel(const __grid_constant__ MuonList l, const __grid_constant__ MuonMaps maps) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + MU_BARS);
  uint64_t *bar_full = bars, *bar_empty = bars + MU_STAGES, *bar_done = bars + 2 * MU_STAGES /* [2] */, *bar_read = bar_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_read + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MU_STAGES; s++) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int s = 0; s < 2; s++) {
      mbar_init(&bar_done[s], 1);
      mbar_init(&bar_read[s], MU_EPI);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MU_EPI) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const long long tiles = l.end[l.count - 1];
  bool ok = true;
  if (warp == MU_EPI + 1) {
    if (lane == 0) {
      uint32_t n = 0;                                    // stages filled
      for (long long tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        const MuonTile m = mu_tile<KIND>(l, tile);
        const int steps = ((KIND == 0 ? l.t[m.which].nn : l.t[m.which].mm) + MU_BK - 1) / MU_BK;
        const CUtensorMap *map_a = &maps.a[m.which], *map_b = KIND == 2 ? &maps.b[m.which] : map_a;
        for (int k = 0; ok && k < steps; k++, n++) {
          const uint32_t s = n % MU_STAGES;
          if (n >= MU_STAGES) ok = mbar_wait(&bar_empty[s], ((n / MU_STAGES) & 1u) ^ 1u, abort_flag, l.status, 101);
          if (!ok) break;
          uint8_t* at = smem + s * MU_STAGE;
          mbar_expect_tx(&bar_full[s], MU_STAGE);
#pragma unroll
          for (int plane = 0; plane < 2; plane++) {
            mu_load(at + plane * MU_PLANE, map_a, k * MU_BK, m.r0, plane, &bar_full[s]);
            uint8_t* b = at + (2 + plane) * MU_PLANE;
            if (KIND == 2) {
              mu_load(b, map_b, m.c0, k * MU_BK, plane, &bar_full[s]);
              mu_load(b + 64 * 128, map_b, m.c0 + 64, k * MU_BK, plane, &bar_full[s]);
            } else {
              mu_load(b, map_b, k * MU_BK, m.c0, plane, &bar_full[s]);
            }
          }
        }
      }
    }
  } else if (warp == MU_EPI) {
    if (lane == 0) {
      // Half-precision operands, fp32 sums; B is K-major (rows of the same matrix) or MN-major (X as it lies).
      constexpr uint32_t idesc = (1u << 4) | ((KIND == 2 ? 1u : 0u) << 16) | ((uint32_t)(MU_BM >> 3) << 17) | ((uint32_t)(MU_BM >> 4) << 24);
      constexpr uint32_t lbo_b = KIND == 2 ? ((64u * 128u) >> 4) << 16 : 1u << 16, step_b = KIND == 2 ? (16u * 128u) >> 4 : 2u;
      uint32_t n = 0, j = 0, turn = 0;                   // stages used, sums begun, tiles
      for (long long tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, turn ^= 1u) {
        const MuonTensor& t = l.t[mu_tile<KIND>(l, tile).which];
        const int steps = ((KIND == 0 ? t.nn : t.mm) + MU_BK - 1) / MU_BK;
        const uint32_t small = tmem + (2 + turn) * MU_BM;
        for (int k = 0; ok && k < steps; k++, n++) {
          const uint32_t s = n % MU_STAGES, place = j & 1u, acc = tmem + place * MU_BM;
          // The sum before last has been read, and with it, where it was a tile's last, that tile's small products.
          if (k % MU_SUM == 0 && j >= 2 && !(ok = mbar_wait(&bar_read[place], ((j >> 1) & 1u) ^ 1u, abort_flag, l.status, 104))) break;
          if (!(ok = mbar_wait(&bar_full[s], (n / MU_STAGES) & 1u, abort_flag, l.status, 102))) break;
          tc_fence_after();
          const uint32_t a_h = (smem_u32(smem + s * MU_STAGE) >> 4) | 1u << 16, a_l = a_h + (MU_PLANE >> 4);
          const uint32_t b_h = (smem_u32(smem + s * MU_STAGE + 2 * MU_PLANE) >> 4) | lbo_b, b_l = b_h + (MU_PLANE >> 4);
#pragma unroll
          for (int ks = 0; ks < MU_BK / 16; ks++) {
            const uint32_t ao = ks * 2u, bo = ks * step_b;
            umma_f16_ss(acc, a_h + ao, b_h + bo, idesc, k % MU_SUM > 0 || ks > 0 ? 1u : 0u);
            umma_f16_ss(small, a_h + ao, b_l + bo, idesc, k > 0 || ks > 0 ? 1u : 0u);
            umma_f16_ss(small, a_l + ao, b_h + bo, idesc, 1u);
          }
          umma_commit(&bar_empty[s]);
          if (k % MU_SUM == MU_SUM - 1 || k == steps - 1) {
            umma_commit(&bar_done[place]);
            j++;
          }
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    uint32_t j = 0, turn = 0;
    for (long long tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, turn ^= 1u) {
      const MuonTile m = mu_tile<KIND>(l, tile);
      const MuonTensor& t = l.t[m.which];
      const int M = t.mm, N = KIND == 2 ? t.nn : t.mm;
      const int steps = ((KIND == 0 ? t.nn : t.mm) + MU_BK - 1) / MU_BK, sums = (steps + MU_SUM - 1) / MU_SUM;
      const int r = m.r0 + (warp & 3) * 32 + lane, first = (warp >> 2) * 64;
      const uint32_t t_lane = tmem + (uint32_t)first + ((uint32_t)((warp & 3) * 32) << 16);
      const MuonPlanes& out = KIND == 0 ? t.gram : KIND == 1 ? t.poly : t.x2;
      const MuonPlanes& in = KIND == 1 ? t.gram : t.x;
      const int row0 = m.r0 + (warp & 3) * 32;
      uint4* stage = reinterpret_cast<uint4*>(smem + MU_TURN) + warp * 32 * MU_PITCH;
      auto wait = [&]() {
        if (lane == 0) ok = mbar_wait(&bar_done[j & 1u], (j >> 1) & 1u, abort_flag, l.status, 103);
        __syncwarp();                                    // what the lane waited for is seen by the others: a vote orders no memory
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      };
      auto read = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&bar_read[j & 1u])) : "memory");
      };
      // What the result adds to is fetched a block of 32 columns ahead, the first one under the products.
      MuonBlock next;
      if (KIND != 0) mu_fetch(in, row0, M, m.c0 + first, N, lane, next);
      wait();
      if (sums > 1) {
        // Added up in fp32, and what comes out put back in the place of the last, so that long and short sums end alike.
        float sum[64];
#pragma unroll
        for (int u = 0; u < 64; u++) sum[u] = 0.f;
        for (int q = 1; ok; q++) {
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t acc[32];
            tmem_ld_32x32b_x32(t_lane + (j & 1u) * MU_BM + (uint32_t)c, acc);
            tmem_ld_wait();
#pragma unroll
            for (int u = 0; u < 32; u++) sum[c + u] += __uint_as_float(acc[u]);
          }
          if (q == sums) break;
          read();
          j++;
          wait();
        }
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t acc[32];
#pragma unroll
          for (int u = 0; u < 32; u++) acc[u] = __float_as_uint(sum[c + u]);
          tmem_st_32x32b_x32(t_lane + (j & 1u) * MU_BM + (uint32_t)c, acc);
        }
        tmem_st_wait();
      }
      if (!ok) break;
#pragma unroll 1
      for (int b = 0; b < 64; b += 32) {
        const int col = m.c0 + first + b;
        if (col >= N) break;                             // the same for the whole warp
        uint32_t acc[32], small[32];
        __syncwarp();
        tmem_ld_32x32b_x32(t_lane + (j & 1u) * MU_BM + (uint32_t)b, acc);
        tmem_ld_32x32b_x32(t_lane + (2 + turn) * MU_BM + (uint32_t)b, small);
        tmem_ld_wait();
        uint4 vh[4], vl[4];
        if (KIND != 0) {
          mu_to_rows(stage, lane, next.h, vh);
          mu_to_rows(stage, lane, next.l, vl);
          if (b == 0) mu_fetch(in, row0, M, col + 32, N, lane, next);
        }
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int u = 0; u < 32; u += 2) {
          __half h[2], w[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float x = __uint_as_float(acc[u + e]) + __uint_as_float(small[u + e]);
            const float y = KIND == 0 ? x * (MU_SG / (MU_SX * MU_SX))
                            : KIND == 1 ? fmaf(MU_C / MU_SG, x, MU_B * mu_value(vh, vl, u + e)) : fmaf(1.f / MU_SG, x, MU_A * mu_value(vh, vl, u + e));
            mu_split(y, &h[e], &w[e]);
          }
          hi[u / 2] = (uint32_t)__half_as_ushort(h[0]) | (uint32_t)__half_as_ushort(h[1]) << 16;
          lo[u / 2] = (uint32_t)__half_as_ushort(w[0]) | (uint32_t)__half_as_ushort(w[1]) << 16;
        }
        mu_put(stage, lane, hi, out.p, out.ld, row0, M, col, N);
        mu_put(stage, lane, lo, out.p + out.plane, out.ld, row0, M, col, N);
        if (r < M) {
          if (KIND != 2 && col / MU_BM < m.r0 / MU_BM) {
            // Mirrored: the lanes of a warp are adjacent there.
#pragma unroll
            for (int u = 0; u < 32; u++) {
              if (col + u >= N) break;
              const long long to = (long long)(col + u) * out.ld + r;
              out.p[to] = __ushort_as_half((unsigned short)(hi[u / 2] >> (16 * (u & 1))));
              out.p[out.plane + to] = __ushort_as_half((unsigned short)(lo[u / 2] >> (16 * (u & 1))));
            }
          }
        }
      }
      read();
      j++;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MU_EPI) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Map of planes [2][rows][cols]: boxes of 64 columns by `box_rows` rows, zeros behind the matrix.
static bool mu_map(CUtensorMap* map, const MuonPlanes& x, int rows, int cols, int box_rows) {
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 2};
  cuuint64_t strides[2] = {(cuuint64_t)x.ld * 2, (cuuint64_t)x.plane * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, x.p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename F>
static int64_t mu_items(MuonList& l, F items) {
  long long end = 0;
  for (int i = 0; i < l.count; i++) l.end[i] = end += items(l.t[i]);
  return end;
}

// Tiles of 128 x 256 gain nothing: twice as many sums a thread are read back no faster than they are made. One square matrix, five steps, those
// against these: 1024 287 and 292 us, 2048 565 and 567, 4096 4080 and 3870.
template <int KIND>
static int32_t mu_product(om_ctx* ctx, MuonList& l, const MuonMaps& maps) {
  const int64_t n = mu_items(l, [](const MuonTensor& t) {
    const int64_t rb = ceil_div(t.mm, MU_BM);
    return KIND == 2 ? rb * ceil_div(t.nn, MU_BM) : rb * (rb + 1) / 2;
  });
  OM_CUDA(ctx, cudaFuncSetAttribute(muon_product_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, MU_SMEM));
  launch_chained(ctx, muon_product_kernel<KIND>, (unsigned)std::min<int64_t>(n, ctx->sm_count), MU_THREADS, MU_SMEM, l, maps);
  return OM_OK;
}

}  // namespace om

using namespace om;

extern "C" {

int32_t om_optim_muon_step(om_ctx* ctx, int32_t n_tensors, float* const* p_host, const float* const* g_host, float* const* m_host,
                           uint16_t* const* p16_host, const int32_t* rows_host, const int32_t* cols_host, const om_muon_hyper* hyper_host,
                           const om_muon_hyper* hyper_dev) {
  OM_CHECK_CTX(ctx);
  if (n_tensors < 0) return fail(ctx, OM_ERR_ARG, "om_optim_muon_step: %d tensors", n_tensors);
  if (n_tensors == 0) return OM_OK;
  if (!p_host || !g_host || !m_host || !rows_host || !cols_host || !hyper_host)
    return fail(ctx, OM_ERR_ARG, "om_optim_muon_step: weights, gradients, momentum, shapes and numbers are required");
  if (hyper_host->steps < 1 || hyper_host->steps > 10) return fail(ctx, OM_ERR_ARG, "om_optim_muon_step: %d steps (1 to 10)", hyper_host->steps);
  double flops = 0, bytes = 0;
  for (int i = 0; i < n_tensors; i++) {
    const int r = rows_host[i], c = cols_host[i];
    if (r < 0 || c < 0 || r > 65536 || c > 65536) return fail(ctx, OM_ERR_SHAPE, "om_optim_muon_step: matrix %d is [%d, %d] (sides of 0 to 65536)", i, r, c);
    if (r == 0 || c == 0) continue;
    if (!p_host[i] || !g_host[i] || !m_host[i]) return fail(ctx, OM_ERR_ARG, "om_optim_muon_step: a pointer of matrix %d is missing", i);
    const double mm = std::min(r, c), nn = std::max(r, c);
    flops += hyper_host->steps * (4.0 * mm * mm * nn + 2.0 * mm * mm * mm);
    bytes += 20.0 * mm * nn;
  }
  // Two matrices over one memory would be updated at the same time: refused.
  struct Span {
    uintptr_t begin, end;
    bool written;
  };
  std::vector<Span> spans;
  for (int i = 0; i < n_tensors; i++) {
    const size_t n = (size_t)rows_host[i] * (size_t)cols_host[i];
    if (n == 0) continue;
    auto span = [&](const void* p, size_t size, bool written) { spans.push_back(Span{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + n * size, written}); };
    span(p_host[i], 4, true);
    span(m_host[i], 4, true);
    span(g_host[i], 4, false);
    if (p16_host && p16_host[i]) span(p16_host[i], 2, true);
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t end = 0, end_written = 0;
  for (const Span& s : spans) {
    if (s.begin < (s.written ? end : end_written)) return fail(ctx, OM_ERR_ARG, "om_optim_muon_step: weights, momentum and gradients overlap");
    end = std::max(end, s.end);
    if (s.written) end_written = std::max(end_written, s.end);
  }
  ProfileScope prof(ctx, "om_optim_muon_step", flops, bytes);
  // The longest sums first, so that no CTA begins one when the others are done (each matrix's result is its own).
  std::vector<int> order(n_tensors);
  for (int i = 0; i < n_tensors; i++) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return std::max(rows_host[a], cols_host[a]) > std::max(rows_host[b], cols_host[b]); });
  for (int next = 0; next < n_tensors;) {
    MuonList l = {};
    l.hyper = *hyper_host;
    l.hyper_dev = hyper_dev;
    l.status = ctx->status_dev;
    std::vector<size_t> offset;
    size_t total = 0;
    auto room = [&](size_t n) {
      const size_t o = total;
      total += (n + 255) & ~(size_t)255;
      return o;
    };
    for (; next < n_tensors && l.count < MU_TENSORS; next++) {
      const int at = order[next];
      if (rows_host[at] == 0 || cols_host[at] == 0) continue;
      MuonTensor& t = l.t[l.count++];
      t.p = p_host[at]; t.g = g_host[at]; t.m = m_host[at]; t.p16 = p16_host ? p16_host[at] : nullptr;
      t.rows = rows_host[at]; t.cols = cols_host[at];
      t.mm = std::min(t.rows, t.cols); t.nn = std::max(t.rows, t.cols);
      t.quads = t.cols % 4 == 0 && ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g) | reinterpret_cast<uintptr_t>(t.m)) & 15) == 0 &&
                (reinterpret_cast<uintptr_t>(t.p16) & 7) == 0;
      t.x.ld = t.x2.ld = (t.nn + 7) & ~7;                // 16-byte pitches: what TMA addresses
      t.gram.ld = t.poly.ld = (t.mm + 7) & ~7;
      t.x.plane = t.x2.plane = (long long)t.mm * t.x.ld;
      t.gram.plane = t.poly.plane = (long long)t.mm * t.gram.ld;
      const size_t x = 4 * (size_t)t.x.plane, g = 4 * (size_t)t.gram.plane;
      for (size_t n : {x, x, g, g, 8 * (size_t)ceil_div((int64_t)t.mm * t.nn, MU_CHUNK)}) offset.push_back(room(n));
    }
    if (l.count == 0) break;
    char* work = nullptr;
    OM_TRY(pool_alloc(ctx, total, false, (void**)&work));
    MuonMaps gram, poly, apply[2];
    bool mapped = encode_fn() != nullptr;
    for (int i = 0; i < l.count && mapped; i++) {
      MuonTensor& t = l.t[i];
      const size_t* o = offset.data() + 5 * i;
      t.x.p = (__half*)(work + o[0]); t.x2.p = (__half*)(work + o[1]); t.gram.p = (__half*)(work + o[2]); t.poly.p = (__half*)(work + o[3]);
      t.partial = (double*)(work + o[4]);
      mapped = mu_map(&poly.a[i], t.gram, t.mm, t.mm, MU_BM) && mu_map(&apply[0].a[i], t.poly, t.mm, t.mm, MU_BM) &&
               mu_map(&apply[0].b[i], t.x, t.mm, t.nn, MU_BK) && mu_map(&apply[1].b[i], t.x2, t.mm, t.nn, MU_BK) &&
               mu_map(&gram.a[i], t.x, t.mm, t.nn, MU_BM) && mu_map(&gram.b[i], t.x2, t.mm, t.nn, MU_BM);
      if (mapped) {
        apply[1].a[i] = apply[0].a[i];
        poly.b[i] = poly.a[i];
      }
    }
    int32_t st = mapped ? OM_OK : fail(ctx, OM_ERR_CUDA, "cuTensorMapEncodeTiled failed for om_optim_muon_step");
    if (st == OM_OK) {
      int64_t n = mu_items(l, [](const MuonTensor& t) { return ceil_div((int64_t)t.rows * t.cols, MU_CHUNK); });
      launch_chained(ctx, muon_momentum_kernel, (unsigned)n, 256, 0, l);
      auto blocks = [](const MuonTensor& t) { return ceil_div(t.rows, 64) * ceil_div(t.cols, 64); };
      n = mu_items(l, blocks);
      launch_chained(ctx, muon_start_kernel, (unsigned)n, 256, 0, l);
      for (int s = 0; s < hyper_host->steps && st == OM_OK; s++) {
        st = mu_product<0>(ctx, l, gram);
        if (st == OM_OK) st = mu_product<1>(ctx, l, poly);
        if (st == OM_OK) st = mu_product<2>(ctx, l, apply[s & 1]);
        for (int i = 0; i < l.count; i++) {
          std::swap(l.t[i].x, l.t[i].x2);
          std::swap(gram.a[i], gram.b[i]);
        }
      }
      if (st == OM_OK) {
        n = mu_items(l, blocks);
        launch_chained(ctx, muon_finish_kernel, (unsigned)n, 256, 0, l);
      }
    }
    pool_free(ctx, work);
    OM_TRY(st);
    OM_LAUNCH_CHECK(ctx, "om_optim_muon_step");
  }
  return OM_OK;
}

}  // extern "C"
