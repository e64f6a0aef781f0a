// The Muon update: momentum, orthogonalisation of the update by Newton-Schulz steps, weight decay and the weights.
//
// A matrix is worked on as X [m, n] with m <= n (transposed where it is taller). One step is
//   G = X X^T,  Y = -4.7750 G + 2.0315 G G,  X' = 3.4445 X + Y X,
// three products; G and Y are symmetric, so the tiles above the diagonal are mirrored instead of computed. All matrices of a
// call go through each launch together: a launch covers the tiles of one product of up to MU_TENSORS matrices, whatever their
// shapes, so a step costs three launches for a whole model.
#include <cuda_bf16.h>
#include <math.h>

#include <vector>

#include "om_common.cuh"

namespace om {

constexpr int MU_TENSORS = 32;
constexpr float MU_A = 3.4445f, MU_B = -4.7750f, MU_C = 2.0315f;   // the quintic's coefficients
constexpr int MU_CHUNK = 8192;                                     // elements of one partial sum of squares
constexpr int MU_T = 64;                                           // tile

struct MuonTensor {
  float *p, *m;
  const float* g;
  uint16_t* p16;
  int rows, cols;        // as the caller has them
  float *x, *x2, *gram, *poly;   // [mm, nn], [mm, nn], [mm, mm], [mm, mm] with mm <= nn
  double* partial;       // [ceil(rows * cols / MU_CHUNK)]
  int mm, nn;
};
struct MuonList {
  om_muon_hyper hyper;
  const om_muon_hyper* hyper_dev;
  int count;
  long long end[MU_TENSORS];      // work items of this launch up to and with tensor i
  MuonTensor t[MU_TENSORS];
};
__device__ __forceinline__ om_muon_hyper mu_hyper(const MuonList& l) { return l.hyper_dev ? *l.hyper_dev : l.hyper; }
__device__ __forceinline__ int mu_find(const MuonList& l, long long item, long long* local) {
  int i = 0;
  while (item >= l.end[i]) i++;
  *local = item - (i ? l.end[i - 1] : 0);
  return i;
}

// m = momentum m + (1 - momentum) g, and the sum of squares of u over this chunk (in double: the chunks of a large matrix
// differ by orders of magnitude in what they add).
__global__ void __launch_bounds__(256) muon_momentum_kernel(const __grid_constant__ MuonList l) {
  long long chunk;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &chunk)];
  const om_muon_hyper h = mu_hyper(l);
  const long long n = (long long)t.rows * t.cols, e0 = chunk * MU_CHUNK, e1 = min(e0 + MU_CHUNK, n);
  double sum = 0.0;
  for (long long e = e0 + threadIdx.x; e < e1; e += 256) {
    const float g = t.g[e] * h.grad_scale * (1.f - h.momentum), m = fmaf(t.m[e], h.momentum, g);
    t.m[e] = m;
    const float u = h.nesterov ? fmaf(m, h.momentum, g) : m;
    sum += (double)u * u;
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

// X = u / max(|u|, eps), transposed where the matrix is taller than wide.
__global__ void __launch_bounds__(256) muon_start_kernel(const __grid_constant__ MuonList l) {
  long long chunk;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &chunk)];
  const om_muon_hyper h = mu_hyper(l);
  const long long n = (long long)t.rows * t.cols, chunks = (n + MU_CHUNK - 1) / MU_CHUNK;
  __shared__ double s[8];
  double sum = 0.0;
  for (long long c = threadIdx.x; c < chunks; c += 256) sum += t.partial[c];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < 8; w++) sum += s[w];
  const float norm = fmaxf((float)sqrt(sum), h.eps);
  const long long e1 = min(chunk * MU_CHUNK + MU_CHUNK, n);
  for (long long e = chunk * MU_CHUNK + threadIdx.x; e < e1; e += 256) {
    const float m = t.m[e], u = h.nesterov ? fmaf(m, h.momentum, t.g[e] * h.grad_scale * (1.f - h.momentum)) : m;
    const long long o = t.rows > t.cols ? e % t.cols * t.rows + e / t.cols : e;
    t.x[o] = u / norm;
  }
}

// One product of a step over every matrix. KIND 0: gram = x x^T; 1: poly = B gram + C gram gram; 2: x2 = A x + poly x.
template <int KIND>
__global__ void __launch_bounds__(256) muon_product_kernel(const __grid_constant__ MuonList l) {
  long long tile;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &tile)];
  const int M = t.mm, N = KIND == 2 ? t.nn : t.mm, K = KIND == 0 ? t.nn : t.mm;
  const int tiles_n = (N + MU_T - 1) / MU_T;
  const int r0 = (int)(tile / tiles_n) * MU_T, c0 = (int)(tile % tiles_n) * MU_T;
  const float *A = KIND == 0 ? t.x : KIND == 1 ? t.gram : t.poly, *B = KIND == 1 ? t.gram : t.x;
  const int lda = K, ldb = KIND == 0 ? K : N;
  __shared__ float As[16][MU_T + 4], Bs[16][MU_T + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int e = threadIdx.x; e < 16 * MU_T; e += 256) {
      const int r = e >> 4, k = e & 15;
      As[k][r] = r0 + r < M && k0 + k < K ? A[(long long)(r0 + r) * lda + k0 + k] : 0.f;
      if (KIND == 0) {
        Bs[k][r] = c0 + r < N && k0 + k < K ? B[(long long)(c0 + r) * ldb + k0 + k] : 0.f;
      } else {
        const int c = e & 63, kk = e >> 6;
        Bs[kk][c] = c0 + c < N && k0 + kk < K ? B[(long long)(k0 + kk) * ldb + c0 + c] : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; k++)
#pragma unroll
      for (int a = 0; a < 4; a++)
#pragma unroll
        for (int b = 0; b < 4; b++) acc[a][b] = fmaf(As[k][ty * 4 + a], Bs[k][tx * 4 + b], acc[a][b]);
    __syncthreads();
  }
  for (int a = 0; a < 4; a++)
    for (int b = 0; b < 4; b++) {
      const int r = r0 + ty * 4 + a, c = c0 + tx * 4 + b;
      if (r >= M || c >= N) continue;
      const long long o = (long long)r * N + c;
      if (KIND == 0) t.gram[o] = acc[a][b];
      if (KIND == 1) t.poly[o] = fmaf(MU_C, acc[a][b], MU_B * t.gram[o]);
      if (KIND == 2) t.x2[o] = fmaf(MU_A, t.x[o], acc[a][b]);
    }
}

// p = (1 - lr weight_decay) p - lr s X, with the bfloat16 copy where it is wanted.
__global__ void __launch_bounds__(256) muon_finish_kernel(const __grid_constant__ MuonList l) {
  long long chunk;
  const MuonTensor& t = l.t[mu_find(l, blockIdx.x, &chunk)];
  const om_muon_hyper h = mu_hyper(l);
  const float s = h.match_rms ? 0.2f * sqrtf((float)max(t.rows, t.cols)) : sqrtf(fmaxf(1.f, (float)t.rows / (float)t.cols));
  const float keep = 1.f - h.lr * h.weight_decay, rate = h.lr * s;
  const long long n = (long long)t.rows * t.cols, e1 = min(chunk * MU_CHUNK + MU_CHUNK, n);
  for (long long e = chunk * MU_CHUNK + threadIdx.x; e < e1; e += 256) {
    const long long o = t.rows > t.cols ? e % t.cols * t.rows + e / t.cols : e;
    const float p = fmaf(-rate, t.x[o], t.p[e] * keep);
    t.p[e] = p;
    if (t.p16) {
      const __nv_bfloat16 v = __float2bfloat16_rn(p);
      t.p16[e] = *reinterpret_cast<const uint16_t*>(&v);
    }
  }
}

template <typename F>
static int64_t mu_items(MuonList& l, F items) {
  long long end = 0;
  for (int i = 0; i < l.count; i++) l.end[i] = end += items(l.t[i]);
  return end;
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
  ProfileScope prof(ctx, "om_optim_muon_step", flops, bytes);
  for (int at = 0; at < n_tensors;) {
    MuonList l = {};
    l.hyper = *hyper_host;
    l.hyper_dev = hyper_dev;
    std::vector<size_t> offset;
    size_t total = 0;
    auto room = [&](size_t n) {
      const size_t o = total;
      total += (n + 255) & ~(size_t)255;
      return o;
    };
    for (; at < n_tensors && l.count < MU_TENSORS; at++) {
      if (rows_host[at] == 0 || cols_host[at] == 0) continue;
      MuonTensor& t = l.t[l.count++];
      t.p = p_host[at]; t.g = g_host[at]; t.m = m_host[at]; t.p16 = p16_host ? p16_host[at] : nullptr;
      t.rows = rows_host[at]; t.cols = cols_host[at];
      t.mm = std::min(t.rows, t.cols); t.nn = std::max(t.rows, t.cols);
      const size_t mn = (size_t)t.mm * t.nn, mm = (size_t)t.mm * t.mm;
      for (size_t n : {4 * mn, 4 * mn, 4 * mm, 4 * mm, 8 * ((mn + MU_CHUNK - 1) / MU_CHUNK)}) offset.push_back(room(n));
    }
    if (l.count == 0) break;
    char* work = nullptr;
    OM_TRY(pool_alloc(ctx, total, false, (void**)&work));
    for (int i = 0; i < l.count; i++) {
      MuonTensor& t = l.t[i];
      const size_t* o = offset.data() + 5 * i;
      t.x = (float*)(work + o[0]); t.x2 = (float*)(work + o[1]); t.gram = (float*)(work + o[2]); t.poly = (float*)(work + o[3]);
      t.partial = (double*)(work + o[4]);
    }
    auto chunks = [](const MuonTensor& t) { return ceil_div((int64_t)t.rows * t.cols, MU_CHUNK); };
    auto square = [](const MuonTensor& t) { return ceil_div(t.mm, MU_T) * ceil_div(t.mm, MU_T); };
    auto wide = [](const MuonTensor& t) { return ceil_div(t.mm, MU_T) * ceil_div(t.nn, MU_T); };
    int64_t n = mu_items(l, chunks);
    muon_momentum_kernel<<<(unsigned)n, 256, 0, ctx->stream>>>(l);
    muon_start_kernel<<<(unsigned)n, 256, 0, ctx->stream>>>(l);
    for (int s = 0; s < hyper_host->steps; s++) {
      n = mu_items(l, square);
      muon_product_kernel<0><<<(unsigned)n, 256, 0, ctx->stream>>>(l);
      muon_product_kernel<1><<<(unsigned)n, 256, 0, ctx->stream>>>(l);
      n = mu_items(l, wide);
      muon_product_kernel<2><<<(unsigned)n, 256, 0, ctx->stream>>>(l);
      for (int i = 0; i < l.count; i++) std::swap(l.t[i].x, l.t[i].x2);
    }
    n = mu_items(l, chunks);
    muon_finish_kernel<<<(unsigned)n, 256, 0, ctx->stream>>>(l);
    pool_free(ctx, work);
    OM_LAUNCH_CHECK(ctx, "om_optim_muon_step");
  }
  return OM_OK;
}

}  // extern "C"
