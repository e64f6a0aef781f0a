// Attention by rule, forward and backward, with fp32 products: the calls of om_rule_attention_* that the tensor-pipe kernels do not
// take (short or oddly shaped fp32 calls, heads beyond 64 columns in fp32, fp32 heads whose values lie too far apart for two
// half-precision numbers, bfloat16 layouts that a tile copy cannot address). The host side of both is here.
//
// One pass over the keys with the running maximum and sum of the softmax: a CTA holds a tile of queries and walks the tiles of
// keys that the rule lets it see, so neither scores nor mask exist in memory. The backward recomputes the weights from the
// forward's log-sum-exp, once for the gradients of the keys (a CTA per tile of keys walks the queries of all heads that share
// them, in increasing order) and once for those of the queries: two walks instead of partial sums in memory or atomics, whose
// order would change the result. Everything is fp32: an FMA lane is what bounds it (4 d or 14 d operations per visible pair).
#include <cuda_bf16.h>
#include <limits.h>
#include <math.h>

#include "om_rule.cuh"

namespace om {

template <typename T>
__device__ __forceinline__ float ra_value(T v);
template <>
__device__ __forceinline__ float ra_value(float v) { return v; }
template <>
__device__ __forceinline__ float ra_value(__nv_bfloat16 v) { return __bfloat162float(v); }

// Lowest and highest document of every 64 rows, the document itself where there is only one and no padding, and which rows are padding.
__global__ void __launch_bounds__(64)
rule_ranges_kernel(const int32_t* docs, int l, int tiles, int4* __restrict__ ranges, uint2* __restrict__ pads) {
  pdl_enter();
  __shared__ int lo_s[2], hi_s[2], pad_s[2];
  const int t = blockIdx.x, b = blockIdx.y, i = t * RULE_GRAIN + threadIdx.x;
  int lo = INT_MAX, hi = -1, pad = 0;
  if (i < l) {
    const int v = docs[(long long)b * l + i];
    if (v >= 0) lo = hi = v;
    else pad = 1;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  pad = (int)__ballot_sync(0xffffffffu, pad != 0);
  if ((threadIdx.x & 31) == 0) {
    lo_s[threadIdx.x >> 5] = lo;
    hi_s[threadIdx.x >> 5] = hi;
    pad_s[threadIdx.x >> 5] = pad;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    lo = min(lo_s[0], lo_s[1]);
    hi = max(hi_s[0], hi_s[1]);
    ranges[(long long)b * tiles + t] = make_int4(lo, hi, (lo == hi && !(pad_s[0] | pad_s[1])) ? lo : -1, (pad_s[0] | pad_s[1]) != 0);
    pads[(long long)b * tiles + t] = make_uint2((uint32_t)pad_s[0], (uint32_t)pad_s[1]);
  }
}

int32_t rule_check(om_ctx* ctx, const char* who, const om_attention_rule* rule, int b, int h, int hkv, int lq, int lk, int d, float scale) {
  if (!rule) return fail(ctx, OM_ERR_ARG, "%s: a rule is required", who);
  if (b < 0 || h < 0 || hkv < 0 || lq < 0 || lk < 0 || lq >= (1 << 30) || lk >= (1 << 30))
    return fail(ctx, OM_ERR_SHAPE, "%s: b %d h %d hkv %d lq %d lk %d", who, b, h, hkv, lq, lk);
  if (d < 1 || d > 256) return fail(ctx, OM_ERR_UNSUPPORTED, "%s: head dimension %d (1 to 256 are built)", who, d);
  if (h > 0 && (hkv == 0 || h % hkv)) return fail(ctx, OM_ERR_SHAPE, "%s: %d query heads do not share %d key heads evenly", who, h, hkv);
  if ((int64_t)b * h > 65535) return fail(ctx, OM_ERR_UNSUPPORTED, "%s: more than 65535 heads in one call", who);
  if ((int64_t)b * h * (((int64_t)lq + 127) / 128 * 128) > INT_MAX) return fail(ctx, OM_ERR_UNSUPPORTED, "%s: more than 2^31 rows in one call", who);
  if (!isfinite(scale)) return fail(ctx, OM_ERR_ARG, "%s: the scale must be finite", who);
  if (rule->window < 0) return fail(ctx, OM_ERR_ARG, "%s: a negative window", who);
  if (rule->q_offset < -(1 << 30) || rule->q_offset > (1 << 30)) return fail(ctx, OM_ERR_ARG, "%s: q_offset %d is beyond 2^30", who, rule->q_offset);
  if (!(rule->softcap >= 0.f) || !isfinite(rule->softcap)) return fail(ctx, OM_ERR_ARG, "%s: the cap must be positive and finite, or 0 for none", who);
  if ((rule->q_documents == nullptr) != (rule->k_documents == nullptr))
    return fail(ctx, OM_ERR_ARG, "%s: documents are given for the queries and the keys or for neither", who);
  return OM_OK;
}
int32_t rule_operand(om_ctx* ctx, const char* who, const void* p, const om_head_strides* s, int d) {
  if (!p) return fail(ctx, OM_ERR_ARG, "%s: a tensor is missing", who);
  if (!s || s->row < d || s->batch < 0 || s->head < 0)
    return fail(ctx, OM_ERR_SHAPE, "%s: rows of an activation must be at least d = %d elements apart and strides non-negative", who, d);
  return OM_OK;
}
int32_t rule_result(om_ctx* ctx, const char* who, const om_head_strides* s, int b, int h, int l, int d) {
  if (l == 0) return OM_OK;     // nothing is written: strides of an empty tensor may be anything
  if (!s || s->row < d || s->batch < 0 || s->head < 0)
    return fail(ctx, OM_ERR_SHAPE, "%s: rows of a result must be at least d = %d elements apart and strides non-negative", who, d);
  if (heads_overlap(*s, b, h, l, d)) return fail(ctx, OM_ERR_SHAPE, "%s: rows of a result overlap", who);
  return OM_OK;
}

int32_t rule_begin(om_ctx* ctx, const om_attention_rule* rule, int b, int h, int hkv, int lq, int lk, int d, float scale, RuleCall* call) {
  RuleArgs& r = call->r;
  r.causal = rule->causal != 0;
  r.window = rule->window;
  r.q_offset = rule->q_offset;
  r.softcap = rule->softcap;
  r.inv_softcap = rule->softcap > 0.f ? 1.f / rule->softcap : 0.f;
  r.scale = scale;
  r.slopes = rule->slopes;
  r.prefix = rule->prefix;
  r.q_docs = rule->q_documents;
  r.k_docs = rule->k_documents;
  r.q_ranges = r.k_ranges = nullptr;
  r.q_pads = r.k_pads = nullptr;
  r.lq = lq;
  r.lk = lk;
  r.nq64 = (lq + RULE_GRAIN - 1) / RULE_GRAIN;
  r.nk64 = (lk + RULE_GRAIN - 1) / RULE_GRAIN;
  call->b = b; call->h = h; call->hkv = hkv; call->d = d;
  call->ranges = nullptr;
  if (r.q_docs && lk > 0) {
    const size_t nq = (size_t)b * r.nq64, n = nq + (size_t)b * r.nk64;
    OM_TRY(pool_alloc(ctx, (sizeof(int4) + sizeof(uint2)) * n, false, (void**)&call->ranges));
    uint2* pads = reinterpret_cast<uint2*>(call->ranges + n);
    launch_chained(ctx, rule_ranges_kernel, dim3((unsigned)r.nq64, (unsigned)b), 64, 0, r.q_docs, lq, r.nq64, call->ranges, pads);
    launch_chained(ctx, rule_ranges_kernel, dim3((unsigned)r.nk64, (unsigned)b), 64, 0, r.k_docs, lk, r.nk64, call->ranges + nq, pads + nq);
    r.q_ranges = call->ranges;
    r.k_ranges = call->ranges + nq;
    r.q_pads = pads;
    r.k_pads = pads + nq;
  }
  return OM_OK;
}
void rule_end(om_ctx* ctx, RuleCall* call) {
  if (call->ranges) pool_free(ctx, call->ranges);
}

struct RaStrides {
  long long batch, head, row;
};
static RaStrides ra_strides(const om_head_strides* s) { return RaStrides{s->batch, s->head, s->row}; }

// A tile of BM rows, zero beyond the tensor's rows and columns and in rows of no document, as fp32 with DP + 4 floats a row: rows a quarter apart in the
// banks, so that 16 threads reading 16 rows at one column, 16 bytes each, meet no conflict.
template <typename T, int BM, int DP>
__device__ __forceinline__ void ra_load(float* dst, const T* base, long long row_stride, int row0, int rows, int d, bool vec, const int32_t* docs) {
  if (vec) {
    constexpr int N = 4;
    for (int e = threadIdx.x; e < BM * (DP / N); e += 256) {
      const int r = e / (DP / N), c = (e % (DP / N)) * N;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row0 + r < rows && c < d && !(docs && docs[row0 + r] < 0)) {
        if (sizeof(T) == 4) {
          v = *reinterpret_cast<const float4*>(base + (long long)(row0 + r) * row_stride + c);
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(base + (long long)(row0 + r) * row_stride + c);
          v = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
        }
      }
      *reinterpret_cast<float4*>(dst + r * (DP + 4) + c) = v;
    }
  } else {
    for (int e = threadIdx.x; e < BM * DP; e += 256) {
      const int r = e / DP, c = e % DP;
      dst[r * (DP + 4) + c] = (row0 + r < rows && c < d && !(docs && docs[row0 + r] < 0)) ? ra_value<T>(base[(long long)(row0 + r) * row_stride + c]) : 0.f;
    }
  }
}

// acc[a][b] += rows (16 rows apart in b) of Y times rows of X over the head's columns.
template <int R, int DP>
__device__ __forceinline__ void ra_scores(const float* X, const float* Y, int ty, int tx, float (&acc)[R][R]) {
#pragma unroll
  for (int a = 0; a < R; a++)
#pragma unroll
    for (int c = 0; c < R; c++) acc[a][c] = 0.f;
#pragma unroll 4
  for (int k = 0; k < DP; k += 4) {
    float4 x[R], y[R];
#pragma unroll
    for (int a = 0; a < R; a++) x[a] = *reinterpret_cast<const float4*>(X + (ty * R + a) * (DP + 4) + k);
#pragma unroll
    for (int c = 0; c < R; c++) y[c] = *reinterpret_cast<const float4*>(Y + (tx + 16 * c) * (DP + 4) + k);
#pragma unroll
    for (int a = 0; a < R; a++)
#pragma unroll
      for (int c = 0; c < R; c++) {
        acc[a][c] = fmaf(x[a].x, y[c].x, acc[a][c]);
        acc[a][c] = fmaf(x[a].y, y[c].y, acc[a][c]);
        acc[a][c] = fmaf(x[a].z, y[c].z, acc[a][c]);
        acc[a][c] = fmaf(x[a].w, y[c].w, acc[a][c]);
      }
  }
}

// Columns of a result that thread tx holds: VW adjacent ones every 16 * VW.
template <int DP>
struct RaCols {
  static constexpr int VW = DP >= 64 ? 4 : 2, GROUPS = DP / (16 * VW), N = VW * GROUPS;
};
// acc[a][:] += sum over j of W(ty * R + a, j) V[j][:]; TRANSPOSED reads W[j][ty * R + a].
template <int BM, int DP, bool TRANSPOSED>
__device__ __forceinline__ void ra_product(const float* W, const float* V, int ty, int tx, float (&acc)[BM / 16][RaCols<DP>::N]) {
  constexpr int R = BM / 16, VW = RaCols<DP>::VW, G = RaCols<DP>::GROUPS, LW = BM + 4;
#pragma unroll 2
  for (int j = 0; j < BM; j++) {
    float w[R];
#pragma unroll
    for (int a = 0; a < R; a++) w[a] = TRANSPOSED ? W[j * LW + ty * R + a] : W[(ty * R + a) * LW + j];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int u = 0; u < VW; u++) {
        const float v = V[j * (DP + 4) + tx * VW + 16 * VW * g + u];
#pragma unroll
        for (int a = 0; a < R; a++) acc[a][g * VW + u] = fmaf(w[a], v, acc[a][g * VW + u]);
      }
  }
}
template <int BM, int DP>
__device__ __forceinline__ void ra_store(float* out, __nv_bfloat16* out16, const RaStrides& s, long long base, int row0, int rows, int d, int ty, int tx,
                                         const float (&acc)[BM / 16][RaCols<DP>::N], float factor) {
  constexpr int R = BM / 16, VW = RaCols<DP>::VW, G = RaCols<DP>::GROUPS;
#pragma unroll
  for (int a = 0; a < R; a++) {
    const int row = row0 + ty * R + a;
    if (row >= rows) continue;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int u = 0; u < VW; u++) {
        const int c = tx * VW + 16 * VW * g + u;
        if (c >= d) continue;
        const float v = acc[a][g * VW + u] * factor;
        if (out) out[base + (long long)row * s.row + c] = v;
        if (out16) out16[base + (long long)row * s.row + c] = __float2bfloat16_rn(v);
      }
  }
}

template <typename T>
struct RaParams {
  RuleArgs r;
  int b, h, hkv, d;
  bool vec;                       // rows of q, k, v (and of the output and its gradient) start where four elements load at once
  const T *q, *k, *v, *g, *o;
  RaStrides qs, ks, vs, gs, os;
  float *out, *lse;               // forward
  __nv_bfloat16* out16;
  const float* lse_in;            // backward
  const float* rows;              // log-sum-exps (plus infinity for a row that sees nothing) and row dots, read by rule_row
  float *dq, *dk, *dv;
  __nv_bfloat16 *dq16, *dk16, *dv16;
  RaStrides dqs, dks, dvs;
  const int32_t* plain;           // not NULL: [b * hkv], the tensor-pipe kernels in front have done the heads for which this is not set
  float unit;                     // of the log-sum-exps in `rows` (log2 e where those kernels read them too)
};

template <typename T, int BM, int DP>
__global__ void __launch_bounds__(256)
rule_attention_fwd_kernel(const __grid_constant__ RaParams<T> p) {
  if (p.plain && ld_global(p.plain + blockIdx.y / (p.h / p.hkv)) == 0) return;
  extern __shared__ __align__(16) float sm[];
  constexpr int R = BM / 16, LD = DP + 4, LW = BM + 4;
  float *Q = sm, *K = Q + BM * LD, *V = K + BM * LD, *P = V + BM * LD;
  int* kdoc = reinterpret_cast<int*>(P + BM * LW);
  const RuleArgs& r = p.r;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int i0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * BM;      // the longest rows of a causal mask first
  const int bh = blockIdx.y, bi = bh / p.h, hi = bh - bi * p.h, hk = hi / (p.h / p.hkv);
  const int prefix = r.prefix ? r.prefix[bi] : 0;
  const int32_t *q_rows = r.q_docs ? r.q_docs + (long long)bi * r.lq : nullptr, *k_rows = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
  const float slope = r.slopes ? r.slopes[hi] : 0.f;
  ra_load<T, BM, DP>(Q, p.q + bi * p.qs.batch + hi * p.qs.head, p.qs.row, i0, r.lq, p.d, p.vec, q_rows);
  float m[R], l[R], acc[R][RaCols<DP>::N];
  int qdoc[R];
#pragma unroll
  for (int a = 0; a < R; a++) {
    m[a] = -INFINITY;
    l[a] = 0.f;
    const int i = i0 + ty * R + a;
    qdoc[a] = r.q_docs && i < r.lq ? r.q_docs[(long long)bi * r.lq + i] : -1;
#pragma unroll
    for (int c = 0; c < RaCols<DP>::N; c++) acc[a][c] = 0.f;
  }
  const RuleTile tile = rule_query_tile(r, prefix, bi, i0 / RULE_GRAIN * RULE_GRAIN, 1);
  const RuleSpan span = rule_keys(r, prefix, i0, min(i0 + BM, r.lq));
  const int first = span.prefix > 0 ? 0 : span.lo / BM * BM, last = max(span.prefix, span.hi);
  for (int j0 = first; j0 < last; j0 += BM) {
    // The document ranges go by 64 rows: a tile of 32 asks for the 64 that hold it.
    if (rule_see<false>(tile, j0 / RULE_GRAIN * RULE_GRAIN, 1) == 0) continue;
    __syncthreads();
    ra_load<T, BM, DP>(K, p.k + bi * p.ks.batch + hk * p.ks.head, p.ks.row, j0, r.lk, p.d, p.vec, k_rows);
    ra_load<T, BM, DP>(V, p.v + bi * p.vs.batch + hk * p.vs.head, p.vs.row, j0, r.lk, p.d, p.vec, k_rows);
    if (r.k_docs)
      for (int e = threadIdx.x; e < BM; e += 256) kdoc[e] = j0 + e < r.lk ? r.k_docs[(long long)bi * r.lk + j0 + e] : -1;
    __syncthreads();
    float s[R][R];
    ra_scores<R, DP>(Q, K, ty, tx, s);
#pragma unroll
    for (int a = 0; a < R; a++) {
      const int i = i0 + ty * R + a;
      float top = m[a];
#pragma unroll
      for (int c = 0; c < R; c++) {
        const int j = j0 + tx + 16 * c;
        float dcap;
        const bool seen = i < r.lq && j < r.lk && rule_visible(r, prefix, i, j, qdoc[a], r.k_docs ? kdoc[tx + 16 * c] : 0);
        s[a][c] = seen ? rule_score(r, slope, i, j, s[a][c], &dcap) : -INFINITY;
        top = fmaxf(top, s[a][c]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float base = top == -INFINITY ? 0.f : top;
      const float shrink = expf(m[a] - base);       // m = -inf: 0
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < R; c++) {
        const float e = expf(s[a][c] - base);
        sum += e;
        P[(ty * R + a) * LW + tx + 16 * c] = e;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[a] = fmaf(l[a], shrink, sum);
      m[a] = top;
#pragma unroll
      for (int c = 0; c < RaCols<DP>::N; c++) acc[a][c] *= shrink;
    }
    __syncwarp();                                    // a row of P is written and read by the same half warp
    ra_product<BM, DP, false>(P, V, ty, tx, acc);
  }
#pragma unroll
  for (int a = 0; a < R; a++) {
    const int i = i0 + ty * R + a;
    const float inv = l[a] == 0.f ? 0.f : 1.f / l[a];
#pragma unroll
    for (int c = 0; c < RaCols<DP>::N; c++) acc[a][c] *= inv;
    if (p.lse && tx == 0 && i < r.lq) p.lse[(long long)bh * r.lq + i] = l[a] == 0.f ? -INFINITY : m[a] + logf(l[a]);
  }
  ra_store<BM, DP>(p.out, p.out16, p.os, bi * p.os.batch + hi * p.os.head, i0, r.lq, p.d, ty, tx, acc, 1.f);
}

// Row dots rowsum(dO o O) beside the log-sum-exp times `unit` (log2 e for the kernels that work with powers of two); rows behind
// the last query, and those that see no key, get plus infinity and 0, so that a weight recomputed from them is 0. A power of two of
// lanes per row, each with 16 bytes of dO at a time (N elements; one where rows do not start on that grid), two rows in flight per lane.
template <typename T, typename O, int N>
__global__ void __launch_bounds__(256)
rule_rows_kernel(const T* g, RaStrides gs, const O* o, RaStrides os, const float* lse, int h, int lq, int lq_pad, int d, int lanes, float unit,
                 long long total, float* __restrict__ rows) {
  pdl_enter();
  struct alignas(N * sizeof(T)) VecG {
    T v[N];
  };
  struct alignas(N == 1 ? sizeof(O) : 16) VecO {
    O v[N];
  };
  const int sub = threadIdx.x & (lanes - 1), per_cta = 256 / lanes;
  for (long long w0 = (long long)blockIdx.x * 2 * per_cta + threadIdx.x / lanes; w0 < total; w0 += (long long)gridDim.x * 2 * per_cta) {
    float dot[2] = {0.f, 0.f};
    long long at[2], bhs[2];
    int is[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      at[u] = w0 + u * per_cta;
      bhs[u] = at[u] / lq_pad;
      is[u] = at[u] < total ? (int)(at[u] - bhs[u] * lq_pad) : lq;
      if (is[u] < lq) {
        const long long bi = bhs[u] / h;
        const int hi = (int)(bhs[u] - bi * h);
        const T* gp = g + bi * gs.batch + hi * gs.head + (long long)is[u] * gs.row;
        const O* op = o + bi * os.batch + hi * os.head + (long long)is[u] * os.row;
        for (int c = sub * N; c < d; c += lanes * N) {
          const VecG a = *reinterpret_cast<const VecG*>(gp + c);
          const VecO b = *reinterpret_cast<const VecO*>(op + c);
#pragma unroll
          for (int e = 0; e < N; e++) dot[u] = fmaf(ra_value<T>(a.v[e]), ra_value<O>(b.v[e]), dot[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      for (int x = lanes >> 1; x > 0; x >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], x);
      if (sub == 0 && at[u] < total) {
        float e = is[u] < lq ? lse[bhs[u] * lq + is[u]] * unit : -INFINITY;
        if (e == -INFINITY) {
          e = INFINITY;
          dot[u] = 0.f;
        }
        rows[at[u] / 128 * 256 + at[u] % 128] = e;
        rows[at[u] / 128 * 256 + at[u] % 128 + 128] = dot[u];
      }
    }
  }
}
template <typename T, typename O>
static void launch_rows(om_ctx* ctx, const T* g, const om_head_strides* gs, const O* o, const om_head_strides* os, const float* lse, int b, int h, int lq, int d,
                        float unit, float* rows) {
  const int lq_pad = rule_row_tiles(lq) * 128;
  const long long total = (long long)b * h * lq_pad;          // a multiple of 128: no warp runs over the end alone
  constexpr int N = 16 / sizeof(T);
  auto grid16 = [&](const void* p, const om_head_strides* s) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s->row % N == 0 && s->head % N == 0 && s->batch % N == 0;
  };
  const bool vec = d % N == 0 && grid16(g, gs) && grid16(o, os);
  int lanes = 1;
  while (lanes < 32 && lanes * (vec ? N : 1) < d) lanes *= 2;
  const int grid = grid_for(ctx, total, 2 * 256 / lanes, 16);
  if (vec) launch_chained(ctx, rule_rows_kernel<T, O, N>, grid, 256, 0, g, ra_strides(gs), o, ra_strides(os), lse, h, lq, lq_pad, d, lanes, unit, total, rows);
  else launch_chained(ctx, rule_rows_kernel<T, O, 1>, grid, 256, 0, g, ra_strides(gs), o, ra_strides(os), lse, h, lq, lq_pad, d, lanes, unit, total, rows);
}

// The weights and the scores' gradients of one tile into P and S, [query][key].
template <typename T, int BM, int DP>
__device__ __forceinline__ void ra_gradients(const RaParams<T>& p, const float* Q, const float* K, const float* V, const float* G, float* P, float* S,
                                             long long bh, const int* qdoc, const int* kdoc, int prefix, float slope, int i0, int j0, int ty, int tx) {
  constexpr int R = BM / 16, LW = BM + 4;
  const RuleArgs& r = p.r;
  float s[R][R], dp[R][R];
  ra_scores<R, DP>(Q, K, ty, tx, s);
  ra_scores<R, DP>(G, V, ty, tx, dp);
#pragma unroll
  for (int a = 0; a < R; a++) {
    const int i = i0 + ty * R + a;
    const float2 row = i < r.lq ? rule_row(p.rows, bh, r.lq, i) : make_float2(INFINITY, 0.f);
#pragma unroll
    for (int c = 0; c < R; c++) {
      const int j = j0 + tx + 16 * c;
      float w = 0.f, ds = 0.f;
      if (i < r.lq && j < r.lk && rule_visible(r, prefix, i, j, r.q_docs ? qdoc[ty * R + a] : 0, r.k_docs ? kdoc[tx + 16 * c] : 0)) {
        float dcap;
        w = expf(rule_score(r, slope, i, j, s[a][c], &dcap) - row.x * p.unit);
        ds = (w * (dp[a][c] - row.y)) * dcap;
      }
      if (P) P[(ty * R + a) * LW + tx + 16 * c] = w;
      S[(ty * R + a) * LW + tx + 16 * c] = ds;
    }
  }
}

template <typename T, int BM, int DP>
__global__ void __launch_bounds__(256)
rule_attention_dkv_kernel(const __grid_constant__ RaParams<T> p) {
  if (p.plain && ld_global(p.plain + blockIdx.y) == 0) return;
  extern __shared__ __align__(16) float sm[];
  constexpr int R = BM / 16, LD = DP + 4, LW = BM + 4;
  float *K = sm, *V = K + BM * LD, *Q = V + BM * LD, *G = Q + BM * LD, *P = G + BM * LD, *S = P + BM * LW;
  int *qdoc = reinterpret_cast<int*>(S + BM * LW), *kdoc = qdoc + BM;
  const RuleArgs& r = p.r;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int j0 = (int)blockIdx.x * BM;
  const int bk = blockIdx.y, bi = bk / p.hkv, hk = bk - bi * p.hkv, group = p.h / p.hkv;
  const int prefix = r.prefix ? r.prefix[bi] : 0;
  const int32_t *q_rows = r.q_docs ? r.q_docs + (long long)bi * r.lq : nullptr, *k_rows = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
  ra_load<T, BM, DP>(K, p.k + bi * p.ks.batch + hk * p.ks.head, p.ks.row, j0, r.lk, p.d, p.vec, k_rows);
  ra_load<T, BM, DP>(V, p.v + bi * p.vs.batch + hk * p.vs.head, p.vs.row, j0, r.lk, p.d, p.vec, k_rows);
  if (r.k_docs)
    for (int e = threadIdx.x; e < BM; e += 256) kdoc[e] = j0 + e < r.lk ? r.k_docs[(long long)bi * r.lk + j0 + e] : -1;
  float dk[R][RaCols<DP>::N], dv[R][RaCols<DP>::N];
#pragma unroll
  for (int a = 0; a < R; a++)
#pragma unroll
    for (int c = 0; c < RaCols<DP>::N; c++) dk[a][c] = dv[a][c] = 0.f;
  const RuleTile tile = rule_key_tile(r, prefix, bi, j0 / RULE_GRAIN * RULE_GRAIN, 1);
  int lo, hi;
  rule_queries(r, prefix, j0, min(j0 + BM, r.lk), &lo, &hi);
  for (int gi = 0; gi < group; gi++) {
    const int head = hk * group + gi;
    const float slope = r.slopes ? r.slopes[head] : 0.f;
    for (int i0 = lo / BM * BM; i0 < hi; i0 += BM) {
      if (rule_see<false>(tile, i0 / RULE_GRAIN * RULE_GRAIN, 1) == 0) continue;
      __syncthreads();
      ra_load<T, BM, DP>(Q, p.q + bi * p.qs.batch + head * p.qs.head, p.qs.row, i0, r.lq, p.d, p.vec, q_rows);
      ra_load<T, BM, DP>(G, p.g + bi * p.gs.batch + head * p.gs.head, p.gs.row, i0, r.lq, p.d, p.vec, q_rows);
      if (r.q_docs)
        for (int e = threadIdx.x; e < BM; e += 256) qdoc[e] = i0 + e < r.lq ? r.q_docs[(long long)bi * r.lq + i0 + e] : -1;
      __syncthreads();
      ra_gradients<T, BM, DP>(p, Q, K, V, G, P, S, (long long)bi * p.h + head, qdoc, kdoc, prefix, slope, i0, j0, ty, tx);
      __syncthreads();
      ra_product<BM, DP, true>(P, G, ty, tx, dv);
      ra_product<BM, DP, true>(S, Q, ty, tx, dk);
    }
  }
  ra_store<BM, DP>(p.dv, p.dv16, p.dvs, bi * p.dvs.batch + hk * p.dvs.head, j0, r.lk, p.d, ty, tx, dv, 1.f);
  ra_store<BM, DP>(p.dk, p.dk16, p.dks, bi * p.dks.batch + hk * p.dks.head, j0, r.lk, p.d, ty, tx, dk, r.scale);
}

template <typename T, int BM, int DP>
__global__ void __launch_bounds__(256)
rule_attention_dq_kernel(const __grid_constant__ RaParams<T> p) {
  if (p.plain && ld_global(p.plain + blockIdx.y / (p.h / p.hkv)) == 0) return;
  extern __shared__ __align__(16) float sm[];
  constexpr int R = BM / 16, LD = DP + 4, LW = BM + 4;
  float *Q = sm, *G = Q + BM * LD, *K = G + BM * LD, *V = K + BM * LD, *S = V + BM * LD;
  int *qdoc = reinterpret_cast<int*>(S + BM * LW), *kdoc = qdoc + BM;
  const RuleArgs& r = p.r;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int i0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * BM;
  const int bh = blockIdx.y, bi = bh / p.h, hi = bh - bi * p.h, hk = hi / (p.h / p.hkv);
  const int prefix = r.prefix ? r.prefix[bi] : 0;
  const int32_t *q_rows = r.q_docs ? r.q_docs + (long long)bi * r.lq : nullptr, *k_rows = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
  const float slope = r.slopes ? r.slopes[hi] : 0.f;
  ra_load<T, BM, DP>(Q, p.q + bi * p.qs.batch + hi * p.qs.head, p.qs.row, i0, r.lq, p.d, p.vec, q_rows);
  ra_load<T, BM, DP>(G, p.g + bi * p.gs.batch + hi * p.gs.head, p.gs.row, i0, r.lq, p.d, p.vec, q_rows);
  if (r.q_docs)
    for (int e = threadIdx.x; e < BM; e += 256) qdoc[e] = i0 + e < r.lq ? r.q_docs[(long long)bi * r.lq + i0 + e] : -1;
  float dq[R][RaCols<DP>::N];
#pragma unroll
  for (int a = 0; a < R; a++)
#pragma unroll
    for (int c = 0; c < RaCols<DP>::N; c++) dq[a][c] = 0.f;
  const RuleTile tile = rule_query_tile(r, prefix, bi, i0 / RULE_GRAIN * RULE_GRAIN, 1);
  const RuleSpan span = rule_keys(r, prefix, i0, min(i0 + BM, r.lq));
  const int first = span.prefix > 0 ? 0 : span.lo / BM * BM, last = max(span.prefix, span.hi);
  for (int j0 = first; j0 < last; j0 += BM) {
    if (rule_see<false>(tile, j0 / RULE_GRAIN * RULE_GRAIN, 1) == 0) continue;
    __syncthreads();
    ra_load<T, BM, DP>(K, p.k + bi * p.ks.batch + hk * p.ks.head, p.ks.row, j0, r.lk, p.d, p.vec, k_rows);
    ra_load<T, BM, DP>(V, p.v + bi * p.vs.batch + hk * p.vs.head, p.vs.row, j0, r.lk, p.d, p.vec, k_rows);
    if (r.k_docs)
      for (int e = threadIdx.x; e < BM; e += 256) kdoc[e] = j0 + e < r.lk ? r.k_docs[(long long)bi * r.lk + j0 + e] : -1;
    __syncthreads();
    ra_gradients<T, BM, DP>(p, Q, K, V, G, nullptr, S, bh, qdoc, kdoc, prefix, slope, i0, j0, ty, tx);
    __syncwarp();
    ra_product<BM, DP, false>(S, K, ty, tx, dq);
  }
  ra_store<BM, DP>(p.dq, p.dq16, p.dqs, bi * p.dqs.batch + hi * p.dqs.head, i0, r.lq, p.d, ty, tx, dq, r.scale);
}

template <typename K, typename P>
static int32_t ra_launch(om_ctx* ctx, K kernel, dim3 grid, size_t smem, const P& p, const char* what) {
  OM_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<grid, 256, smem, ctx->stream>>>(p);
  OM_LAUNCH_CHECK(ctx, what);
  return OM_OK;
}

// Tiles of 64 rows; of 32 where four tiles of 64 rows of 256 columns would not fit an SM's shared memory.
template <typename T, int BM, int DP>
static int32_t ra_fwd(om_ctx* ctx, const RaParams<T>& p) {
  const size_t smem = sizeof(float) * (3 * (size_t)BM * (DP + 4) + (size_t)BM * (BM + 4) + BM);
  return ra_launch(ctx, rule_attention_fwd_kernel<T, BM, DP>, dim3((unsigned)ceil_div(p.r.lq, BM), (unsigned)(p.b * p.h)), smem, p, "om_rule_attention_fwd");
}
template <typename T, int BM, int DP>
static int32_t ra_bwd(om_ctx* ctx, const RaParams<T>& p) {
  const size_t smem = sizeof(float) * (4 * (size_t)BM * (DP + 4) + 2 * (size_t)BM * (BM + 4) + 2 * BM);
  if (p.dk || p.dv || p.dk16 || p.dv16)
    OM_TRY(ra_launch(ctx, rule_attention_dkv_kernel<T, BM, DP>, dim3((unsigned)ceil_div(p.r.lk, BM), (unsigned)(p.b * p.hkv)), smem, p, "om_rule_attention_bwd"));
  if (p.dq || p.dq16)
    OM_TRY(ra_launch(ctx, rule_attention_dq_kernel<T, BM, DP>, dim3((unsigned)ceil_div(p.r.lq, BM), (unsigned)(p.b * p.h)), smem, p, "om_rule_attention_bwd"));
  return OM_OK;
}
template <typename T>
static int32_t ra_fwd_by_width(om_ctx* ctx, const RaParams<T>& p) {
  if (p.d <= 32) return ra_fwd<T, 64, 32>(ctx, p);
  if (p.d <= 64) return ra_fwd<T, 64, 64>(ctx, p);
  if (p.d <= 128) return ra_fwd<T, 64, 128>(ctx, p);
  return ra_fwd<T, 32, 256>(ctx, p);
}
template <typename T>
static int32_t ra_bwd_by_width(om_ctx* ctx, const RaParams<T>& p) {
  if (p.d <= 32) return ra_bwd<T, 64, 32>(ctx, p);
  if (p.d <= 64) return ra_bwd<T, 64, 64>(ctx, p);
  if (p.d <= 128) return ra_bwd<T, 64, 128>(ctx, p);
  return ra_bwd<T, 32, 256>(ctx, p);
}
static bool ra_quads(const void* p, const om_head_strides* s, int size) {
  return (reinterpret_cast<uintptr_t>(p) % (4 * size)) == 0 && s->row % 4 == 0 && s->head % 4 == 0 && s->batch % 4 == 0;
}
// No keys, or no element of a gradient's heads looked at by anybody: zeros.
template <typename T>
static int32_t ra_zero(om_ctx* ctx, T* out, const om_head_strides* s, int b, int h, int l, int d);
template <typename T>
__global__ void __launch_bounds__(256) rule_zero_kernel(T* out, RaStrides s, int h, int l, int d, long long total) {
  pdl_enter();
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const int c = (int)(e % d);
    const long long row = e / d, bh = row / l;
    out[bh / h * s.batch + bh % h * s.head + row % l * s.row + c] = T(0.f);
  }
}
template <typename T>
static int32_t ra_zero(om_ctx* ctx, T* out, const om_head_strides* s, int b, int h, int l, int d) {
  if (!out) return OM_OK;
  const long long total = (long long)b * h * l * d;
  if (total == 0) return OM_OK;
  launch_chained(ctx, rule_zero_kernel<T>, grid_for(ctx, total, 256), 256, 0, out, ra_strides(s), h, l, d, total);
  OM_LAUNCH_CHECK(ctx, "om_rule_attention");
  return OM_OK;
}
__global__ void __launch_bounds__(256) rule_fill_kernel(float* out, long long total, float v) {
  pdl_enter();
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) out[e] = v;
}

template <typename T>
static int32_t rule_fwd(om_ctx* ctx, const char* who, const om_attention_rule* rule, const T* q, const om_head_strides* qs, const T* k,
                        const om_head_strides* ks, const T* v, const om_head_strides* vs, int b, int h, int hkv, int lq, int lk, int d, float scale,
                        float* out, __nv_bfloat16* out16, const om_head_strides* os, float* lse) {
  OM_TRY(rule_check(ctx, who, rule, b, h, hkv, lq, lk, d, scale));
  if ((int64_t)b * h * lq == 0) return OM_OK;
  if (!out && !out16) return fail(ctx, OM_ERR_ARG, "%s: room for the output is required", who);
  OM_TRY(rule_operand(ctx, who, q, qs, d));
  OM_TRY(rule_result(ctx, who, os, b, h, lq, d));
  if (lk == 0) {
    OM_TRY(ra_zero(ctx, out, os, b, h, lq, d));
    OM_TRY(ra_zero(ctx, out16, os, b, h, lq, d));
    if (lse) launch_chained(ctx, rule_fill_kernel, grid_for(ctx, (int64_t)b * h * lq, 256), 256, 0, lse, (long long)b * h * lq, -INFINITY);
    OM_LAUNCH_CHECK(ctx, who);
    return OM_OK;
  }
  OM_TRY(rule_operand(ctx, who, k, ks, d));
  OM_TRY(rule_operand(ctx, who, v, vs, d));
  ProfileScope prof(ctx, "om_rule_attention_fwd", 4.0 * b * h * (double)lq * lk * d, sizeof(T) * (2.0 * b * h * (double)lq * d + 2.0 * b * hkv * (double)lk * d));
  RuleCall call;
  OM_TRY(rule_begin(ctx, rule, b, h, hkv, lq, lk, d, scale, &call));
  if (sizeof(T) == 2 && rule16_fwd_takes(call, q, qs, k, ks, v, vs, out, out16, os)) {
    const int32_t st = rule16_fwd(ctx, call, q, qs, k, ks, v, vs, out, out16, os, lse, nullptr);
    rule_end(ctx, &call);
    return st;
  }
  RaParams<T> p = {};
  p.r = call.r; p.b = b; p.h = h; p.hkv = hkv; p.d = d;
  p.q = q; p.k = k; p.v = v; p.qs = ra_strides(qs); p.ks = ra_strides(ks); p.vs = ra_strides(vs);
  p.vec = d % 4 == 0 && ra_quads(q, qs, sizeof(T)) && ra_quads(k, ks, sizeof(T)) && ra_quads(v, vs, sizeof(T));
  p.out = out; p.out16 = out16; p.os = ra_strides(os); p.lse = lse;
  RulePlanes planes = {};
  int32_t st = OM_OK;
  if (sizeof(T) == 4 && rule16_planes_take(call, false) && rule16_result_fits(out, os)) {
    st = rule16_planes(ctx, call, (const float*)q, qs, (const float*)k, ks, (const float*)v, vs, nullptr, nullptr, &planes);
    if (st == OM_OK) st = rule16_fwd(ctx, call, planes.p[0], &planes.q, planes.p[1], &planes.k, planes.p[2], &planes.k, out, nullptr, os, lse, &planes);
    p.plain = planes.plain;
  }
  if (st == OM_OK) st = ra_fwd_by_width<T>(ctx, p);
  rule16_planes_end(ctx, &planes);
  rule_end(ctx, &call);
  return st;
}

template <typename T>
static int32_t rule_bwd(om_ctx* ctx, const char* who, const om_attention_rule* rule, const T* g, const om_head_strides* gs, const T* q,
                        const om_head_strides* qs, const T* k, const om_head_strides* ks, const T* v, const om_head_strides* vs, const T* out,
                        const float* out32, const om_head_strides* os, const float* lse, int b, int h, int hkv, int lq, int lk, int d, float scale, float* dq,
                        __nv_bfloat16* dq16, const om_head_strides* dqs, float* dk, __nv_bfloat16* dk16, const om_head_strides* dks, float* dv,
                        __nv_bfloat16* dv16, const om_head_strides* dvs) {
  OM_TRY(rule_check(ctx, who, rule, b, h, hkv, lq, lk, d, scale));
  if (b == 0 || hkv == 0) return OM_OK;
  if (h > 0 && (dq || dq16)) OM_TRY(rule_result(ctx, who, dqs, b, h, lq, d));
  if (dk || dk16) OM_TRY(rule_result(ctx, who, dks, b, hkv, lk, d));
  if (dv || dv16) OM_TRY(rule_result(ctx, who, dvs, b, hkv, lk, d));
  if (h == 0 || lq == 0 || lk == 0) {                      // zeros, for the key heads of no query head too
    if (lq > 0) {
      OM_TRY(ra_zero(ctx, dq, dqs, b, h, lq, d));
      OM_TRY(ra_zero(ctx, dq16, dqs, b, h, lq, d));
    }
    if (lk > 0) {
      OM_TRY(ra_zero(ctx, dk, dks, b, hkv, lk, d));
      OM_TRY(ra_zero(ctx, dk16, dks, b, hkv, lk, d));
      OM_TRY(ra_zero(ctx, dv, dvs, b, hkv, lk, d));
      OM_TRY(ra_zero(ctx, dv16, dvs, b, hkv, lk, d));
    }
    return OM_OK;
  }
  if (!lse) return fail(ctx, OM_ERR_ARG, "%s: the forward's log-sum-exp is required", who);
  OM_TRY(rule_operand(ctx, who, g, gs, d));
  OM_TRY(rule_operand(ctx, who, q, qs, d));
  OM_TRY(rule_operand(ctx, who, k, ks, d));
  OM_TRY(rule_operand(ctx, who, v, vs, d));
  OM_TRY(rule_operand(ctx, who, out32 ? (const void*)out32 : out, os, d));
  ProfileScope prof(ctx, "om_rule_attention_bwd", 10.0 * b * h * (double)lq * lk * d, sizeof(T) * (4.0 * b * h * (double)lq * d + 4.0 * b * hkv * (double)lk * d));
  RuleCall call;
  OM_TRY(rule_begin(ctx, rule, b, h, hkv, lq, lk, d, scale, &call));
  const int lq_pad = rule_row_tiles(lq) * 128;
  float* rows = nullptr;
  int32_t st = pool_alloc(ctx, 2 * sizeof(float) * (size_t)b * h * lq_pad, false, (void**)&rows);
  if (st == OM_OK) {
    const bool tensor = sizeof(T) == 2 && rule16_bwd_takes(call, g, gs, q, qs, k, ks, v, vs, dq, dq16, dqs, dk, dk16, dks, dv, dv16, dvs);
    const bool apart = sizeof(T) == 4 && rule16_planes_take(call, true) && rule16_result_fits(dq, dqs) && rule16_result_fits(dk, dks) && rule16_result_fits(dv, dvs);
    const float unit = tensor || apart ? 1.4426950408889634f : 1.f;
    if (out32) launch_rows(ctx, g, gs, out32, os, lse, b, h, lq, d, unit, rows);
    else launch_rows(ctx, g, gs, out, os, lse, b, h, lq, d, unit, rows);
    if (tensor) {
      st = rule16_bwd(ctx, call, g, gs, q, qs, k, ks, v, vs, rows, dq, dq16, dqs, dk, dk16, dks, dv, dv16, dvs, nullptr);
      pool_free(ctx, rows);
      rule_end(ctx, &call);
      return st;
    }
    RaParams<T> p = {};
    p.r = call.r; p.b = b; p.h = h; p.hkv = hkv; p.d = d;
    p.q = q; p.k = k; p.v = v; p.g = g; p.qs = ra_strides(qs); p.ks = ra_strides(ks); p.vs = ra_strides(vs); p.gs = ra_strides(gs);
    p.vec = d % 4 == 0 && ra_quads(q, qs, sizeof(T)) && ra_quads(k, ks, sizeof(T)) && ra_quads(v, vs, sizeof(T)) && ra_quads(g, gs, sizeof(T));
    p.rows = rows;
    p.dq = dq; p.dk = dk; p.dv = dv; p.dq16 = dq16; p.dk16 = dk16; p.dv16 = dv16;
    if (dq || dq16) p.dqs = ra_strides(dqs);
    if (dk || dk16) p.dks = ra_strides(dks);
    if (dv || dv16) p.dvs = ra_strides(dvs);
    p.unit = apart ? 0.6931471805599453f : 1.f;
    RulePlanes planes = {};
    if (apart) {
      st = rule16_planes(ctx, call, (const float*)q, qs, (const float*)k, ks, (const float*)v, vs, (const float*)g, gs, &planes);
      if (st == OM_OK)
        st = rule16_bwd(ctx, call, planes.p[3], &planes.q, planes.p[0], &planes.q, planes.p[1], &planes.k, planes.p[2], &planes.k, rows, dq, nullptr, dqs, dk, nullptr, dks, dv,
                        nullptr, dvs, &planes);
      p.plain = planes.plain;
    }
    if (st == OM_OK) st = ra_bwd_by_width<T>(ctx, p);
    rule16_planes_end(ctx, &planes);
    pool_free(ctx, rows);
  }
  rule_end(ctx, &call);
  return st;
}

}  // namespace om

using namespace om;

extern "C" {

int32_t om_rule_attention_fwd(om_ctx* ctx, const om_attention_rule* rule, const float* q, const om_head_strides* qs, const float* k,
                              const om_head_strides* ks, const float* v, const om_head_strides* vs, int32_t b, int32_t h, int32_t hkv, int32_t lq,
                              int32_t lk, int32_t d, float scale, float* out, const om_head_strides* os, float* lse) {
  OM_CHECK_CTX(ctx);
  return rule_fwd<float>(ctx, "om_rule_attention_fwd", rule, q, qs, k, ks, v, vs, b, h, hkv, lq, lk, d, scale, out, nullptr, os, lse);
}

int32_t om_rule_attention_bwd(om_ctx* ctx, const om_attention_rule* rule, const float* g, const om_head_strides* gs, const float* q,
                              const om_head_strides* qs, const float* k, const om_head_strides* ks, const float* v, const om_head_strides* vs,
                              const float* out, const om_head_strides* os, const float* lse, int32_t b, int32_t h, int32_t hkv, int32_t lq, int32_t lk,
                              int32_t d, float scale, float* dq, const om_head_strides* dqs, float* dk, const om_head_strides* dks, float* dv,
                              const om_head_strides* dvs) {
  OM_CHECK_CTX(ctx);
  return rule_bwd<float>(ctx, "om_rule_attention_bwd", rule, g, gs, q, qs, k, ks, v, vs, out, nullptr, os, lse, b, h, hkv, lq, lk, d, scale, dq, nullptr, dqs, dk,
                         nullptr, dks, dv, nullptr, dvs);
}

int32_t om_rule_attention_fwd_bf16(om_ctx* ctx, const om_attention_rule* rule, const uint16_t* q16, const om_head_strides* qs, const uint16_t* k16,
                                   const om_head_strides* ks, const uint16_t* v16, const om_head_strides* vs, int32_t b, int32_t h, int32_t hkv,
                                   int32_t lq, int32_t lk, int32_t d, float scale, float* out, uint16_t* out16, const om_head_strides* os, float* lse) {
  OM_CHECK_CTX(ctx);
  typedef __nv_bfloat16 T;
  return rule_fwd<T>(ctx, "om_rule_attention_fwd_bf16", rule, reinterpret_cast<const T*>(q16), qs, reinterpret_cast<const T*>(k16), ks,
                     reinterpret_cast<const T*>(v16), vs, b, h, hkv, lq, lk, d, scale, out, reinterpret_cast<T*>(out16), os, lse);
}

int32_t om_rule_attention_bwd_bf16(om_ctx* ctx, const om_attention_rule* rule, const uint16_t* g16, const om_head_strides* gs, const uint16_t* q16,
                                   const om_head_strides* qs, const uint16_t* k16, const om_head_strides* ks, const uint16_t* v16,
                                   const om_head_strides* vs, const uint16_t* out16, const om_head_strides* os, const float* lse, int32_t b, int32_t h,
                                   int32_t hkv, int32_t lq, int32_t lk, int32_t d, float scale, float* dq, uint16_t* dq16, const om_head_strides* dqs,
                                   float* dk, uint16_t* dk16, const om_head_strides* dks, float* dv, uint16_t* dv16, const om_head_strides* dvs) {
  OM_CHECK_CTX(ctx);
  typedef __nv_bfloat16 T;
  return rule_bwd<T>(ctx, "om_rule_attention_bwd_bf16", rule, reinterpret_cast<const T*>(g16), gs, reinterpret_cast<const T*>(q16), qs,
                     reinterpret_cast<const T*>(k16), ks, reinterpret_cast<const T*>(v16), vs, reinterpret_cast<const T*>(out16), nullptr, os, lse, b, h, hkv,
                     lq, lk, d, scale, dq, reinterpret_cast<T*>(dq16), dqs, dk, reinterpret_cast<T*>(dk16), dks, dv, reinterpret_cast<T*>(dv16), dvs);
}

int32_t om_rule_attention_bwd_bf16_out32(om_ctx* ctx, const om_attention_rule* rule, const uint16_t* g16, const om_head_strides* gs, const uint16_t* q16,
                                         const om_head_strides* qs, const uint16_t* k16, const om_head_strides* ks, const uint16_t* v16,
                                         const om_head_strides* vs, const float* out, const om_head_strides* os, const float* lse, int32_t b, int32_t h,
                                         int32_t hkv, int32_t lq, int32_t lk, int32_t d, float scale, float* dq, uint16_t* dq16, const om_head_strides* dqs,
                                         float* dk, uint16_t* dk16, const om_head_strides* dks, float* dv, uint16_t* dv16, const om_head_strides* dvs) {
  OM_CHECK_CTX(ctx);
  typedef __nv_bfloat16 T;
  return rule_bwd<T>(ctx, "om_rule_attention_bwd_bf16_out32", rule, reinterpret_cast<const T*>(g16), gs, reinterpret_cast<const T*>(q16), qs,
                     reinterpret_cast<const T*>(k16), ks, reinterpret_cast<const T*>(v16), vs, nullptr, out, os, lse, b, h, hkv, lq, lk, d, scale, dq,
                     reinterpret_cast<T*>(dq16), dqs, dk, reinterpret_cast<T*>(dk16), dks, dv, reinterpret_cast<T*>(dv16), dvs);
}

}  // extern "C"
