// Rotary positions: the leading columns of every head turned pair by pair, y = magnitude R(position * f_j) x.
//
// A pass reads and writes each element once (its floor) and computes the sine and cosine of an angle once for a token's pair and
// all the heads of a thread's slice. Angles are formed and reduced to an eighth of a turn in double: at position 10^5 an fp32
// product is off by 4e-3 radians, and double costs a few instructions per (token, pair) only, none per head.
#include <cuda_bf16.h>
#include <math.h>

#include "om_common.cuh"

namespace om {

constexpr int ROT_PAIRS = 128;

struct RotaryParams {
  double inv_freq[ROT_PAIRS];
  const int32_t* positions;
  long long positions_batch;
  int first_position;
  int heads, pairs, d, tail_chunks, slices;
  long long tokens;            // b * l
  int l;
  float magnitude;
  int inverse;
  long long xb, xh, xr, yb, yh, yr;
};

template <typename T>
__device__ __forceinline__ float rot_value(T v);
template <>
__device__ __forceinline__ float rot_value(float v) { return v; }
template <>
__device__ __forceinline__ float rot_value(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T rot_round(float v);
template <>
__device__ __forceinline__ float rot_round(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 rot_round(float v) { return __float2bfloat16_rn(v); }

// N elements moved at once: one 16-byte access, or one element where the layout allows no more.
template <typename T, int N>
struct alignas(sizeof(T) * N) RotVec {
  T v[N];
};

// Cosine and sine of position * inv_freq: t = q pi/2 + r with |r| <= pi/4 in double (pi/2 as two doubles, so r keeps the double
// product's own error only), then the Taylor series of both in fp32, whose first dropped terms are below 2e-9 there.
__device__ __forceinline__ void rot_angle(double position, double inv_freq, float magnitude, int inverse, float* c, float* s) {
  const double t = position * inv_freq;
  const double q = rint(t * 0.63661977236758134308);
  const float r = (float)__fma_rn(-q, 6.12323399573676603587e-17, __fma_rn(-q, 1.57079632679489655800, t));
  const float r2 = r * r;
  const float sn = fmaf(r * r2, fmaf(r2, fmaf(r2, fmaf(r2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), r);
  const float cs = fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const int quadrant = (int)((long long)q & 3);
  const float cr = (quadrant & 1) ? sn : cs, sr = (quadrant & 1) ? cs : sn;
  *c = (((quadrant + 1) & 2) ? -cr : cr) * magnitude;
  const float ss = ((quadrant & 2) ? -sr : sr) * magnitude;
  *s = inverse ? -ss : ss;
}

// A thread owns a group of P pairs of one token (or one vector of the columns behind them) and walks a slice of the heads.
// Half layout: P = the elements of one vector, taken at column j and at column j + pairs. Adjacent layout: P pairs are one vector.
template <typename T, int N, bool ADJACENT>
__global__ void __launch_bounds__(256)
rotary_kernel(const T* x, T* y, const __grid_constant__ RotaryParams p) {
  pdl_enter();
  constexpr int P = ADJACENT ? (N > 1 ? N / 2 : 1) : N;
  const int turn_chunks = p.pairs / P;               // the host picks N so that P divides the pairs
  const int chunks = turn_chunks + p.tail_chunks;
  const long long items = p.tokens * chunks;
  const long long total = items * p.slices;
  for (long long w = (long long)blockIdx.x * blockDim.x + threadIdx.x; w < total; w += (long long)gridDim.x * blockDim.x) {
    const int slice = (int)(w / items);
    const long long it = w - (long long)slice * items;
    const long long token = it / chunks;
    const int c = (int)(it - token * chunks);
    const long long bi = token / p.l;
    const int li = (int)(token - bi * p.l);
    const int h0 = (int)((long long)p.heads * slice / p.slices), h1 = (int)((long long)p.heads * (slice + 1) / p.slices);
    const T* xp = x + bi * p.xb + (long long)li * p.xr;
    T* yp = y + bi * p.yb + (long long)li * p.yr;
    if (c >= turn_chunks) {                           // columns that are not turned
      const int col = 2 * p.pairs + (c - turn_chunks) * N;
      for (int h = h0; h < h1; h++)
        *reinterpret_cast<RotVec<T, N>*>(yp + h * p.yh + col) = *reinterpret_cast<const RotVec<T, N>*>(xp + h * p.xh + col);
      continue;
    }
    const double position = (double)p.first_position + (double)(p.positions ? ld_global(p.positions + bi * p.positions_batch + li) : li);
    float cs[P], sn[P];
#pragma unroll
    for (int u = 0; u < P; u++) rot_angle(position, p.inv_freq[c * P + u], p.magnitude, p.inverse, &cs[u], &sn[u]);
    if (ADJACENT) {
      if (N == 1) {                                   // elements one by one: a pair is two of them
        for (int h = h0; h < h1; h++) {
          const long long xo = h * p.xh + 2 * c, yo = h * p.yh + 2 * c;
          const float a = rot_value(xp[xo]), b = rot_value(xp[xo + 1]);
          yp[yo] = rot_round<T>(fmaf(a, cs[0], -(b * sn[0])));
          yp[yo + 1] = rot_round<T>(fmaf(a, sn[0], b * cs[0]));
        }
      } else {
#pragma unroll 4
        for (int h = h0; h < h1; h++) {
          RotVec<T, N> in = *reinterpret_cast<const RotVec<T, N>*>(xp + h * p.xh + c * N), out;
#pragma unroll
          for (int u = 0; u < P; u++) {
            const float a = rot_value(in.v[(2 * u) % N]), b = rot_value(in.v[(2 * u + 1) % N]);
            out.v[(2 * u) % N] = rot_round<T>(fmaf(a, cs[u], -(b * sn[u])));
            out.v[(2 * u + 1) % N] = rot_round<T>(fmaf(a, sn[u], b * cs[u]));
          }
          *reinterpret_cast<RotVec<T, N>*>(yp + h * p.yh + c * N) = out;
        }
      }
    } else {
#pragma unroll 4
      for (int h = h0; h < h1; h++) {
        const RotVec<T, N> lo = *reinterpret_cast<const RotVec<T, N>*>(xp + h * p.xh + c * N);
        const RotVec<T, N> hi = *reinterpret_cast<const RotVec<T, N>*>(xp + h * p.xh + p.pairs + c * N);
        RotVec<T, N> olo, ohi;
#pragma unroll
        for (int u = 0; u < N; u++) {
          const float a = rot_value(lo.v[u]), b = rot_value(hi.v[u]);
          olo.v[u] = rot_round<T>(fmaf(a, cs[u], -(b * sn[u])));
          ohi.v[u] = rot_round<T>(fmaf(a, sn[u], b * cs[u]));
        }
        *reinterpret_cast<RotVec<T, N>*>(yp + h * p.yh + c * N) = olo;
        *reinterpret_cast<RotVec<T, N>*>(yp + h * p.yh + p.pairs + c * N) = ohi;
      }
    }
  }
}

template <typename T, int N, bool ADJACENT>
static void launch_rotary(om_ctx* ctx, const T* x, T* y, RotaryParams& p, bool copy_tail) {
  constexpr int P = ADJACENT ? (N > 1 ? N / 2 : 1) : N;
  p.tail_chunks = copy_tail ? (p.d - 2 * p.pairs) / N : 0;
  const long long items = p.tokens * (p.pairs / P + p.tail_chunks);
  // One slice of the heads per thread while that fills the device; few tokens are spread over the heads as well.
  const long long fill = (long long)ctx->sm_count * 2048;
  p.slices = (int)std::min<long long>(p.heads, std::max<long long>(1, fill / std::max<long long>(1, items)));
  const int grid = (int)std::min<long long>(ceil_div(items * p.slices, 256), (long long)ctx->sm_count * 64);
  launch_chained(ctx, rotary_kernel<T, N, ADJACENT>, grid, 256, 0, x, y, p);
}

template <typename T>
static int32_t rotary(om_ctx* ctx, const char* who, const T* x, const om_head_strides* xs, const int32_t* positions, int64_t positions_batch_stride,
                      int32_t first_position, int32_t b, int32_t h, int32_t l, int32_t d, const double* inv_freq, int32_t pairs, int32_t adjacent,
                      float magnitude, int32_t inverse, T* y, const om_head_strides* ys) {
  if (b < 0 || h < 0 || l < 0 || d < 0) return fail(ctx, OM_ERR_SHAPE, "%s: b %d h %d l %d d %d", who, b, h, l, d);
  if (pairs < 1 || pairs > ROT_PAIRS || 2 * pairs > d)
    return fail(ctx, OM_ERR_SHAPE, "%s: %d pairs of columns do not fit heads of %d columns (at most %d pairs)", who, pairs, d, ROT_PAIRS);
  if (!xs || !ys || xs->row < d || ys->row < d || xs->batch < 0 || xs->head < 0 || (b > 1 && ys->batch < 0) || (h > 1 && ys->head < 0))
    return fail(ctx, OM_ERR_SHAPE, "%s: rows of an activation must be at least d = %d elements apart and strides non-negative", who, d);
  if (!inv_freq) return fail(ctx, OM_ERR_ARG, "%s: the frequencies are required", who);
  if (!isfinite(magnitude)) return fail(ctx, OM_ERR_ARG, "%s: the magnitude must be finite", who);
  if (positions && positions_batch_stride < 0) return fail(ctx, OM_ERR_SHAPE, "%s: a negative stride of the positions", who);
  for (int j = 0; j < pairs; j++)
    if (!(fabs(inv_freq[j]) <= 1e6)) return fail(ctx, OM_ERR_ARG, "%s: frequency %d is not a number of at most 1e6 radians a position", who, j);
  if ((long long)b * h * l == 0) return OM_OK;
  if (!x || !y) return fail(ctx, OM_ERR_ARG, "%s: a tensor is missing", who);
  const bool in_place = x == y;
  if (in_place && ((b > 1 && xs->batch != ys->batch) || (h > 1 && xs->head != ys->head) || (l > 1 && xs->row != ys->row)))
    return fail(ctx, OM_ERR_SHAPE, "%s: in place needs the same strides on both sides", who);
  if (heads_overlap(*ys, b, h, l, d)) return fail(ctx, OM_ERR_SHAPE, "%s: rows of the result overlap", who);
  ProfileScope prof(ctx, "om_rotary", 3.0 * b * h * (double)l * 2 * pairs, 2.0 * sizeof(T) * b * h * (double)l * d);
  RotaryParams p;
  for (int j = 0; j < pairs; j++) p.inv_freq[j] = inv_freq[j];
  for (int j = pairs; j < ROT_PAIRS; j++) p.inv_freq[j] = 0;
  p.positions = positions; p.positions_batch = positions_batch_stride; p.first_position = first_position;
  p.heads = h; p.pairs = pairs; p.d = d; p.tokens = (long long)b * l; p.l = l; p.magnitude = magnitude; p.inverse = inverse;
  p.xb = xs->batch; p.xh = xs->head; p.xr = xs->row; p.yb = ys->batch; p.yh = ys->head; p.yr = ys->row;
  const bool tail = !in_place && d > 2 * pairs;
  // 16-byte vectors where every start that a thread computes lies on that grid: bases, strides, the pair groups and (in the
  // half layout) the second halves; else element by element (a 16-byte access is eight times fewer instructions for bfloat16).
  constexpr int N = 16 / sizeof(T);
  auto on_grid = [&](const void* q, const om_head_strides* s) {
    return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && s->row % N == 0 && (b == 1 || s->batch % N == 0) && (h == 1 || s->head % N == 0);
  };
  const bool grid = on_grid(x, xs) && on_grid(y, ys) && (!tail || (d % N == 0 && (2 * pairs) % N == 0));
  if (adjacent) {
    if (grid && pairs % (N / 2) == 0) launch_rotary<T, N, true>(ctx, x, y, p, tail);
    else launch_rotary<T, 1, true>(ctx, x, y, p, tail);
  } else {
    if (grid && pairs % N == 0) launch_rotary<T, N, false>(ctx, x, y, p, tail);
    else launch_rotary<T, 1, false>(ctx, x, y, p, tail);
  }
  OM_LAUNCH_CHECK(ctx, who);
  return OM_OK;
}

}  // namespace om

using namespace om;

extern "C" {

int32_t om_rotary_frequencies(om_ctx* ctx, const om_rotary_spec* spec, double* inv_freq_host) {
  auto bad = [&](int32_t code, const char* what) { return ctx ? fail(ctx, code, "om_rotary_frequencies: %s", what) : code; };
  if (!spec || !inv_freq_host) return bad(OM_ERR_ARG, "a specification and room for the frequencies are required");
  const int n = spec->columns;
  if (n < 2 || n > 2 * ROT_PAIRS || (n & 1)) return bad(OM_ERR_SHAPE, "the turned columns must be an even number from 2 to 256");
  if (!(spec->base > 1.0) || !std::isfinite(spec->base)) return bad(OM_ERR_ARG, "the base must be above 1 and finite");
  if (spec->scaling < OM_ROTARY_PLAIN || spec->scaling > OM_ROTARY_PARTS) return bad(OM_ERR_ARG, "unknown scaling");
  if (spec->scaling != OM_ROTARY_PLAIN && !(spec->factor >= 1.0 && std::isfinite(spec->factor))) return bad(OM_ERR_ARG, "the factor must be 1 or more and finite");
  if (spec->scaling == OM_ROTARY_BASE && n < 4) return bad(OM_ERR_SHAPE, "a raised base needs two pairs of columns at least");
  if (spec->scaling == OM_ROTARY_PARTS && (!(spec->original_context > 0.0) || !std::isfinite(spec->original_context) || !(spec->low_turns >= 0.0) ||
                                           !(spec->high_turns > spec->low_turns) || !std::isfinite(spec->high_turns)))
    return bad(OM_ERR_ARG, "a positive original context and 0 <= low < high turns are required");
  const double base = spec->scaling == OM_ROTARY_BASE ? spec->base * pow(spec->factor, (double)n / (n - 2)) : spec->base;
  if (!std::isfinite(base)) return bad(OM_ERR_ARG, "the raised base is not finite");
  for (int j = 0; j < n / 2; j++) {
    double f = pow(base, -2.0 * j / n);
    if (spec->scaling == OM_ROTARY_LINEAR) f /= spec->factor;
    if (spec->scaling == OM_ROTARY_PARTS) {
      const double turns = spec->original_context * f / (2.0 * 3.14159265358979323846);
      double kept = (turns - spec->low_turns) / (spec->high_turns - spec->low_turns);
      kept = kept < 0.0 ? 0.0 : kept > 1.0 ? 1.0 : kept;
      f *= (1.0 - kept) / spec->factor + kept;
    }
    inv_freq_host[j] = f;
  }
  return OM_OK;
}

int32_t om_rotary(om_ctx* ctx, const float* x, const om_head_strides* xs, const int32_t* positions, int64_t positions_batch_stride,
                  int32_t first_position, int32_t b, int32_t h, int32_t l, int32_t d, const double* inv_freq_host, int32_t pairs, int32_t adjacent,
                  float magnitude, int32_t inverse, float* y, const om_head_strides* ys) {
  OM_CHECK_CTX(ctx);
  return rotary<float>(ctx, "om_rotary", x, xs, positions, positions_batch_stride, first_position, b, h, l, d, inv_freq_host, pairs, adjacent, magnitude,
                       inverse, y, ys);
}

int32_t om_rotary_bf16(om_ctx* ctx, const uint16_t* x16, const om_head_strides* xs, const int32_t* positions, int64_t positions_batch_stride,
                       int32_t first_position, int32_t b, int32_t h, int32_t l, int32_t d, const double* inv_freq_host, int32_t pairs, int32_t adjacent,
                       float magnitude, int32_t inverse, uint16_t* y16, const om_head_strides* ys) {
  OM_CHECK_CTX(ctx);
  return rotary<__nv_bfloat16>(ctx, "om_rotary_bf16", reinterpret_cast<const __nv_bfloat16*>(x16), xs, positions, positions_batch_stride, first_position, b,
                               h, l, d, inv_freq_host, pairs, adjacent, magnitude, inverse, reinterpret_cast<__nv_bfloat16*>(y16), ys);
}

}  // extern "C"
