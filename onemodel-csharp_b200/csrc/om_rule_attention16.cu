// Attention by rule with bfloat16 operands on the tensor pipe (tcgen05), forward and backward, for head dimensions up to 128.
//
// Forward: a CTA holds 128 queries and walks the tiles of 128 keys that the rule lets them see. Two warps share 32 rows, a half of a step's
// keys each: the running maximum goes between them through shared memory, the sums meet at the end. S = Q K^T in fp32 in tensor memory
// -> weights exp2(S - m), rounded to bfloat16, in tensor memory -> O += P V with P read from there. Scores and weights have two places
// each, so the tensor pipe is a step ahead and the rows never wait for a product: at 128 columns a step takes 2260 cycles, of which the
// rows' exponentials 1250, maximum 350, waits 400; the pipe's two products 1500. (Two tiles of queries a CTA with one place each, rows
// through their scores twice: 8 x 32 single tokens 66 us instead of 61, three documents' batches forward 66 instead of 50, a window
// 207 instead of 226, 4 x 16 x 4096^2 344 instead of 372.) O stays in tensor memory; it is rescaled only when a row's maximum has grown
// by more than 2^8 over the one in use, which changes no result: numerator and denominator share the factor.
// With few rows the walk over the keys is split over CTAs that leave their sums, maxima and O for rule16_join_kernel, and the query
// heads that share a key head become rows of one tile, so that keys and values are read once.
//
// Backward: the weights come back from the forward's log-sum-exp, once in rule16_dkv_kernel (a CTA per 128 keys walks the queries of
// all heads that share them; rows are keys: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q) and once in rule16_dq_kernel (a
// CTA per 128 queries walks the keys: dQ += dS K). Seven products for five, but no partial sums through memory: a part of dQ per
// (query tile, key tile) is 128 KB of traffic against 0.3 us of tensor time for the two products that are done again.
// P and dS are rounded to bfloat16 as operands; the row dots come from the output as the caller has kept it, fp32 or bfloat16. Other
// roundings of the backward are the results' alone.
//
// fp32 operands of heads up to 64 columns run on the same kernels (PL = 2) with fp32 accuracy: every value as two half-precision numbers
// h + l, 22 significant bits, side by side in a row of 128 columns where two blocks of 64 lie otherwise, and a product as h h' + h l' +
// l h'. Weights and gradients of scores are taken apart the same way, those of each row and step over a unit of their own. A
// power of two per (batch, key head) brings each operand's largest value to 2^14 ... 2^15, so values down to 2^-14 of it keep all 22 bits;
// rule16_split_kernel, which makes the planes, sets a flag where a row's own largest is smaller than that (or the largest of all beyond
// 2^45, or not finite), and then these kernels do nothing and the fp32 ones behind them work.
//
// What a CTA sees of the other axis is worked out before its walk, a byte per 128 indices: worked out along the way it cost the rows as
// much as their exponentials. Every wait is bounded (om_tc.cuh). All sums are fp32 in an order that the shapes alone decide.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "om_rule.cuh"
#include "om_tc.cuh"

namespace om {

constexpr int R16_T = 128;                         // rows of every tile
constexpr int R16_CHUNK = R16_T * 128;             // bytes of a [128 x 64] bfloat16 block, 128-byte swizzled rows
constexpr int R16_ROW_WARPS = 8;
constexpr int R16_THREADS = 32 * (R16_ROW_WARPS + 2);   // warps 0-7: rows; warp 8: MMA issue; warp 9: TMA
constexpr int R16_PLAN = 1024;                     // tiles of the other axis that a CTA walks at most
constexpr float R16_LOG2E = 1.4426950408889634f, R16_LN2 = 0.6931471805599453f;

__device__ __forceinline__ void r16_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ float r16_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float r16_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t r16_pack(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The lower word of a shared-memory descriptor: (address >> 4) with the leading offset, one block of 64 columns for MN-major operands.
constexpr uint32_t R16_LBO_K = 1u << 16, R16_LBO_MN = ((uint32_t)R16_CHUNK >> 4) << 16;
__device__ __forceinline__ uint32_t r16_desc_k(const void* p) { return (smem_u32(p) >> 4) | R16_LBO_K; }
__device__ __forceinline__ uint32_t r16_desc_mn(const void* p) { return (smem_u32(p) >> 4) | R16_LBO_MN; }
// kind::f16 with bfloat16 (PL = 1) or half-precision operands and fp32 sums, M = 128.
__device__ __forceinline__ constexpr uint32_t r16_idesc(int pl, bool b_mn, int n) {
  return (1u << 4) | (pl == 1 ? (1u << 7) | (1u << 10) : 0u) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(R16_T >> 4) << 24);
}
// A from tensor memory: row r in lane r, elements 2 c and 2 c + 1 of the contraction in column c.
__device__ __forceinline__ void r16_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, {%6, %6, %6, %6}, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(UMMA_DESC_HI), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void r16_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Bytes of a tile of 128 rows.
template <int DP, int PL>
constexpr int r16_tile_bytes() { return (PL == 2 ? 2 : DP / 64) * R16_CHUNK; }
// D[128 x 128] = A B^T over the head's columns, both operands K-major in shared memory.
template <int DP, int PL>
__device__ __forceinline__ void r16_scores(uint32_t d, uint32_t a_k, uint32_t b_k) {
  constexpr uint32_t idesc = r16_idesc(PL, false, R16_T), CH = R16_CHUNK >> 4;
  if (PL == 2) {
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
      const uint32_t o = (uint32_t)ks * 2;
      umma_f16_ss(d, a_k + o, b_k + CH + o, idesc, ks > 0 ? 1u : 0u);
      umma_f16_ss(d, a_k + CH + o, b_k + o, idesc, 1u);
    }
#pragma unroll
    for (int ks = 0; ks < 4; ks++) umma_f16_ss(d, a_k + (uint32_t)ks * 2, b_k + (uint32_t)ks * 2, idesc, 1u);
  } else {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ks++) {
      const uint32_t o = (uint32_t)(ks / 4) * CH + (uint32_t)(ks % 4) * 2;
      umma_f16_ss(d, a_k + o, b_k + o, idesc, ks > 0 ? 1u : 0u);
    }
  }
}
// D[128 x DP] (+)= A B over the 128 rows of B: A in tensor memory, B MN-major in shared memory. Where A lies over what it came from, a
// row thread packs the results of its COLS columns over the first half of them: elements COLS t ... of the contraction are at COLS t.
// Two planes fill the place of what they came from, 32 columns at a time: 16 of h, 16 of l.
template <int DP, int COLS, int PL>
__device__ __forceinline__ void r16_gather(uint32_t d, uint32_t a, uint32_t b_mn, uint32_t accumulate) {
  constexpr uint32_t idesc = r16_idesc(PL, true, DP);
  constexpr int STEPS = (PL == 2 ? 32 : COLS) / 16, STRIDE = PL == 2 ? 32 : COLS;
  if (PL == 2) {
    // The small products first: the tensor core cuts off what a sum cannot hold at every addition.
#pragma unroll
    for (int ks = 0; ks < R16_T / 16; ks++) {
      const uint32_t h = a + (uint32_t)((ks / STEPS) * STRIDE + (ks % STEPS) * 8), b = b_mn + (uint32_t)ks * 128u;
      r16_mma_ts(d, h, b + (R16_CHUNK >> 4), idesc, ks > 0 ? 1u : accumulate);
      r16_mma_ts(d, h + 16u, b, idesc, 1u);
    }
  }
#pragma unroll
  for (int ks = 0; ks < R16_T / 16; ks++) {
    const uint32_t h = a + (uint32_t)((ks / STEPS) * STRIDE + (ks % STEPS) * 8), b = b_mn + (uint32_t)ks * 128u;
    r16_mma_ts(d, h, b, idesc, PL == 2 || ks > 0 ? 1u : accumulate);
  }
}
// The last step, which is in o: o = whole keep + o unit.
__device__ __forceinline__ void r16_add_whole(uint32_t whole, uint32_t (&o)[32], bool only, float keep, float unit) {
  uint32_t w[32];
  if (!only) {
    tmem_ld_32x32b_x32(whole, w);
    tmem_ld_wait();
  }
#pragma unroll
  for (int u = 0; u < 32; u++) {
    const float mine = __uint_as_float(o[u]) * unit;
    o[u] = __float_as_uint(only ? mine : fmaf(__uint_as_float(w[u]), keep, mine));
  }
}
// Two planes: the tensor core's own sums over a walk of thousands would lose digits (8 additions that are cut off, a tile, 2e-7; 192
// of them 5e-6), so each step's product is a sum of its own, which the rows add to the whole in fp32: whole = whole keep + step unit,
// COLS columns of both in tensor memory.
template <int COLS>
__device__ __forceinline__ void r16_fold(uint32_t whole, uint32_t step, bool first, float keep, float unit) {
#pragma unroll 1
  for (int c = 0; c < COLS; c += 16) {
    uint32_t a[16], b[16];
    tmem_ld_32x32b_x16(step + (uint32_t)c, a);
    if (!first) tmem_ld_32x32b_x16(whole + (uint32_t)c, b);
    tmem_ld_wait();
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const float mine = __uint_as_float(a[u]) * unit;
      a[u] = __float_as_uint(first ? mine : fmaf(__uint_as_float(b[u]), keep, mine));
    }
    r16_st16(whole + (uint32_t)c, a);
  }
}
// 32 results into tensor memory as operands: packed bfloat16, or two planes of halves.
__device__ __forceinline__ uint32_t r16_pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void r16_take_apart(float a, float b, uint32_t* h, uint32_t* l) {
  const __half2 hh = __floats2half2_rn(a, b);
  const float2 back = __half22float2(hh);
  *h = *reinterpret_cast<const uint32_t*>(&hh);
  *l = r16_pack_half(a - back.x, b - back.y);
}
template <int DP, int PL>
__device__ __forceinline__ void r16_load_tile(uint8_t* dst, const CUtensorMap* map, int row0, int head, int batch, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < (PL == 2 ? 2 : DP / 64); c++) tma_load_4d(dst + c * R16_CHUNK, map, c * 64, row0, head, batch, bar);
}

__device__ __forceinline__ void r16_load_rows(float* dst, const float* src, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 1024, [%2];" ::"r"(smem_u32(dst)), "l"(src), "r"(smem_u32(bar)) : "memory");
}

// Which of the indices at, at + 1, ... of one row's other axis are seen: [0, prefix), [lo, hi), none beyond `end`.
struct R16Row {
  int prefix, lo, hi, end, doc;
};
__device__ __forceinline__ R16Row r16_query_row(const RuleArgs& r, int prefix, int b, int i) {
  R16Row w;
  const RuleSpan s = rule_keys(r, prefix, i, i + 1);
  w.prefix = s.prefix;
  w.lo = s.lo;
  w.hi = s.hi;
  w.end = r.lk;
  w.doc = r.q_docs && i < r.lq ? r.q_docs[(long long)b * r.lq + i] : -1;
  return w;
}
__device__ __forceinline__ R16Row r16_key_row(const RuleArgs& r, int prefix, int b, int j) {
  R16Row w;
  w.prefix = 0;
  rule_queries(r, prefix, j, j + 1, &w.lo, &w.hi);
  w.end = r.lq;
  w.doc = r.k_docs && j < r.lk ? r.k_docs[(long long)b * r.lk + j] : -1;
  return w;
}
// Bit u: index at + u of the 32 from `at` on is seen.
__device__ __forceinline__ uint32_t r16_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t r16_bits(const R16Row& w, int at, const int32_t* docs) {
  uint32_t v = ((r16_below(w.hi - at) & ~r16_below(w.lo - at)) | r16_below(w.prefix - at)) & r16_below(w.end - at);
  if (docs) {
    uint32_t same = 0;
#pragma unroll 8
    for (int u = 0; u < 32; u++)
      if (at + u < w.end) same |= (docs[at + u] == w.doc ? 1u : 0u) << u;
    v &= w.doc >= 0 ? same : 0u;
  }
  return v;
}
__device__ __forceinline__ void r16_hide(uint32_t (&x)[32], uint32_t bits) {
#pragma unroll
  for (int u = 0; u < 32; u++)
    if (!((bits >> u) & 1u)) x[u] = 0xff800000u;
}
// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t r16_two(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void r16_fma2(float& a, float& b, uint32_t x, uint32_t y, uint64_t m, uint64_t c) {
  asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%2, %3};\n\tfma.rn.f32x2 t, t, %4, %5;\n\tmov.b64 {%0, %1}, t;\n\t}" : "=f"(a), "=f"(b) : "r"(x), "r"(y), "l"(m), "l"(c));
}
__device__ __forceinline__ uint64_t r16_add2(uint64_t s, float a, float b) {
  uint64_t v;
  asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%2, %3};\n\tadd.rn.f32x2 %0, %1, t;\n\t}" : "=l"(v) : "l"(s), "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float r16_max3(float a, float b, float c) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}
// What is done to a product in front of the softmax: 0 scaled, 1 and lowered with the distance, 2 capped (and lowered). Scores are in powers
// of two: scale, cap and slope come times log2 e. `far`: the signed distance of the first index of a run, as a float (a conversion for
// every score would take the unit that the exponentials need).
struct R16Score {
  float scale, angle, cap, slope;                        // angle: of the tanh's argument, scale / cap
};
// unit: of the products (1, or the powers of two that the planes were divided by).
template <int MODE>
__device__ __forceinline__ R16Score r16_score_of(const RuleArgs& r, int head, float unit) {
  R16Score c;
  c.scale = r.scale * unit * R16_LOG2E;
  c.angle = fminf(r.scale * unit * r.inv_softcap, 1e38f);   // a finite number, so that 0 times it is 0
  c.cap = r.softcap * R16_LOG2E;
  c.slope = MODE > 0 && r.slopes ? r.slopes[head] * R16_LOG2E : 0.f;
  return c;
}
// tanh(x) = 1 - 2 / (exp(2 x) + 1) is off by 2^-22 at most, absolutely: 2^-20 of its value from |x| = 0.3 on. Below, the Taylor series of
// tanh(x) / x, whose first term left out is 2^-24 there: the score times it, so that a cap far above the scores leaves them as they are
// (with the first form alone, a cap of 1000 put errors of 1e-4 on every score, one of 10^8 made them meaningless). LOW: |x| is known to be.
constexpr float R16_LOW = 0.3f;
template <int MODE, bool LOW>
__device__ __forceinline__ float r16_score(const R16Score& c, float far, float dot, float* dcap) {
  float s = dot * c.scale;
  if (MODE == 2) {
    const float x = dot * c.angle, x2 = x * x;
    const float ratio = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    float t = x * ratio;
    s *= ratio;
    if (!LOW && !(fabsf(x) < R16_LOW)) {
      t = fmaf(-2.f, r16_rcp(r16_ex2(x * (2.f * R16_LOG2E)) + 1.f), 1.f);
      s = c.cap * t;
    }
    *dcap = fmaf(-t, t, 1.f);
  }
  return fmaf(-c.slope, fabsf(far), s);
}
// 32 scores of a row; use(u, score, derivative of the cap). step: of the signed distance from one to the next. Caps are mostly far above the
// scores, so a warp looks first whether all of its own are low: 10 operations for each then, in place of two on the unit that the
// exponentials need (three documents' batches both ways: 168 us with the first form alone, 187 with both for every score, 172 so).
template <int MODE, typename F>
__device__ __forceinline__ void r16_scores32(const R16Score& c, const uint32_t (&x)[32], float far, float step, F use) {
  float dcap = 1.f;
  if (MODE == 2) {
    float big = 0.f;
#pragma unroll
    for (int u = 0; u < 32; u += 2) big = r16_max3(big, fabsf(__uint_as_float(x[u])), fabsf(__uint_as_float(x[u + 1])));
    if (__all_sync(0xffffffffu, big * c.angle < R16_LOW)) {
#pragma unroll
      for (int u = 0; u < 32; u++) {
        const float s = r16_score<MODE, true>(c, far + step * (float)u, __uint_as_float(x[u]), &dcap);
        use(u, s, dcap);
      }
      return;
    }
  }
#pragma unroll
  for (int u = 0; u < 32; u++) {
    const float s = r16_score<MODE, false>(c, far + step * (float)u, __uint_as_float(x[u]), &dcap);
    use(u, s, dcap);
  }
}

// A row of N fp32 values to fp32 and bfloat16 results, both 16 bytes at a time; columns behind d stay unwritten (d is a multiple of 8).
template <int N>
__device__ __forceinline__ void r16_write(const uint32_t (&v)[N], float factor, float* out, __nv_bfloat16* out16, long long at, int col, int d) {
#pragma unroll
  for (int c = 0; c < N; c += 8) {
    if (col + c >= d) break;
    float f[8];
#pragma unroll
    for (int u = 0; u < 8; u++) f[u] = __uint_as_float(v[c + u]) * factor;
    if (out) {
      *reinterpret_cast<float4*>(out + at + c) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(out + at + c + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
    if (out16) *reinterpret_cast<uint4*>(out16 + at + c) = make_uint4(r16_pack(f[0], f[1]), r16_pack(f[2], f[3]), r16_pack(f[4], f[5]), r16_pack(f[6], f[7]));
  }
}

// Looks once before it starts to count the time (om_tc.cuh).
__device__ __forceinline__ bool r16_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* status, int where) {
  return mbar_try_wait(bar, parity) || mbar_wait(bar, parity, abort_flag, status, where);
}
// A wait of all 32 rows of a warp: they go on together or not at all (what follows is issued by the whole warp).
__device__ __forceinline__ bool r16_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* status, int where) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = r16_bar(bar, parity, abort_flag, status, where);   // one lane asks: 32 asking alike cost the issue slots of the others
  __syncwarp();                                          // what the lane waited for is seen by the others: a vote orders no memory
  return __all_sync(0xffffffffu, ok);
}
// One arrival for a warp whose rows are done with tensor memory and shared memory.
__device__ __forceinline__ void r16_arrive_warp(uint64_t* bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) r16_arrive(bar);
}
struct R16Strides {
  long long batch, head, row;
};
struct R16Fwd {
  RuleArgs r;
  int h, hkv, d;
  int packed;                     // rows of a tile are (head of the group, query): h / hkv * lq of them
  int splits;
  float* out;
  __nv_bfloat16* out16;
  R16Strides os;
  float* lse;
  float* part;                    // [splits][b * h * lq][d] and [splits][b * h * lq] (maximum, sum) where splits > 1
  float2* part_ml;
  long long rows;                 // b * h * lq
  const float* units;             // two planes: [4][b * hkv] powers of two that q, k, v, g were divided by, and the flag that they were not
  const int32_t* plain;
  int32_t* status;
};

// A CTA's plan: the tiles of 128 of the other axis that some row tile sees anything of, in order, with rule_see's answer for each row
// tile (two bits, from bit 10 on) and whether rows of it are padding (bit 12). Made by one warp; returns their number.
__device__ __forceinline__ int r16_tile_of(uint32_t step) { return (int)(step & (R16_PLAN - 1)); }
__device__ __forceinline__ int r16_sees_of(uint32_t step) { return (int)(step >> 10) & 3; }
__device__ __forceinline__ bool r16_padded(uint32_t step) { return (step >> 12) & 1u; }
template <bool FULL>
__device__ __forceinline__ uint32_t r16_look(const RuleTile& t, int at) {
  const uint32_t sees = (uint32_t)rule_see<FULL>(t, at, 2);
  return sees == 1 && rule_padding(t, at, 2) ? 5u : sees;
}
// Padding of a bfloat16 tile that a product adds up over, to zeros: its weights are 0, but 0 times what is not a number is not one. A
// row warp has 16 rows of the tile, which no product reads at the time, and then tells the product that does through a barrier as ever.
template <int DP>
__device__ __forceinline__ void r16_clear(uint8_t* tile, const uint2* pads, int at64, int n64, int warp, int lane) {
  constexpr int PIECES = DP / 8;                         // of 16 bytes in a row
  const uint2 v = at64 + (warp >> 2) < n64 ? pads[at64 + (warp >> 2)] : make_uint2(0u, 0u);
  const uint32_t bits = ((warp & 2) ? v.y : v.x) >> (16 * (warp & 1));
#pragma unroll
  for (int e = lane; e < 16 * PIECES; e += 32) {
    const int row = e / PIECES, c = e % PIECES;
    if ((bits >> row) & 1u) *reinterpret_cast<uint4*>(tile + (c / 8) * R16_CHUNK + (16 * warp + row) * 128 + (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
template <typename F>
__device__ __forceinline__ int r16_plan(uint16_t* steps, int tiles, int lane, F see) {
  int n = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const int t = t0 + lane;
    const uint32_t a = t < tiles ? see(t) : 0u, some = __ballot_sync(0xffffffffu, a != 0);
    if (a) steps[n + __popc(some & ((1u << lane) - 1u))] = (uint16_t)((uint32_t)t | a << 10);
    n += __popc(some);
  }
  return n;
}

template <int DP, int PL>
struct R16FwdShape {
  static constexpr int TILE = r16_tile_bytes<DP, PL>();
  static constexpr int STAGES = TILE > R16_CHUNK ? 5 : 8; // of K and V tiles
  static constexpr int TURN = (1 + STAGES) * TILE;        // what the two warps of a row tell each other, [place][half][row]
  static constexpr int RULES = TURN + 4096;
  static constexpr int PLAN = RULES + 64;
  static constexpr int BARS = PLAN + R16_PLAN * 2 + 16;
  static constexpr int SMEM = BARS + 512;
};
// The two warps of a row. Both come here once a step whatever has happened to either, so neither waits for one that has left.
__device__ __forceinline__ void r16_meet(int barrier) { asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory"); }

template <int DP, int MODE, int PL>
__global__ void __launch_bounds__(R16_THREADS, 1)
rule16_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ R16Fwd p) {
  typedef R16FwdShape<DP, PL> W;
  // Scores in two places, O, and the weights in two places of their own; two planes of weights lie over the scores they came from, and
  // their O has a step's sum and the whole side by side.
  constexpr uint32_t COL_S = 0, COL_O = 256, COL_P = PL == 1 ? 384 : 0, P_STEP = PL == 1 ? 64 : 128;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *slot_q = smem, *ring = smem + W::TILE;
  uint16_t* steps = reinterpret_cast<uint16_t*>(smem + W::PLAN);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  uint64_t *bar_q = bars, *bar_s = bars + 1 /* [place] */, *bar_read = bars + 3 /* [place] */, *bar_p = bars + 5 /* [place] */, *bar_o = bars + 7 /* [place] */,
           *bar_full = bars + 9 /* [STAGES] */, *bar_empty = bar_full + W::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_empty + W::STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const RuleArgs& r = p.r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.h / p.hkv;
  const int split = blockIdx.z;
  int bi, hi, hk, i0;
  if (p.packed) {
    bi = blockIdx.x / p.hkv;
    hk = blockIdx.x - bi * p.hkv;
    hi = hk * group;
    i0 = 0;
  } else {
    bi = blockIdx.x / p.h;
    hi = blockIdx.x - bi * p.h;
    hk = hi / group;
    i0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * R16_T;      // the longest walks of a causal mask first
  }

  if (threadIdx.x == 0) {
    mbar_init(bar_q, 1);
    for (int a = 0; a < 2; a++) {
      mbar_init(&bar_s[a], 1);
      mbar_init(&bar_read[a], R16_ROW_WARPS);
      mbar_init(&bar_p[a], R16_ROW_WARPS);
      mbar_init(&bar_o[a], 1);
    }
    for (int a = 0; a < W::STAGES; a++) {
      mbar_init(&bar_full[a], 1);
      mbar_init(&bar_empty[a], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == R16_ROW_WARPS) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const int prefix = r.prefix ? r.prefix[bi] : 0;
  RuleTile* tile = reinterpret_cast<RuleTile*>(smem + W::RULES);
  if (threadIdx.x == 0) *tile = rule_query_tile(r, prefix, bi, i0, 2);
  const RuleSpan span = rule_keys(r, prefix, i0, min(p.packed ? r.lq : i0 + R16_T, r.lq));
  int first = span.prefix > 0 ? 0 : span.lo / R16_T, last = (max(span.prefix, span.hi) + R16_T - 1) / R16_T;
  const int per = max(0, last - first + p.splits - 1) / p.splits;
  first += split * per;
  last = min(first + per, last);
  __syncthreads();
  if (warp == 0) {
    const int n = r16_plan(steps, last - first, lane, [&](int t) { return r16_look<true>(*tile, (first + t) * R16_T); });
    if (lane == 0) steps[R16_PLAN] = (uint16_t)n;
  }
  __syncthreads();
  const int walk = (int)steps[R16_PLAN];

  bool ok = true;
  if (PL == 2 && ld_global(p.plain + bi * p.hkv + hk) != 0) {
    // values beyond what two halves hold: the fp32 kernel behind does these heads
  } else if (warp == R16_ROW_WARPS + 1) {
    if (lane == 0) {
      mbar_expect_tx(bar_q, p.packed ? (uint32_t)(W::TILE / R16_CHUNK) * (uint32_t)(group * r.lq) * 128u : (uint32_t)W::TILE);
      r16_load_tile<DP, PL>(slot_q, &map_q, i0, hi, bi, bar_q);
      int s = 0;
      uint32_t phase = 0;
      bool again = false;
      auto load = [&](const CUtensorMap* map, int n) {
        if (again) ok = ok && r16_bar(&bar_empty[s], phase ^ 1u, abort_flag, p.status, 61);
        if (!ok) return;
        mbar_expect_tx(&bar_full[s], W::TILE);
        r16_load_tile<DP, PL>(ring + s * W::TILE, map, (first + r16_tile_of(steps[n])) * R16_T, hk, bi, &bar_full[s]);
        if (++s == W::STAGES) {
          s = 0;
          phase ^= 1u;
          again = true;
        }
      };
      // In the order that the products take them.
      if (walk > 0) load(&map_k, 0);
      for (int n = 0; ok && n < walk; n++) {
        if (n + 1 < walk) load(&map_k, n + 1);
        load(&map_v, n);
      }
    }
  } else if (warp == R16_ROW_WARPS) {
    if (lane == 0) {
      ok = r16_bar(bar_q, 0, abort_flag, p.status, 62);
      int s = 0;                                          // the ring's next tile
      uint32_t phase = 0;
      auto take = [&]() {
        const int at = s;
        ok = ok && r16_bar(&bar_full[s], phase, abort_flag, p.status, 63);
        if (++s == W::STAGES) {
          s = 0;
          phase ^= 1u;
        }
        return at;
      };
      auto scores = [&](int n) {
        const int place = n & 1, ks = take();
        // The rows have the scores before last, or (two planes) the product that reads the weights over them is complete.
        if (n >= 2) ok = ok && r16_bar(PL == 1 ? &bar_read[place] : &bar_o[place], ((n - 2) >> 1) & 1u, abort_flag, p.status, 64);
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP, PL>(tmem + COL_S + 128u * place, r16_desc_k(slot_q), r16_desc_k(ring + ks * W::TILE));
        umma_commit(&bar_s[place]);
        umma_commit(&bar_empty[ks]);
      };
      if (ok && walk > 0) scores(0);
      for (int n = 0; ok && n < walk; n++) {
        const int place = n & 1;
        if (n + 1 < walk) scores(n + 1);
        const int vs = take();
        ok = ok && r16_bar(&bar_p[place], (n >> 1) & 1u, abort_flag, p.status, 65);
        if (!ok) break;
        tc_fence_after();
        r16_gather<DP, 128, PL>(tmem + COL_O, tmem + COL_P + P_STEP * place, r16_desc_mn(ring + vs * W::TILE), PL == 1 && n > 0 ? 1u : 0u);
        umma_commit(&bar_o[place]);
        umma_commit(&bar_empty[vs]);
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    const int half = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    int i = i0 + row, head = hi;
    bool valid = i < r.lq;
    if (p.packed) {
      const int gi = row / r.lq;
      valid = gi < group;
      i = valid ? row - gi * r.lq : 0;
      head = valid ? hi + gi : hi;
    }
    const int at_unit = bi * p.hkv + hk, n_units = (int)(p.rows / ((long long)p.h * r.lq)) * p.hkv;
    const float unit = PL == 2 ? p.units[at_unit] * p.units[n_units + at_unit] : 1.f, unit_v = PL == 2 ? p.units[2 * n_units + at_unit] : 1.f;
    const R16Score score = r16_score_of<MODE>(r, head, unit);
    const R16Row seen = r16_query_row(r, prefix, bi, min(i, r.lq - 1));
    const int32_t* docs = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16), t_o = lane_base + COL_O + (uint32_t)(DP / 2) * half;   // its half of O's columns
    float2* turn = reinterpret_cast<float2*>(smem + W::TURN);
    const int mine = half * 128 + row, other = (half ^ 1) * 128 + row;
    const float mult = MODE ? 1.f : r.scale * unit * R16_LOG2E;
    const uint64_t mult2 = r16_two(mult, mult);
    float m = -INFINITY, l = 0.f;                        // l: of its half
    float keep = 1.f, unit_o = 1.f;                      // two planes: what the whole and the step's product are added up with, a step later
    bool gone = false;                                   // both warps of a row know it
    for (int n = 0; n < walk; n++) {
      const uint32_t step = steps[n], place = n & 1u;
      const int sees = r16_sees_of(step), at = (first + r16_tile_of(step)) * R16_T + 64 * half;
      const uint32_t t_s = lane_base + COL_S + 128u * place + 64u * half, t_p = lane_base + COL_P + P_STEP * place + (PL == 1 ? 32u : 64u) * half;
      ok = ok && r16_wait(&bar_s[place], (n >> 1) & 1u, abort_flag, p.status, 66);
      tc_fence_after();
      uint32_t x[2][32];
      tmem_ld_32x32b_x32(t_s, x[0]);
      tmem_ld_32x32b_x32(t_s + 32u, x[1]);
      tmem_ld_wait();
      if (PL == 1) r16_arrive_warp(&bar_read[place], lane);
      float tops[2];
#pragma unroll
      for (int c = 0; c < 2; c++) {
        uint32_t(&v)[32] = x[c];
        if (MODE) {
          r16_scores32<MODE>(score, v, (float)(i + r.q_offset - at - 32 * c), -1.f, [&](int u, float s, float) { v[u] = __float_as_uint(s); });
        }
        if (sees == 1) r16_hide(v, r16_bits(seen, at + 32 * c, docs));
        float t[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          t[e] = fmaxf(__uint_as_float(v[8 * e]), __uint_as_float(v[8 * e + 1]));
#pragma unroll
          for (int u = 2; u < 8; u += 2) t[e] = r16_max3(t[e], __uint_as_float(v[8 * e + u]), __uint_as_float(v[8 * e + u + 1]));
        }
        tops[c] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      }
      // The other half's, by turns in two places: whoever writes one again has met the other warp since it was read. A wait that ran out is
      // told here.
      const float part_top = fmaxf(tops[0], tops[1]);
      turn[place * 256 + mine] = make_float2(part_top, ok ? 1.f : 0.f);
      r16_meet(1 + quad);
      const float2 theirs = turn[place * 256 + other];
      gone = !__all_sync(0xffffffffu, ok && theirs.y != 0.f);
      if (gone) break;
      const float top = fmaxf(part_top, theirs.x) * mult;
      const bool grown = top > (PL == 2 ? m : m + 8.f) || (m == -INFINITY && top > -INFINITY);
      const float shrink = grown ? r16_ex2(m - top) : 1.f;      // m = -inf: 0
      if (grown) m = top;
      // Two planes: weights over the step's own maximum, which goes to 2^15, so that small ones keep their digits however far the row's
      // maximum is above them: thousands of them can add up to something. Their sum and product come back over the row's maximum.
      const float step_unit = PL == 2 ? (top == -INFINITY ? 0.f : r16_ex2(top - m)) : 1.f;
      const float base = PL == 2 ? (top == -INFINITY ? 0.f : top) - 15.f : m == -INFINITY ? 0.f : m;
      const uint64_t base2 = r16_two(-base, -base);
      uint64_t sum[2] = {0ull, 0ull};
      // These scores came after the product before last, so its weights' place is free.
#pragma unroll
      for (int c = 0; c < 2; c++) {
        uint32_t w[16], wl[16];
#pragma unroll
        for (int u = 0; u < 16; u++) {
          float a, b;
          r16_fma2(a, b, x[c][2 * u], x[c][2 * u + 1], mult2, base2);
          a = r16_ex2(a);
          b = r16_ex2(b);
          sum[u & 1] = r16_add2(sum[u & 1], a, b);
          if (PL == 2) r16_take_apart(a, b, &w[u], &wl[u]);
          else w[u] = r16_pack(a, b);
        }
        r16_st16(t_p + (PL == 2 ? 32u : 16u) * c, w);
        if (PL == 2) r16_st16(t_p + 32u * c + 16u, wl);
      }
      const float2 s0 = *reinterpret_cast<const float2*>(&sum[0]), s1 = *reinterpret_cast<const float2*>(&sum[1]);
      l = l * shrink + ((s0.x + s0.y) + (s1.x + s1.y)) * step_unit;
      // O, before the product that adds these weights to it and after the one before: rescaled, or the step before added to the whole.
      if (n > 0 && (PL == 2 || __any_sync(0xffffffffu, grown))) {
        ok = r16_wait(&bar_o[place ^ 1u], ((n - 1) >> 1) & 1u, abort_flag, p.status, 69);
        tc_fence_after();
        if (PL == 2) {
          r16_fold<DP / 2>(t_o + 64u, t_o, n == 1, keep, unit_o);
        } else {
#pragma unroll 1
          for (int c = 0; c < DP / 2; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + (uint32_t)c, o);
            tmem_ld_wait();
#pragma unroll
            for (int u = 0; u < 32; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * shrink);
            tmem_st_32x32b_x32(t_o + (uint32_t)c, o);
          }
        }
      }
      if (PL == 2) {
        keep = shrink;
        unit_o = step_unit;
      }
      if (PL == 1 && r16_padded(step)) {
        const int stage = n + 1 < walk ? 2 * n + 2 : 2 * n + 1;   // of the values, in the order of the loads
        ok = ok && r16_wait(&bar_full[stage % W::STAGES], (stage / W::STAGES) & 1u, abort_flag, p.status, 68);
        if (ok) r16_clear<DP>(ring + stage % W::STAGES * W::TILE, r.k_pads + (long long)bi * r.nk64, (first + r16_tile_of(step)) * (R16_T / RULE_GRAIN), r.nk64, warp, lane);
      }
      tmem_st_wait();
      r16_arrive_warp(&bar_p[place], lane);
    }
    if (!gone) {
      // The row's sum is both halves'.
      if (walk > 0) ok = ok && r16_wait(&bar_o[(walk - 1) & 1], ((walk - 1) >> 1) & 1u, abort_flag, p.status, 67);
      turn[(walk & 1) * 256 + mine] = make_float2(l, 0.f);
      r16_meet(1 + quad);
      l += turn[(walk & 1) * 256 + other].x;
    }
    if (ok && !gone) {
      tc_fence_after();
      const long long at_row = ((long long)bi * p.h + head) * r.lq + i;
      float inv = l == 0.f ? 0.f : unit_v / l;
      float* out = p.out;
      __nv_bfloat16* out16 = p.out16;
      long long at = bi * p.os.batch + head * p.os.head + (long long)i * p.os.row;
      if (p.splits > 1) {
        inv = unit_v;
        out = p.part;
        out16 = nullptr;
        at = ((long long)split * p.rows + at_row) * p.d;
        if (valid && half == 0) p.part_ml[(long long)split * p.rows + at_row] = make_float2(PL == 2 ? m - 15.f : m, l);
      } else if (p.lse && valid && half == 0) {
        p.lse[at_row] = l == 0.f ? -INFINITY : ((PL == 2 ? m - 15.f : m) + log2f(l)) * R16_LN2;
      }
#pragma unroll 1
      for (int c = 0; c < DP / 2; c += 32) {
        uint32_t o[32];
        __syncwarp();
        if (walk > 0) {
          tmem_ld_32x32b_x32(t_o + (uint32_t)c, o);
          tmem_ld_wait();
        }
        if (PL == 2 && walk > 0) r16_add_whole(t_o + 64u + (uint32_t)c, o, walk == 1, keep, unit_o);
        if (walk == 0 || l == 0.f) {
#pragma unroll
          for (int u = 0; u < 32; u++) o[u] = 0u;
        }
        const int col = half * (DP / 2) + c;
        if (valid) r16_write(o, inv, out, out16, at + col, col, p.d);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == R16_ROW_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The parts of split walks: out = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s in increasing order of the splits. A warp per row.
__global__ void __launch_bounds__(256)
rule16_join_kernel(const __grid_constant__ R16Fwd p) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < p.rows; row += (long long)gridDim.x * 8) {
    const long long bh = row / p.r.lq;
    const int i = (int)(row - bh * p.r.lq), bi = (int)(bh / p.h), hi = (int)(bh - (long long)bi * p.h);
    if (p.plain && ld_global(p.plain + bi * p.hkv + hi / (p.h / p.hkv)) != 0) continue;
    float m = -INFINITY;
    for (int s = 0; s < p.splits; s++) {
      const float2 v = p.part_ml[s * p.rows + row];
      if (v.y != 0.f) m = fmaxf(m, v.x);
    }
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const int c = lane * 4;
    for (int s = 0; s < p.splits; s++) {
      const float2 v = p.part_ml[s * p.rows + row];
      if (v.y == 0.f) continue;                       // this part saw nothing
      const float f = r16_ex2(v.x - base);
      l = fmaf(v.y, f, l);
      if (c < p.d) {
        const float4 o = *reinterpret_cast<const float4*>(p.part + (s * p.rows + row) * p.d + c);
        acc = make_float4(fmaf(o.x, f, acc.x), fmaf(o.y, f, acc.y), fmaf(o.z, f, acc.z), fmaf(o.w, f, acc.w));
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (c < p.d) {
      const long long at = bi * p.os.batch + hi * p.os.head + (long long)i * p.os.row + c;
      acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (p.out) *reinterpret_cast<float4*>(p.out + at) = acc;
      if (p.out16) *reinterpret_cast<uint2*>(p.out16 + at) = make_uint2(r16_pack(acc.x, acc.y), r16_pack(acc.z, acc.w));
    }
    if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * R16_LN2;
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------

struct R16Bwd {
  RuleArgs r;
  int h, hkv, d;
  const float* rows;              // [b * h][tiles of 128 queries][2][128]: log-sum-exp in powers of two, row dots
  int tiles;
  float *d0, *d1;                 // dv and dk, or dq and nothing
  __nv_bfloat16 *d0_16, *d1_16;
  R16Strides s0, s1;
  const float* units;             // as in R16Fwd
  int units_n;                    // b * hkv
  const int32_t* plain;
  int32_t* status;
};

// Two stationary tiles, a ring of the tiles that two products read, the second one late (Q, or K), and a ring of the others (dO, or V).
// dQ's kernel has room for a third K at 128 columns; with two, the next scores waited for a load that waited for the product before.
template <int DP, int PL, bool KEYS>
struct R16BwdShape {
  static constexpr int TILE = r16_tile_bytes<DP, PL>();
  static constexpr int RING_A = TILE == R16_CHUNK ? 4 : KEYS ? 2 : 3, RING_B = TILE == R16_CHUNK ? 4 : 2;
  static constexpr int ROWS = (2 + RING_A + RING_B) * TILE;     // the queries' log-sum-exps and row dots, 1 KB a stage
  static constexpr int TURN = ROWS + (KEYS ? RING_A * 1024 : 0);   // two planes: what the two warps of a row tell each other, [place][half][row]
  static constexpr int RULES = TURN + (PL == 2 ? 512 : 0);
  static constexpr int PLAN = RULES + 64;
  static constexpr int BARS = PLAN + R16_PLAN * 2 + 16;
  static constexpr int SMEM = BARS + 256;
};

// Scores of one row (32 of them, a quarter of a tile) to weights: packed as bfloat16 in w where they are wanted, and in x, times the
// cap's derivative, for r16_gradients. Rows are keys (COLUMNS: the log-sum-exps go with the columns) or queries.
template <int MODE, bool COLUMNS, int PL>
__device__ __forceinline__ void r16_weights(const R16Score& score, uint32_t (&x)[32], uint32_t (&w)[16], uint32_t (&wl)[16], const float* lses, float lse, float lift, float far, float mult,
                                            bool partial, uint32_t bits) {
  float dcap[MODE == 2 ? 32 : 1];
  if (MODE)
    r16_scores32<MODE>(score, x, far, COLUMNS ? 1.f : -1.f, [&](int u, float s, float d) {
      x[u] = __float_as_uint(s);
      if (MODE == 2) dcap[u] = d;
    });
  if (partial) r16_hide(x, bits);
  const uint64_t mult2 = r16_two(mult, mult);
#pragma unroll
  for (int u = 0; u < 32; u += 4) {
    float e[4] = {lse, lse, lse, lse}, p[4];
    if (COLUMNS) {
      const float4 v = *reinterpret_cast<const float4*>(lses + u);
      e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
    }
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      r16_fma2(p[t], p[t + 1], x[u + t], x[u + t + 1], mult2, PL == 2 && COLUMNS ? r16_two(lift - e[t], lift - e[t + 1]) : r16_two(-e[t], -e[t + 1]));
      p[t] = r16_ex2(p[t]);
      p[t + 1] = r16_ex2(p[t + 1]);
      if (COLUMNS && PL == 2) r16_take_apart(p[t], p[t + 1], &w[(u + t) / 2], &wl[(u + t) / 2]);
      else if (COLUMNS) w[(u + t) / 2] = r16_pack(p[t], p[t + 1]);
    }
#pragma unroll
    for (int t = 0; t < 4; t++) x[u + t] = __float_as_uint(MODE == 2 ? p[t] == 0.f ? 0.f : p[t] * dcap[MODE == 2 ? u + t : 0] : p[t]);
  }
}
// The largest exponent of the 32 weights of a row whose columns have the log-sum-exps (of 32 scores, which are formed and read
// again for the weights).
template <int MODE>
__device__ __forceinline__ float r16_top(const R16Score& score, const uint32_t (&x)[32], const float* lses, float far, float mult, bool partial, uint32_t bits) {
  float top = -INFINITY;
  auto take = [&](int u, float s) { top = fmaxf(top, partial && !((bits >> u) & 1u) ? -INFINITY : s); };
  if (MODE) {
    r16_scores32<MODE>(score, x, far, 1.f, [&](int u, float s, float) { take(u, s - lses[u]); });
  } else {
#pragma unroll
    for (int u = 0; u < 32; u++) take(u, fmaf(__uint_as_float(x[u]), mult, -lses[u]));
  }
  return top;
}
// dS = weight (dP - dot), 32 of them, in v. partial: some are hidden, and 0 whatever dP is there. dP comes over `unit` (two planes).
template <bool COLUMNS, int PL>
__device__ __forceinline__ void r16_gradients(const uint32_t (&x)[32], const uint32_t (&dp)[32], float (&v)[32], const float* dots, float dot, float unit, bool partial) {
#pragma unroll
  for (int u = 0; u < 32; u += 4) {
    float d[4] = {dot, dot, dot, dot};
    if (COLUMNS) {
      const float4 f = *reinterpret_cast<const float4*>(dots + u);
      d[0] = f.x; d[1] = f.y; d[2] = f.z; d[3] = f.w;
    }
#pragma unroll
    for (int t = 0; t < 4; t++)
      v[u + t] = __uint_as_float(x[u + t]) * (PL == 2 ? fmaf(__uint_as_float(dp[u + t]), unit, -d[t]) : __uint_as_float(dp[u + t]) - d[t]);
  }
  if (partial) {
#pragma unroll
    for (int u = 0; u < 32; u++) v[u] = x[u] == 0u ? 0.f : v[u];
  }
}
template <bool COLUMNS>
__device__ __forceinline__ void r16_gradients16(const uint32_t (&x)[32], const uint32_t (&dp)[32], uint32_t (&w)[16], const float* dots, float dot, bool partial) {
  float v[32];
  r16_gradients<COLUMNS, 1>(x, dp, v, dots, dot, 1.f, partial);
#pragma unroll
  for (int u = 0; u < 32; u += 2) w[u / 2] = r16_pack(v[u], v[u + 1]);
}
// Two planes: a row's gradients of a step over a power of two of their own, which brings the largest of them to 2^14 ... 2^15, whatever
// it is: a unit for the whole head, from bounds of |dO| and |V|, left few digits to the rows far below the bound (a row of dO at 2^-13 of the
// largest: its dQ off by 2e-4). The row's two warps tell each other the exponent of the largest, in a byte; 255: a wait ran out.
struct R16Unit {
  float to, back;                                        // the power of two that the row is multiplied with, and the one that undoes it
};
__device__ __forceinline__ R16Unit r16_unit(uint32_t exponent) {
  const uint32_t e = max(exponent, 15u);
  return R16Unit{__uint_as_float((268u - e) << 23), __uint_as_float((e - 14u) << 23)};
}
__device__ __forceinline__ bool r16_share(uint8_t* turn, int half, int row, int quad, bool ok, uint32_t& exponent) {
  exponent = min(exponent, 254u);
  turn[128 * half + row] = (uint8_t)(ok ? exponent : 255u);
  r16_meet(1 + quad);
  const uint32_t theirs = turn[128 * (half ^ 1) + row];
  exponent = max(exponent, theirs);
  return __all_sync(0xffffffffu, ok && theirs != 255u);
}
template <bool COLUMNS>
__device__ __forceinline__ void r16_gradients2(uint32_t (&x)[32], const uint32_t (&dp)[32], const float* dots, float dot, float unit, bool partial, float& largest) {
  float v[32];
  r16_gradients<COLUMNS, 2>(x, dp, v, dots, dot, unit, partial);
#pragma unroll
  for (int u = 0; u < 32; u += 2) {
    largest = r16_max3(largest, fabsf(v[u]), fabsf(v[u + 1]));
    x[u] = __float_as_uint(v[u]);
    x[u + 1] = __float_as_uint(v[u + 1]);
  }
}
__device__ __forceinline__ void r16_apart(const uint32_t (&x)[32], float to, uint32_t (&h)[16], uint32_t (&l)[16]) {
#pragma unroll
  for (int u = 0; u < 32; u += 2) r16_take_apart(__uint_as_float(x[u]) * to, __uint_as_float(x[u + 1]) * to, &h[u / 2], &l[u / 2]);
}

template <int DP, int MODE, int PL>
__global__ void __launch_bounds__(R16_THREADS, 1)
rule16_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ CUtensorMap map_g, const __grid_constant__ R16Bwd p) {
  typedef R16BwdShape<DP, PL, true> W;
  constexpr uint32_t COL_S = 0 /* and P over it */, COL_DP = 128 /* and dS */, COL_DV = 256, COL_DK = 384;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *slot_k = smem, *slot_v = smem + W::TILE, *ring_q = smem + 2 * W::TILE, *ring_g = ring_q + W::RING_A * W::TILE;
  uint16_t* steps = reinterpret_cast<uint16_t*>(smem + W::PLAN);
  float* ring_rows = reinterpret_cast<float*>(smem + W::ROWS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  uint64_t *bar_kv = bars, *bar_done = bars + 1, *bar_s = bars + 2, *bar_dp = bars + 3, *bar_p = bars + 4, *bar_ds = bars + 5, *bar_dv = bars + 6, *bar_dk = bars + 7,
           *full_q = bars + 8, *empty_q = full_q + W::RING_A, *full_g = empty_q + W::RING_A, *empty_g = full_g + W::RING_B;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty_g + W::RING_B);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const RuleArgs& r = p.r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j0 = blockIdx.y * R16_T, bi = blockIdx.x / p.hkv, hk = blockIdx.x - bi * p.hkv, group = p.h / p.hkv;   // the longest walks of a causal mask first

  if (threadIdx.x == 0) {
    mbar_init(bar_kv, 1);
    mbar_init(bar_done, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_dp, 1);
    mbar_init(bar_p, R16_ROW_WARPS);
    mbar_init(bar_ds, R16_ROW_WARPS);
    mbar_init(bar_dv, 1);
    mbar_init(bar_dk, 1);
    static_assert(W::RING_A == W::RING_B, "one stage number serves both rings");
    for (int a = 0; a < W::RING_A; a++) {
      mbar_init(&full_q[a], 1);
      mbar_init(&empty_q[a], 1);
      mbar_init(&full_g[a], 1);
      mbar_init(&empty_g[a], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == R16_ROW_WARPS) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const int prefix = r.prefix ? r.prefix[bi] : 0;
  RuleTile* tile = reinterpret_cast<RuleTile*>(smem + W::RULES);
  if (threadIdx.x == 0) *tile = rule_key_tile(r, prefix, bi, j0, 2);
  __syncthreads();
  const int first = tile->lo / R16_T, tiles = max(0, (min(tile->hi, r.lq) + R16_T - 1) / R16_T - first);
  if (warp == 0) {
    const int n = r16_plan(steps, tiles, lane, [&](int t) { return r16_look<false>(*tile, (first + t) * R16_T); });
    if (lane == 0) steps[R16_PLAN] = (uint16_t)n;
  }
  __syncthreads();
  // The same steps for every head that shares the keys, head by head.
  const int round = (int)steps[R16_PLAN], walk = round * group;
  int gi = 0, k = -1;                                    // the head, and its step
  auto forth = [&]() {
    if (++k == round) {
      k = 0;
      gi++;
    }
    return (uint32_t)steps[k];
  };

  bool ok = true;
  if (PL == 2 && ld_global(p.plain + bi * p.hkv + hk) != 0) {
    // values beyond what two halves hold: the fp32 kernel behind does these heads
  } else if (warp == R16_ROW_WARPS + 1) {
    if (lane == 0) {
      mbar_expect_tx(bar_kv, 2 * W::TILE);
      r16_load_tile<DP, PL>(slot_k, &map_k, j0, hk, bi, bar_kv);
      r16_load_tile<DP, PL>(slot_v, &map_v, j0, hk, bi, bar_kv);
      for (int n = 0; ok && n < walk; n++) {
        const uint32_t step = forth();
        const int a = n % W::RING_A, head = hk * group + gi, at = first + r16_tile_of(step);
        const uint32_t before = ((n / W::RING_A) & 1u) ^ 1u;
        // The keys' gradient of the tile before in this stage has read it, after the rows were done with its log-sum-exps and dots.
        if (n >= W::RING_A) ok = r16_bar(&empty_q[a], before, abort_flag, p.status, 71);
        if (!ok) break;
        mbar_expect_tx(&full_q[a], W::TILE + 1024);
        r16_load_tile<DP, PL>(ring_q + a * W::TILE, &map_q, at * R16_T, head, bi, &full_q[a]);
        r16_load_rows(ring_rows + a * 256, p.rows + (((long long)bi * p.h + head) * p.tiles + at) * 256, &full_q[a]);
        if (n >= W::RING_A) ok = r16_bar(&empty_g[a], before, abort_flag, p.status, 72);
        if (!ok) break;
        mbar_expect_tx(&full_g[a], W::TILE);
        r16_load_tile<DP, PL>(ring_g + a * W::TILE, &map_g, at * R16_T, head, bi, &full_g[a]);
      }
    }
  } else if (warp == R16_ROW_WARPS) {
    if (lane == 0) {
      ok = r16_bar(bar_kv, 0, abort_flag, p.status, 73);
      auto scores = [&](int n, uint64_t* full, uint64_t* bar, const uint8_t* keep, const uint8_t* ring, uint32_t col) {
        const int a = n % W::RING_A;
        ok = ok && r16_bar(&full[a], (n / W::RING_A) & 1u, abort_flag, p.status, 74);
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP, PL>(tmem + col, r16_desc_k(keep), r16_desc_k(ring + a * W::TILE));
        umma_commit(bar);
      };
      if (ok && walk > 0) {
        scores(0, full_q, bar_s, slot_k, ring_q, COL_S);
        scores(0, full_g, bar_dp, slot_v, ring_g, COL_DP);
      }
      for (int n = 0; ok && n < walk; n++) {
        const int a = n % W::RING_A;
        const uint32_t phase = n & 1u;
        const bool more = n + 1 < walk;
        // dV += P^T dO, then the next scores as soon as it has read P, which lies over these.
        if (!(ok = r16_bar(bar_p, phase, abort_flag, p.status, 76))) break;
        tc_fence_after();
        r16_gather<DP, 64, PL>(tmem + COL_DV, tmem + COL_S, r16_desc_mn(ring_g + a * W::TILE), PL == 1 && n > 0 ? 1u : 0u);
        umma_commit(bar_dv);
        umma_commit(&empty_g[a]);
        if (more) {
          ok = r16_bar(bar_dv, phase, abort_flag, p.status, 77);
          scores(n + 1, full_q, bar_s, slot_k, ring_q, COL_S);
        }
        // dK += dS^T Q, then the next dP.
        if (!(ok = ok && r16_bar(bar_ds, phase, abort_flag, p.status, 78))) break;
        tc_fence_after();
        r16_gather<DP, 64, PL>(tmem + COL_DK, tmem + COL_DP, r16_desc_mn(ring_q + a * W::TILE), PL == 1 && n > 0 ? 1u : 0u);
        umma_commit(bar_dk);
        umma_commit(&empty_q[a]);
        if (more) {
          ok = r16_bar(bar_dk, phase, abort_flag, p.status, 79);
          scores(n + 1, full_g, bar_dp, slot_v, ring_g, COL_DP);
        }
      }
      if (ok) umma_commit(bar_done);
      else *abort_flag = 1;
    }
  } else {
    const int half = warp >> 2, quad = warp & 3, row = quad * 32 + lane, j = j0 + row;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_s = lane_base + COL_S + 64u * half, t_dp = lane_base + COL_DP + 64u * half;
    const R16Row seen = r16_key_row(r, prefix, bi, min(j, r.lk - 1));
    const int32_t* docs = r.q_docs ? r.q_docs + (long long)bi * r.lq : nullptr;
    // Units of the planes. The weights of a row and step are kept over a power of two, too: the largest is brought to 2^13 ... 2^14.
    const int at_unit = bi * p.hkv + hk, n_units = p.units_n;
    const float unit_q = PL == 2 ? p.units[at_unit] : 1.f, unit_k = PL == 2 ? p.units[n_units + at_unit] : 1.f, unit_v = PL == 2 ? p.units[2 * n_units + at_unit] : 1.f,
                unit_g = PL == 2 ? p.units[3 * n_units + at_unit] : 1.f, unit = unit_q * unit_k;
    uint8_t* turn = smem + W::TURN;
    float lift = 0.f, unit_dv = 1.f, unit_dk = 1.f;        // the units: of the step's products that are not yet added to the whole
    const float mult = MODE ? 1.f : r.scale * unit * R16_LOG2E;
    for (int n = 0; ok && n < walk; n++) {
      const uint32_t step = forth(), phase = n & 1u;
      const int a = n % W::RING_A, at = (first + r16_tile_of(step)) * R16_T + half * 64;
      const bool partial = r16_sees_of(step) == 1;
      const R16Score score = r16_score_of<MODE>(r, hk * group + gi, unit);
      const float* rows = ring_rows + a * 256 + half * 64;
      // The queries' log-sum-exps came with the queries, which the scores have waited for; this wait makes them seen here.
      ok = r16_wait(&full_q[a], (n / W::RING_A) & 1u, abort_flag, p.status, 94) && r16_wait(bar_s, phase, abort_flag, p.status, 80);
      if (PL == 1 && !ok) break;                           // two planes: both warps of a row leave together, below
      tc_fence_after();
      // The scores came after the product before, and the next one waits for these weights.
      if (PL == 2 && n > 0) r16_fold<32>(lane_base + COL_DV + 64u + 32u * half, lane_base + COL_DV + 32u * half, n == 1, 1.f, unit_dv);
      uint32_t x[2][32], w[16], wl[16];
      if (PL == 1) {
        tmem_ld_32x32b_x32(t_s, x[0]);
        tmem_ld_32x32b_x32(t_s + 32u, x[1]);
        tmem_ld_wait();
      }
      uint32_t bits[2] = {~0u, ~0u};
      if (partial) {
        bits[0] = r16_bits(seen, at, docs);
        bits[1] = r16_bits(seen, at + 32, docs);
      }
      if (PL == 2) {
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          tmem_ld_32x32b_x32(t_s + 32u * c, x[c]);
          tmem_ld_wait();
          top = fmaxf(top, r16_top<MODE>(score, x[c], rows + c * 32, (float)(at + c * 32 + r.q_offset - j), mult, partial, bits[c]));
        }
        uint32_t up = (uint32_t)(min(max((int)ceilf(top), -110), 110) + 140);
        if (!(ok = r16_share(turn, half, row, quad, ok, up))) break;
        lift = 154.f - (float)up;                          // weights times 2^lift
        unit_dv = __uint_as_float((up - 27u) << 23);
      }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        if (PL == 2) {                                     // again: 64 scores and what becomes of them do not fit the registers
          tmem_ld_32x32b_x32(t_s + 32u * c, x[c]);
          tmem_ld_wait();
        }
        r16_weights<MODE, true, PL>(score, x[c], w, wl, rows + c * 32, 0.f, lift, (float)(at + c * 32 + r.q_offset - j), mult, partial, bits[c]);
        r16_st16(t_s + (PL == 2 ? 32u : 16u) * c, w);
        if (PL == 2) r16_st16(t_s + 32u * c + 16u, wl);
      }
      if (PL == 1 && r16_padded(step)) {
        // Both tiles, once the product that forms dP from one of them is complete (the scores are).
        if (!(ok = r16_wait(bar_dp, phase, abort_flag, p.status, 96))) break;
        const uint2* pads = r.q_pads + (long long)bi * r.nq64;
        const int at64 = (first + r16_tile_of(step)) * (R16_T / RULE_GRAIN);
        r16_clear<DP>(ring_g + a * W::TILE, pads, at64, r.nq64, warp, lane);
        r16_clear<DP>(ring_q + a * W::TILE, pads, at64, r.nq64, warp, lane);
      }
      tmem_st_wait();
      r16_arrive_warp(bar_p, lane);
      ok = ok && r16_wait(bar_dp, phase, abort_flag, p.status, 81);
      if (PL == 1 && !ok) break;
      tc_fence_after();
      if (PL == 2) {
        if (n > 0) r16_fold<32>(lane_base + COL_DK + 64u + 32u * half, lane_base + COL_DK + 32u * half, n == 1, 1.f, unit_dk);
        float largest = 0.f;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t dp[32];
          tmem_ld_32x32b_x32(t_dp + 32u * c, dp);
          tmem_ld_wait();
          r16_gradients2<true>(x[c], dp, rows + 128 + 32 * c, 0.f, unit_g * unit_v, partial, largest);
        }
        uint32_t exponent = __float_as_uint(largest) >> 23;
        if (!(ok = r16_share(turn + 256, half, row, quad, ok, exponent))) break;
        const R16Unit step_unit = r16_unit(exponent);
        unit_dk = step_unit.back * unit_dv;                // the weights' factor is in them
#pragma unroll
        for (int c = 0; c < 2; c++) {
          r16_apart(x[c], step_unit.to, w, wl);
          r16_st16(t_dp + 32u * c, w);
          r16_st16(t_dp + 32u * c + 16u, wl);
        }
      } else {
        uint32_t dp[2][32];
        tmem_ld_32x32b_x32(t_dp, dp[0]);
        tmem_ld_wait();
        tmem_ld_32x32b_x32(t_dp + 32u, dp[1]);
        r16_gradients16<true>(x[0], dp[0], w, rows + 128, 0.f, partial);
        tmem_ld_wait();
        r16_st16(t_dp, w);
        r16_gradients16<true>(x[1], dp[1], w, rows + 160, 0.f, partial);
        r16_st16(t_dp + 16u, w);
      }
      tmem_st_wait();
      r16_arrive_warp(bar_ds, lane);
    }
    if (ok) ok = r16_wait(bar_done, 0, abort_flag, p.status, 82);
    if (ok) {
      tc_fence_after();
      // dV by the first four warps, dK by the others.
      float* out = half == 0 ? p.d0 : p.d1;
      __nv_bfloat16* out16 = half == 0 ? p.d0_16 : p.d1_16;
      const R16Strides& s = half == 0 ? p.s0 : p.s1;
      if (out || out16) {
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          __syncwarp();
          if (walk > 0) {
            tmem_ld_32x32b_x32(lane_base + (half == 0 ? COL_DV : COL_DK) + (uint32_t)c, o);
            tmem_ld_wait();
            if (PL == 2) r16_add_whole(lane_base + (half == 0 ? COL_DV : COL_DK) + 64u + (uint32_t)c, o, walk == 1, 1.f, half == 0 ? unit_dv : unit_dk);
          } else {
#pragma unroll
            for (int u = 0; u < 32; u++) o[u] = 0u;
          }
          if (j < r.lk) r16_write(o, half == 0 ? unit_g : r.scale * unit_q, out, out16, bi * s.batch + hk * s.head + (long long)j * s.row + c, c, p.d);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == R16_ROW_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, int MODE, int PL>
__global__ void __launch_bounds__(R16_THREADS, 1)
rule16_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_g, const __grid_constant__ R16Bwd p) {
  typedef R16BwdShape<DP, PL, false> W;
  constexpr uint32_t COL_S = 0 /* two places, and dS over either */, COL_DP = 256, COL_DQ = 384;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *slot_q = smem, *slot_g = smem + W::TILE, *ring_k = smem + 2 * W::TILE, *ring_v = ring_k + W::RING_A * W::TILE;
  uint16_t* steps = reinterpret_cast<uint16_t*>(smem + W::PLAN);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  uint64_t *bar_qg = bars, *bar_done = bars + 1, *bar_s = bars + 2 /* [place] */, *bar_ds = bars + 4 /* [place] */, *bar_dq = bars + 6 /* [place] */, *bar_dp = bars + 8,
           *read_dp = bars + 9, *full_k = bars + 10, *empty_k = full_k + W::RING_A, *full_v = empty_k + W::RING_A, *empty_v = full_v + W::RING_B;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty_v + W::RING_B);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const RuleArgs& r = p.r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * R16_T, bi = blockIdx.x / p.h, hi = blockIdx.x - bi * p.h, hk = hi / (p.h / p.hkv);

  if (threadIdx.x == 0) {
    mbar_init(bar_qg, 1);
    mbar_init(bar_done, 1);
    mbar_init(bar_dp, 1);
    mbar_init(read_dp, R16_ROW_WARPS);
    for (int a = 0; a < 2; a++) {
      mbar_init(&bar_s[a], 1);
      mbar_init(&bar_ds[a], R16_ROW_WARPS);
      mbar_init(&bar_dq[a], 1);
    }
    for (int a = 0; a < W::RING_A; a++) {
      mbar_init(&full_k[a], 1);
      mbar_init(&empty_k[a], 1);
    }
    for (int a = 0; a < W::RING_B; a++) {
      mbar_init(&full_v[a], 1);
      mbar_init(&empty_v[a], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == R16_ROW_WARPS) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const int prefix = r.prefix ? r.prefix[bi] : 0;
  RuleTile* tile = reinterpret_cast<RuleTile*>(smem + W::RULES);
  if (threadIdx.x == 0) *tile = rule_query_tile(r, prefix, bi, i0, 2);
  __syncthreads();
  const int first = tile->pre > 0 ? 0 : tile->lo / R16_T, tiles = max(0, (min(max(tile->pre, tile->hi), r.lk) + R16_T - 1) / R16_T - first);
  if (warp == 0) {
    const int n = r16_plan(steps, tiles, lane, [&](int t) { return r16_look<true>(*tile, (first + t) * R16_T); });
    if (lane == 0) steps[R16_PLAN] = (uint16_t)n;
  }
  __syncthreads();
  const int walk = (int)steps[R16_PLAN];

  bool ok = true;
  if (PL == 2 && ld_global(p.plain + bi * p.hkv + hk) != 0) {
    // values beyond what two halves hold: the fp32 kernel behind does these heads
  } else if (warp == R16_ROW_WARPS + 1) {
    if (lane == 0) {
      mbar_expect_tx(bar_qg, 2 * W::TILE);
      r16_load_tile<DP, PL>(slot_q, &map_q, i0, hi, bi, bar_qg);
      r16_load_tile<DP, PL>(slot_g, &map_g, i0, hi, bi, bar_qg);
      for (int n = 0; ok && n < walk; n++) {
        const int a = n % W::RING_A, b = n % W::RING_B, at = (first + r16_tile_of(steps[n])) * R16_T;
        if (n >= W::RING_A) ok = r16_bar(&empty_k[a], ((n / W::RING_A) & 1u) ^ 1u, abort_flag, p.status, 83);
        if (!ok) break;
        mbar_expect_tx(&full_k[a], W::TILE);
        r16_load_tile<DP, PL>(ring_k + a * W::TILE, &map_k, at, hk, bi, &full_k[a]);
        if (n >= W::RING_B) ok = r16_bar(&empty_v[b], ((n / W::RING_B) & 1u) ^ 1u, abort_flag, p.status, 84);
        if (!ok) break;
        mbar_expect_tx(&full_v[b], W::TILE);
        r16_load_tile<DP, PL>(ring_v + b * W::TILE, &map_v, at, hk, bi, &full_v[b]);
      }
    }
  } else if (warp == R16_ROW_WARPS) {
    if (lane == 0) {
      ok = r16_bar(bar_qg, 0, abort_flag, p.status, 85);
      auto scores = [&](int n) {
        const int a = n % W::RING_A, b = n % W::RING_B;
        const uint32_t place = n & 1u;
        // Over the gradients of the step before last, which their product has read.
        ok = r16_bar(&full_k[a], (n / W::RING_A) & 1u, abort_flag, p.status, 86) && (n < 2 || r16_bar(&bar_dq[place], ((n - 2) >> 1) & 1u, abort_flag, p.status, 87));
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP, PL>(tmem + COL_S + 128u * place, r16_desc_k(slot_q), r16_desc_k(ring_k + a * W::TILE));
        umma_commit(&bar_s[place]);
        // Once the rows have taken the dP before.
        ok = r16_bar(&full_v[b], (n / W::RING_B) & 1u, abort_flag, p.status, 88) && (n < 1 || r16_bar(read_dp, (n - 1) & 1u, abort_flag, p.status, 89));
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP, PL>(tmem + COL_DP, r16_desc_k(slot_g), r16_desc_k(ring_v + b * W::TILE));
        umma_commit(bar_dp);
        umma_commit(&empty_v[b]);
      };
      if (ok && walk > 0) scores(0);
      for (int n = 0; ok && n < walk; n++) {
        const uint32_t place = n & 1u;
        if (n + 1 < walk) scores(n + 1);
        if (!(ok = ok && r16_bar(&bar_ds[place], (n >> 1) & 1u, abort_flag, p.status, 90))) break;
        tc_fence_after();
        r16_gather<DP, 64, PL>(tmem + COL_DQ, tmem + COL_S + 128u * place, r16_desc_mn(ring_k + (n % W::RING_A) * W::TILE), PL == 1 && n > 0 ? 1u : 0u);
        umma_commit(&bar_dq[place]);
        umma_commit(&empty_k[n % W::RING_A]);
      }
      if (ok) umma_commit(bar_done);
      else *abort_flag = 1;
    }
  } else {
    const int half = warp >> 2, quad = warp & 3, row = quad * 32 + lane, i = i0 + row;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16), t_dp = lane_base + COL_DP + 64u * half;
    const int at_unit = bi * p.hkv + hk, n_units = p.units_n;    // as in rule16_dkv_kernel
    const float unit_q = PL == 2 ? p.units[at_unit] : 1.f, unit_k = PL == 2 ? p.units[n_units + at_unit] : 1.f, unit_v = PL == 2 ? p.units[2 * n_units + at_unit] : 1.f,
                unit_g = PL == 2 ? p.units[3 * n_units + at_unit] : 1.f, unit = unit_q * unit_k;
    uint8_t* turn = smem + W::TURN;
    float unit_dq = 1.f;
    const R16Score score = r16_score_of<MODE>(r, hi, unit);
    const R16Row seen = r16_query_row(r, prefix, bi, min(i, r.lq - 1));
    const int32_t* docs = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
    const float mult = MODE ? 1.f : r.scale * unit * R16_LOG2E;
    const float2 stat = rule_row(p.rows, (long long)bi * p.h + hi, r.lq, i);
    for (int n = 0; ok && n < walk; n++) {
      const uint32_t step = steps[n], place = n & 1u, phase = (n >> 1) & 1u, t_s = lane_base + COL_S + 128u * place + 64u * half;
      const int at = (first + r16_tile_of(step)) * R16_T + half * 64;
      const bool partial = r16_sees_of(step) == 1;
      ok = r16_wait(&bar_s[place], phase, abort_flag, p.status, 91);
      if (PL == 1 && !ok) break;                           // two planes: both warps of a row leave together, below
      tc_fence_after();
      uint32_t x[2][32], w[16], wl[16];
      tmem_ld_32x32b_x32(t_s, x[0]);
      tmem_ld_32x32b_x32(t_s + 32u, x[1]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 2; c++)
        r16_weights<MODE, false, PL>(score, x[c], w, wl, nullptr, stat.x, 0.f, (float)(i + r.q_offset - at - c * 32), mult, partial,
                                     partial ? r16_bits(seen, at + c * 32, docs) : ~0u);
      ok = ok && r16_wait(bar_dp, n & 1u, abort_flag, p.status, 92);
      if (PL == 1 && !ok) break;
      tc_fence_after();
      if (PL == 2) {
        if (n > 0) {
          // The product before; the next one waits for these gradients.
          ok = ok && r16_wait(&bar_dq[place ^ 1u], ((n - 1) >> 1) & 1u, abort_flag, p.status, 95);
          tc_fence_after();
          r16_fold<32>(lane_base + COL_DQ + 64u + 32u * half, lane_base + COL_DQ + 32u * half, n == 1, 1.f, unit_dq);
        }
        float largest = 0.f;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t dp[32];
          tmem_ld_32x32b_x32(t_dp + 32u * c, dp);
          tmem_ld_wait();
          r16_gradients2<false>(x[c], dp, nullptr, stat.y, unit_g * unit_v, partial, largest);
        }
        r16_arrive_warp(read_dp, lane);
        uint32_t exponent = __float_as_uint(largest) >> 23;
        if (!(ok = r16_share(turn + 256 * place, half, row, quad, ok, exponent))) break;
        const R16Unit step_unit = r16_unit(exponent);
        unit_dq = step_unit.back;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          r16_apart(x[c], step_unit.to, w, wl);
          r16_st16(t_s + 32u * c, w);
          r16_st16(t_s + 32u * c + 16u, wl);
        }
      } else {
        uint32_t dp[2][32];
        tmem_ld_32x32b_x32(t_dp, dp[0]);
        tmem_ld_32x32b_x32(t_dp + 32u, dp[1]);
        tmem_ld_wait();
        r16_arrive_warp(read_dp, lane);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          r16_gradients16<false>(x[c], dp[c], w, nullptr, stat.y, partial);
          r16_st16(t_s + 16u * c, w);
        }
      }
      if (PL == 1 && r16_padded(step))
        r16_clear<DP>(ring_k + n % W::RING_A * W::TILE, r.k_pads + (long long)bi * r.nk64, (first + r16_tile_of(step)) * (R16_T / RULE_GRAIN), r.nk64, warp, lane);
      tmem_st_wait();
      r16_arrive_warp(&bar_ds[place], lane);
    }
    if (ok) ok = r16_wait(bar_done, 0, abort_flag, p.status, 93);
    if (ok) {
      tc_fence_after();
      // Half of dQ's columns by each four warps.
#pragma unroll 1
      for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
        uint32_t o[32];
        __syncwarp();
        if (walk > 0) {
          tmem_ld_32x32b_x32(lane_base + COL_DQ + (uint32_t)c, o);
          tmem_ld_wait();
          if (PL == 2) r16_add_whole(lane_base + COL_DQ + 64u + (uint32_t)c, o, walk == 1, 1.f, unit_dq);
        } else {
#pragma unroll
          for (int u = 0; u < 32; u++) o[u] = 0u;
        }
        if (i < r.lq) r16_write(o, r.scale * unit_k, p.d0, p.d0_16, bi * p.s0.batch + hi * p.s0.head + (long long)i * p.s0.row + c, c, p.d);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == R16_ROW_WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// Rank-4 map over a bfloat16 activation seen as [B, H, L, D] through element strides; box = [64 columns, rows, heads, 1]. Columns
// behind D and rows behind L come as zeros.
static bool r16_map(CUtensorMap* map, const void* base, int d, int l, int heads, int batch, const om_head_strides* s, int box_rows, int box_heads) {
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)l, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t row = (cuuint64_t)s->row * 2;
  cuuint64_t strides[3] = {row, heads > 1 ? (cuuint64_t)s->head * 2 : row, batch > 1 ? (cuuint64_t)s->batch * 2 : row};
  cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_heads, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// What TMA addresses: a 16-byte aligned base, strides that are positive multiples of 16 bytes below 2^40.
static bool r16_operand(const void* p, const om_head_strides* s, int heads, int batch) {
  auto fits = [](int64_t v) { return v > 0 && v % 8 == 0 && v < (1ll << 38); };
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && fits(s->row) && (heads == 1 || fits(s->head)) && (batch == 1 || fits(s->batch));
}
// Rows of results are written 16 bytes at a time.
static bool r16_result(const float* p, const void* p16, const om_head_strides* s) {
  if (p && ((reinterpret_cast<uintptr_t>(p) & 15) || s->row % 4 || s->head % 4 || s->batch % 4)) return false;
  return !p16 || !((reinterpret_cast<uintptr_t>(p16) & 15) || s->row % 8 || s->head % 8 || s->batch % 8);
}
// Tiles are the grid's second axis, 65535 of them at most.
static bool r16_shape(const RuleCall& c) {
  return encode_fn() && c.d % 8 == 0 && c.d <= 128 && c.r.scale > 0.f && c.r.lq <= 65535 * R16_T && c.r.lk <= 65535 * R16_T;
}
static R16Strides r16_strides(const om_head_strides* s) { return R16Strides{s->batch, s->head, s->row}; }

bool rule16_fwd_takes(const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                      const om_head_strides* vs, const float* out, const void* out16, const om_head_strides* os) {
  return r16_shape(c) && r16_operand(q, qs, c.h, c.b) && r16_operand(k, ks, c.hkv, c.b) && r16_operand(v, vs, c.hkv, c.b) && r16_result(out, out16, os);
}
bool rule16_bwd_takes(const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                      const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* dq, const void* dq16, const om_head_strides* dqs,
                      const float* dk, const void* dk16, const om_head_strides* dks, const float* dv, const void* dv16, const om_head_strides* dvs) {
  // Both axes are walked whole, within a plan.
  return r16_shape(c) && c.r.lq <= R16_PLAN * R16_T && c.r.lk <= R16_PLAN * R16_T && r16_operand(g, gs, c.h, c.b) && r16_operand(q, qs, c.h, c.b) && r16_operand(k, ks, c.hkv, c.b) && r16_operand(v, vs, c.hkv, c.b) &&
         (!(dq || dq16) || r16_result(dq, dq16, dqs)) && (!(dk || dk16) || r16_result(dk, dk16, dks)) && (!(dv || dv16) || r16_result(dv, dv16, dvs));
}

template <typename K>
static int32_t r16_room(om_ctx* ctx, K kernel, int smem) {
  OM_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  return OM_OK;
}

template <int DP, int MODE, int PL>
static int32_t r16_fwd(om_ctx* ctx, dim3 grid, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const R16Fwd& p) {
  OM_TRY(r16_room(ctx, rule16_fwd_kernel<DP, MODE, PL>, R16FwdShape<DP, PL>::SMEM));
  launch_chained(ctx, rule16_fwd_kernel<DP, MODE, PL>, grid, R16_THREADS, R16FwdShape<DP, PL>::SMEM, mq, mk, mv, p);
  return OM_OK;
}

template <int DP, int PL>
static int32_t r16_fwd_by_mode(om_ctx* ctx, dim3 grid, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const R16Fwd& p) {
  if (p.r.softcap > 0.f) return r16_fwd<DP, 2, PL>(ctx, grid, mq, mk, mv, p);
  return p.r.slopes ? r16_fwd<DP, 1, PL>(ctx, grid, mq, mk, mv, p) : r16_fwd<DP, 0, PL>(ctx, grid, mq, mk, mv, p);
}

int32_t rule16_fwd(om_ctx* ctx, const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                   const om_head_strides* vs, float* out, void* out16, const om_head_strides* os, float* lse, const RulePlanes* planes) {
  const int group = c.h / c.hkv, lq = c.r.lq, lk = c.r.lk;
  R16Fwd p = {};
  p.r = c.r; p.h = c.h; p.hkv = c.hkv; p.d = c.d;
  p.out = out; p.out16 = reinterpret_cast<__nv_bfloat16*>(out16); p.os = r16_strides(os); p.lse = lse;
  p.rows = (long long)c.b * c.h * lq;
  p.status = ctx->status_dev;
  const int width = planes ? 128 : c.d;                  // columns of the operands: those of two planes are full
  if (planes) {
    p.units = planes->units;
    p.plain = planes->plain;
  }
  // Heads that share keys as rows of one tile where they fit it: keys and values are read once for all of them.
  p.packed = (long long)group * lq <= R16_T && (group > 1);
  dim3 grid((unsigned)(c.b * (p.packed ? c.hkv : c.h)), p.packed ? 1u : (unsigned)ceil_div(lq, R16_T), 1);
  // A walk is split where the CTAs leave SMs without one, four tiles of keys a part at least: a part costs its CTA's start and a
  // row of O per query in memory, twice.
  const int64_t ctas = (int64_t)grid.x * grid.y;
  const int64_t span = c.r.window && !c.r.prefix ? std::min<int64_t>(lk, 2ll * c.r.window + lq) : lk;
  const int64_t tiles = ceil_div(span, R16_T);
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(ctx->sm_count / std::max<int64_t>(ctas, 1), tiles / 4));
  p.splits = (int)std::max<int64_t>(p.splits, ceil_div(ceil_div(lk, R16_T) + 1, R16_PLAN));   // a part is at most a plan long
  grid.z = (unsigned)p.splits;
  CUtensorMap mq, mk, mv;
  if (!r16_map(&mq, q, width, lq, c.h, c.b, qs, p.packed ? lq : R16_T, p.packed ? group : 1) || !r16_map(&mk, k, width, lk, c.hkv, c.b, ks, R16_T, 1) ||
      !r16_map(&mv, v, width, lk, c.hkv, c.b, vs, R16_T, 1))
    return fail(ctx, OM_ERR_CUDA, "cuTensorMapEncodeTiled failed for the operands of om_rule_attention_fwd");
  char* part = nullptr;
  if (p.splits > 1) {
    const size_t ml = ((size_t)p.splits * p.rows * sizeof(float2) + 255) & ~(size_t)255;
    OM_TRY(pool_alloc(ctx, ml + (size_t)p.splits * p.rows * c.d * sizeof(float), false, (void**)&part));
    p.part_ml = reinterpret_cast<float2*>(part);
    p.part = reinterpret_cast<float*>(part + ml);
  }
  const int32_t st = planes ? r16_fwd_by_mode<64, 2>(ctx, grid, mq, mk, mv, p) : c.d <= 64 ? r16_fwd_by_mode<64, 1>(ctx, grid, mq, mk, mv, p) : r16_fwd_by_mode<128, 1>(ctx, grid, mq, mk, mv, p);
  if (p.splits > 1) {
    if (st == OM_OK) launch_chained(ctx, rule16_join_kernel, grid_for(ctx, p.rows, 8), 256, 0, p);
    pool_free(ctx, part);
  }
  OM_TRY(st);
  OM_LAUNCH_CHECK(ctx, "om_rule_attention_fwd_bf16");
  return OM_OK;
}

template <int DP, int MODE, int PL>
static int32_t r16_bwd(om_ctx* ctx, const RuleCall& c, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mg,
                       const R16Bwd& kv, const R16Bwd& q) {
  if (kv.d0 || kv.d0_16 || kv.d1 || kv.d1_16) {
    constexpr int smem = R16BwdShape<DP, PL, true>::SMEM;
    OM_TRY(r16_room(ctx, rule16_dkv_kernel<DP, MODE, PL>, smem));
    launch_chained(ctx, rule16_dkv_kernel<DP, MODE, PL>, dim3((unsigned)(c.b * c.hkv), (unsigned)ceil_div(c.r.lk, R16_T)), R16_THREADS, smem, mq, mk, mv, mg, kv);
  }
  if (q.d0 || q.d0_16) {
    constexpr int smem = R16BwdShape<DP, PL, false>::SMEM;
    OM_TRY(r16_room(ctx, rule16_dq_kernel<DP, MODE, PL>, smem));
    launch_chained(ctx, rule16_dq_kernel<DP, MODE, PL>, dim3((unsigned)(c.b * c.h), (unsigned)ceil_div(c.r.lq, R16_T)), R16_THREADS, smem, mq, mk, mv, mg, q);
  }
  return OM_OK;
}

template <int DP, int PL>
static int32_t r16_bwd_by_mode(om_ctx* ctx, const RuleCall& c, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mg,
                               const R16Bwd& kv, const R16Bwd& q) {
  if (c.r.softcap > 0.f) return r16_bwd<DP, 2, PL>(ctx, c, mq, mk, mv, mg, kv, q);
  return c.r.slopes ? r16_bwd<DP, 1, PL>(ctx, c, mq, mk, mv, mg, kv, q) : r16_bwd<DP, 0, PL>(ctx, c, mq, mk, mv, mg, kv, q);
}

int32_t rule16_bwd(om_ctx* ctx, const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                   const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* rows, float* dq, void* dq16,
                   const om_head_strides* dqs, float* dk, void* dk16, const om_head_strides* dks, float* dv, void* dv16, const om_head_strides* dvs,
                   const RulePlanes* planes) {
  const int lq = c.r.lq, lk = c.r.lk, width = planes ? 128 : c.d;
  CUtensorMap mq, mk, mv, mg;
  if (!r16_map(&mq, q, width, lq, c.h, c.b, qs, R16_T, 1) || !r16_map(&mk, k, width, lk, c.hkv, c.b, ks, R16_T, 1) ||
      !r16_map(&mv, v, width, lk, c.hkv, c.b, vs, R16_T, 1) || !r16_map(&mg, g, width, lq, c.h, c.b, gs, R16_T, 1))
    return fail(ctx, OM_ERR_CUDA, "cuTensorMapEncodeTiled failed for the operands of om_rule_attention_bwd_bf16");
  R16Bwd kv = {};
  kv.r = c.r; kv.h = c.h; kv.hkv = c.hkv; kv.d = c.d; kv.rows = rows; kv.tiles = rule_row_tiles(lq); kv.status = ctx->status_dev;
  if (planes) {
    kv.units = planes->units;
    kv.units_n = c.b * c.hkv;
    kv.plain = planes->plain;
  }
  R16Bwd one = kv;
  kv.d0 = dv; kv.d1 = dk; kv.d0_16 = reinterpret_cast<__nv_bfloat16*>(dv16); kv.d1_16 = reinterpret_cast<__nv_bfloat16*>(dk16);
  if (dv || dv16) kv.s0 = r16_strides(dvs);
  if (dk || dk16) kv.s1 = r16_strides(dks);
  one.d0 = dq; one.d0_16 = reinterpret_cast<__nv_bfloat16*>(dq16);
  if (dq || dq16) one.s0 = r16_strides(dqs);
  const int32_t st = planes ? r16_bwd_by_mode<64, 2>(ctx, c, mq, mk, mv, mg, kv, one)
                     : c.d <= 64 ? r16_bwd_by_mode<64, 1>(ctx, c, mq, mk, mv, mg, kv, one) : r16_bwd_by_mode<128, 1>(ctx, c, mq, mk, mv, mg, kv, one);
  OM_TRY(st);
  OM_LAUNCH_CHECK(ctx, "om_rule_attention_bwd_bf16");
  return OM_OK;
}

// ---- two planes -----------------------------------------------------------------------------------------------------------------

struct R16Source {
  const float* x;                 // [b, heads, l, d] through strides
  R16Strides s;
  __half* planes;                 // [b * heads][l][128]: h in columns 0 to 63, l behind, zeros beyond d
  int heads, l, quads;
  const int32_t* docs;            // [b, l] or NULL: rows of no document are taken for zeros, so that what they hold changes nothing
};
struct R16Split {
  R16Source t[4];                 // q, k, v, g
  int d, hkv, b;
  uint32_t* top;                  // [4][b * hkv] bits of the largest absolute value
  float* units;                   // [4][b * hkv]: of q, k, v and g
  int32_t* plain;                 // [b * hkv]
};
constexpr int R16_SPLIT_ROWS = 64;

// A CTA has 64 rows of one head of one operand, four threads a row with 16 columns each.
__device__ __forceinline__ void r16_fetch(const R16Split& p, const R16Source& t, int bh, int row, float (&v)[16]) {
  const int c0 = (threadIdx.x & 3) * 16, bi = bh / t.heads, hi = bh - bi * t.heads;
  const float* x = t.x + bi * t.s.batch + hi * t.s.head + (long long)row * t.s.row;
  const bool some = row < t.l && (!t.docs || ld_global(t.docs + (long long)bi * t.l + row) >= 0);
#pragma unroll
  for (int c = 0; c < 16; c += 4) {
    if (some && t.quads && c0 + c < p.d) {
      const float4 f = *reinterpret_cast<const float4*>(x + c0 + c);
      v[c] = f.x; v[c + 1] = f.y; v[c + 2] = f.z; v[c + 3] = f.w;
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++) v[c + u] = some && c0 + c + u < p.d ? x[c0 + c + u] : 0.f;
    }
  }
}
__device__ __forceinline__ uint32_t r16_largest(const float (&v)[16]) {
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < 16; u++) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);   // of bits: what is not a number counts as the largest
  return m;
}
__global__ void __launch_bounds__(256) rule16_largest_kernel(const __grid_constant__ R16Split p) {
  pdl_enter();
  const R16Source& t = p.t[blockIdx.z];
  const int bh = blockIdx.x, row = blockIdx.y * R16_SPLIT_ROWS + (threadIdx.x >> 2);
  if (!t.x || bh >= p.b * t.heads || (int)blockIdx.y * R16_SPLIT_ROWS >= t.l) return;
  float v[16];
  r16_fetch(p, t, bh, row, v);
  uint32_t m = __reduce_max_sync(0xffffffffu, r16_largest(v));
  __shared__ uint32_t all[8];
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; w++) m = max(m, all[w]);
    const int bi = bh / t.heads, hk = (bh - bi * t.heads) / (t.heads / p.hkv);
    const int at = ((int)blockIdx.z * p.b + bi) * p.hkv + hk;
    atomicMax(&p.top[at], m);                            // whole numbers: the order does not matter
  }
}
__global__ void __launch_bounds__(256) rule16_split_kernel(const __grid_constant__ R16Split p) {
  pdl_enter();
  const R16Source& t = p.t[blockIdx.z];
  const int bh = blockIdx.x, row = blockIdx.y * R16_SPLIT_ROWS + (threadIdx.x >> 2);
  if (!t.x || bh >= p.b * t.heads || (int)blockIdx.y * R16_SPLIT_ROWS >= t.l) return;
  float v[16];
  r16_fetch(p, t, bh, row, v);
  const int bi = bh / t.heads, hk = (bh - bi * t.heads) / (t.heads / p.hkv), at = ((int)blockIdx.z * p.b + bi) * p.hkv + hk;
  const uint32_t top = ld_global(p.top + at);
  uint32_t mine = r16_largest(v);
  mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
  // The largest goes to 2^14 ... 2^15. Units below 2^-60 would leave fp32 in their products, and so would, above 2^30 (values of 2^45), the
  // gradients of scores times half-precision values of 2^15.
  const int e = top == 0 ? 0 : (int)(top >> 23) - 127 - 14;
  const bool fits = top < 0x7f800000u && e >= -60 && e <= 30;
  const bool far = mine != 0 && (mine >> 23) + 14 < (top >> 23);
  if ((threadIdx.x & 3) == 0 && (!fits || far)) p.plain[bi * p.hkv + hk] = 1;
  const float unit = __uint_as_float((uint32_t)((fits ? e : 0) + 127) << 23), to = __uint_as_float((uint32_t)(127 - (fits ? e : 0)) << 23);
  if (threadIdx.x == 0) p.units[at] = unit;
  if (row >= t.l) return;
  uint32_t h[8], l[8];
#pragma unroll
  for (int u = 0; u < 8; u++) r16_take_apart(v[2 * u] * to, v[2 * u + 1] * to, &h[u], &l[u]);
  uint4* out = reinterpret_cast<uint4*>(t.planes + ((long long)bh * t.l + row) * 128 + (threadIdx.x & 3) * 16);
  out[0] = make_uint4(h[0], h[1], h[2], h[3]);
  out[1] = make_uint4(h[4], h[5], h[6], h[7]);
  out[8] = make_uint4(l[0], l[1], l[2], l[3]);
  out[9] = make_uint4(l[4], l[5], l[6], l[7]);
}

// fp32 calls that are worth the two passes over the operands in front. What decides is the longest walk of a block: the fp32 kernels take
// 0.2 to 0.4 us for each key or query of it, however little else there is, these a fixed 25 us forward and 60 us both ways and hardly more
// for a long walk. Forward and backward of 12 heads of 64, fp32 kernels against these: length 64, one batch 58 and 65 us, 64 batches
// 225 and 275; 96, one batch 85 and 63, 16 batches 181 and 117; 128, one batch 92 and 66; 256 163 and 74; 1024 818 and 143. One query to 512
// keys, forward, 68 and 25. 96 is where both directions together come out even or better with every number of batches and with heads of 8 to 64.
constexpr int R16_WALK = 96;
bool rule16_planes_take(const RuleCall& c, bool backward) {
  return r16_shape(c) && c.d <= 64 && c.r.lk <= R16_PLAN * R16_T && (!backward || c.r.lq <= R16_PLAN * R16_T) &&
         (backward ? std::max(c.r.lq, c.r.lk) : c.r.lk) >= R16_WALK && ceil_div(std::max(c.r.lq, c.r.lk), R16_SPLIT_ROWS) <= 65535;
}
bool rule16_result_fits(const float* p, const om_head_strides* s) { return p == nullptr || r16_result(p, nullptr, s); }

int32_t rule16_planes(om_ctx* ctx, const RuleCall& c, const float* q, const om_head_strides* qs, const float* k, const om_head_strides* ks, const float* v,
                      const om_head_strides* vs, const float* g, const om_head_strides* gs, RulePlanes* out) {
  const size_t nq = (size_t)c.b * c.h * c.r.lq * 128, nk = (size_t)c.b * c.hkv * c.r.lk * 128, units = (size_t)c.b * c.hkv * 4;
  const size_t head = sizeof(uint32_t) * (units + units / 4), bytes = sizeof(__half) * (nq * (g ? 2 : 1) + 2 * nk);
  out->small = out->large = nullptr;
  OM_TRY(pool_alloc(ctx, head, true, &out->small));
  const int32_t st = pool_alloc(ctx, bytes + sizeof(float) * units, false, &out->large);
  if (st != OM_OK) {
    rule16_planes_end(ctx, out);
    return st;
  }
  __half* at = reinterpret_cast<__half*>(out->large);
  R16Split p = {};
  p.d = c.d; p.hkv = c.hkv; p.b = c.b;
  p.top = reinterpret_cast<uint32_t*>(out->small);
  p.plain = reinterpret_cast<int32_t*>(p.top + units);
  auto source = [&](const float* x, const om_head_strides* s, int heads, int l, const int32_t* docs) {
    R16Source t = {};
    t.x = x; t.s = r16_strides(s); t.planes = at; t.heads = heads; t.l = l; t.docs = docs;
    t.quads = c.d % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && s->row % 4 == 0 && s->head % 4 == 0 && s->batch % 4 == 0;
    at += (size_t)c.b * heads * l * 128;
    return t;
  };
  p.t[0] = source(q, qs, c.h, c.r.lq, c.r.q_docs);
  p.t[1] = source(k, ks, c.hkv, c.r.lk, c.r.k_docs);
  p.t[2] = source(v, vs, c.hkv, c.r.lk, c.r.k_docs);
  if (g) p.t[3] = source(g, gs, c.h, c.r.lq, c.r.q_docs);
  p.units = reinterpret_cast<float*>(at);
  for (int i = 0; i < 4; i++) out->p[i] = p.t[i].planes;
  out->q = om_head_strides{(int64_t)c.h * c.r.lq * 128, (int64_t)c.r.lq * 128, 128};
  out->k = om_head_strides{(int64_t)c.hkv * c.r.lk * 128, (int64_t)c.r.lk * 128, 128};
  out->units = p.units;
  out->plain = p.plain;
  const dim3 grid((unsigned)(c.b * c.h), (unsigned)ceil_div(std::max(c.r.lq, c.r.lk), R16_SPLIT_ROWS), g ? 4u : 3u);
  launch_chained(ctx, rule16_largest_kernel, grid, 256, 0, p);
  launch_chained(ctx, rule16_split_kernel, grid, 256, 0, p);
  return OM_OK;
}
void rule16_planes_end(om_ctx* ctx, RulePlanes* planes) {
  if (planes->small) pool_free(ctx, planes->small);
  if (planes->large) pool_free(ctx, planes->large);
}

}  // namespace om
