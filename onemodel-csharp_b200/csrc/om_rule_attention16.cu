// Attention by rule with bfloat16 operands on the tensor pipe (tcgen05), forward and backward, for head dimensions up to 128.
//
// Forward: a CTA holds 256 queries as two tiles of 128 and walks the keys that the rule lets them see, 64 at a time. Eight warps per
// query tile keep the running maximum and sum of its rows, two threads a row. Scores S = Q K^T come to tensor memory in fp32; the rows
// take them to registers, which frees their place for the next scores at once, and put the weights exp2(S - m), rounded to bfloat16,
// into one of two places beside them, from where O += P V reads them. So the tensor pipe works on the next scores of both tiles and on
// the products behind while the rows form exponentials, and every reuse of a place in tensor memory has a barrier of its own. O stays
// in tensor memory; it is rescaled only when a row's maximum has grown by more than 2^8 over the one in use, which changes no result:
// numerator and denominator share the factor.
// With few rows the walk over the keys is split over CTAs that leave their sums, maxima and O for rule16_join_kernel, and the query
// heads that share a key head become rows of one tile, so that keys and values are read once.
//
// Backward: the weights come back from the forward's log-sum-exp, once in rule16_dkv_kernel (a CTA per 128 keys walks the queries of
// all heads that share them; rows are keys: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q) and once in rule16_dq_kernel (a
// CTA per 128 queries walks the keys: dQ += dS K). Seven products for five, but no partial sums through memory: a part of dQ per
// (query tile, key tile) is 128 KB of traffic against 0.3 us of tensor time for the two products that are done again.
// Two sets of eight warps of rows take turns, so that a set has two steps' time for one. P and dS are rounded to bfloat16 as operands
// (the only roundings of the backward besides the results').
//
// What a CTA sees of the other axis is worked out before its walk, a byte per 128 indices: worked out along the way it cost the rows as
// much as their exponentials. Every wait is bounded (om_tc.cuh). All sums are fp32 in an order that the shapes alone decide.
#include <cuda_bf16.h>
#include <math.h>

#include "om_rule.cuh"
#include "om_tc.cuh"

namespace om {

constexpr int R16_T = 128;                         // rows of every tile
constexpr int R16_CHUNK = R16_T * 128;             // bytes of a [128 x 64] bfloat16 block, 128-byte swizzled rows
constexpr int R16_ROW_WARPS = 16;
constexpr int R16_THREADS = 32 * (R16_ROW_WARPS + 2);   // warps 0-15: rows; warp 16: MMA issue; warp 17: TMA
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
// tanh(x) = 1 - 2 / (exp(2 x) + 1): off by 2^-22 at most, absolutely, which a cap times it carries into a score.
__device__ __forceinline__ float r16_tanh(float x) { return fmaf(-2.f, r16_rcp(r16_ex2(x * (2.f * R16_LOG2E)) + 1.f), 1.f); }
__device__ __forceinline__ uint32_t r16_pack(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Shared-memory descriptors share their upper word (stride offset 1024 bytes, version 1, 128-byte swizzle); the lower one is
// (address >> 4) with the leading offset, one block of 64 columns for MN-major operands.
constexpr uint32_t R16_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t R16_LBO_K = 1u << 16, R16_LBO_MN = ((uint32_t)R16_CHUNK >> 4) << 16;
__device__ __forceinline__ uint32_t r16_desc_k(const void* p) { return (smem_u32(p) >> 4) | R16_LBO_K; }
__device__ __forceinline__ uint32_t r16_desc_mn(const void* p) { return (smem_u32(p) >> 4) | R16_LBO_MN; }
// kind::f16 with bfloat16 operands and fp32 sums, M = 128.
__device__ __forceinline__ constexpr uint32_t r16_idesc(bool b_mn, int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(R16_T >> 4) << 24);
}
__device__ __forceinline__ void r16_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, {%6, %6, %6, %6}, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(R16_DESC_HI), "r"(0u)
      : "memory");
}
// A from tensor memory: row r in lane r, elements 2 c and 2 c + 1 of the contraction in column c.
__device__ __forceinline__ void r16_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, {%6, %6, %6, %6}, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(R16_DESC_HI), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void r16_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void r16_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void r16_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[128 x 64] = A B^T over the head's columns, both operands K-major in shared memory; b_k: 64 rows of B.
template <int DP>
__device__ __forceinline__ void r16_scores(uint32_t d, uint32_t a_k, uint32_t b_k) {
  constexpr uint32_t idesc = r16_idesc(false, 64);
#pragma unroll
  for (int ks = 0; ks < DP / 16; ks++) {
    const uint32_t o = (uint32_t)(ks / 4) * (R16_CHUNK >> 4) + (uint32_t)(ks % 4) * 2;
    r16_mma_ss(d, a_k + o, b_k + o, idesc, ks > 0 ? 1u : 0u);
  }
}
constexpr uint32_t R16_HALF_K = (64u * 128u) >> 4, R16_HALF_MN = (64u * 128u) >> 4;   // the second 64 rows of a tile
// D[128 x DP] (+)= A B over 64 rows of B: A [128 x 64] packed in 32 columns of tensor memory, B MN-major in shared memory.
template <int DP>
__device__ __forceinline__ void r16_gather(uint32_t d, uint32_t a, uint32_t b_mn, uint32_t accumulate) {
  constexpr uint32_t idesc = r16_idesc(true, DP);
#pragma unroll
  for (int ks = 0; ks < 4; ks++) r16_mma_ts(d, a + (uint32_t)ks * 8u, b_mn + (uint32_t)ks * 128u, idesc, ks > 0 ? 1u : accumulate);
}
template <int DP>
__device__ __forceinline__ void r16_load_tile(uint8_t* dst, const CUtensorMap* map, int row0, int head, int batch, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < DP / 64; c++) tma_load_4d(dst + c * R16_CHUNK, map, c * 64, row0, head, batch, bar);
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
// The score in powers of two of a product, and the cap's derivative.
__device__ __forceinline__ float r16_score(const RuleArgs& r, float slope, int far, float dot, float* dcap) {
  float s = dot * r.scale;
  if (r.softcap > 0.f) {
    const float t = r16_tanh(s * r.inv_softcap);
    *dcap = fmaf(-t, t, 1.f);
    s = r.softcap * t;
  } else {
    *dcap = 1.f;
  }
  return fmaf(-slope, (float)abs(far), s) * R16_LOG2E;
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
  int32_t* status;
};

// A CTA's plan: the steps of its walk in order, a step being 64 indices of the other axis that some row tile sees anything of.
constexpr uint32_t R16_OPENS = 1u << 12, R16_CLOSES = 1u << 13;      // the first, the last step of its tile of 128
__device__ __forceinline__ int r16_tile_of(uint32_t step) { return (int)(step & 1023u); }
__device__ __forceinline__ uint32_t r16_half_of(uint32_t step) { return (step >> 10) & 1u; }
__device__ __forceinline__ int r16_sees_of(uint32_t step, int tile) { return (int)(step >> (16 + 2 * tile)) & 3; }
// By one warp: `see(tile, half)` gives rule_see's answers, two bits a row tile. Returns the number of steps.
template <typename F>
__device__ __forceinline__ int r16_plan(uint32_t* steps, int tiles, int lane, F see) {
  int n = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const int t = t0 + lane;
    uint32_t a = 0, b = 0;
    if (t < tiles) {
      a = see(t, 0);
      b = see(t, 1);
    }
    const uint32_t first = __ballot_sync(0xffffffffu, a != 0), second = __ballot_sync(0xffffffffu, b != 0), below = (1u << lane) - 1u;
    int at = n + __popc(first & below) + __popc(second & below);
    if (a) steps[at++] = (uint32_t)t | R16_OPENS | (b ? 0u : R16_CLOSES) | a << 16;
    if (b) steps[at] = (uint32_t)t | 1u << 10 | (a ? 0u : R16_OPENS) | R16_CLOSES | b << 16;
    n += __popc(first) + __popc(second);
  }
  return n;
}

template <int DP>
struct R16FwdShape {
  static constexpr int TILE = DP / 64 * R16_CHUNK;
  static constexpr int STAGES = DP == 128 ? 4 : 8;       // of K and V tiles in turn
  static constexpr int MAXIMA = (2 + STAGES) * TILE;     // [parity][query tile][half][128] floats, and the halves' sums in the end
  static constexpr int RULES = MAXIMA + 4096;
  static constexpr int PLAN = RULES + 128;
  static constexpr int BARS = PLAN + 2 * R16_PLAN * 4 + 16;
  static constexpr int SMEM = BARS + 512 + 1024;
};

template <int DP, bool EXTRA>
__global__ void __launch_bounds__(R16_THREADS, 1)
rule16_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ R16Fwd p) {
  typedef R16FwdShape<DP> W;
  // Of query tile g at 64 g: the scores; at 128 + 64 g: the two places of its weights, 32 columns each; at 256 + 128 g: O.
  constexpr uint32_t COL_S = 0, COL_P = 128, COL_O = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *slot_q = smem, *ring = smem + 2 * W::TILE;
  uint32_t* steps = reinterpret_cast<uint32_t*>(smem + W::PLAN);
  float* maxima = reinterpret_cast<float*>(smem + W::MAXIMA);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  uint64_t *bar_q = bars, *bar_s = bars + 1 /* [tile] */, *bar_read = bars + 3 /* [tile] */, *bar_p = bars + 5 /* [tile][place] */, *bar_o = bars + 9 /* [tile][place] */,
           *bar_max = bars + 13 /* [tile][quad] */, *bar_full = bars + 21 /* [STAGES] */, *bar_empty = bar_full + W::STAGES;
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
    i0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * 2 * R16_T;      // the longest walks of a causal mask first
  }
  const int both = !p.packed && i0 + R16_T < r.lq;

  if (threadIdx.x == 0) {
    mbar_init(bar_q, 1);
    for (int a = 0; a < 2; a++) {
      mbar_init(&bar_s[a], 1);
      mbar_init(&bar_read[a], R16_ROW_WARPS / 2);
    }
    for (int a = 0; a < 4; a++) {
      mbar_init(&bar_p[a], R16_ROW_WARPS / 2);
      mbar_init(&bar_o[a], 1);
    }
    for (int a = 0; a < 8; a++) mbar_init(&bar_max[a], 2);
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
  RuleTile* tiles = reinterpret_cast<RuleTile*>(smem + W::RULES);
  if (threadIdx.x < 64 && lane == 0) tiles[warp] = rule_query_tile(r, prefix, bi, warp == 0 ? i0 : both ? i0 + R16_T : r.lq, 2);
  const RuleSpan span = rule_keys(r, prefix, i0, min(p.packed ? r.lq : i0 + 2 * R16_T, r.lq));
  int first = span.prefix > 0 ? 0 : span.lo / R16_T, last = (max(span.prefix, span.hi) + R16_T - 1) / R16_T;
  const int per = max(0, last - first + p.splits - 1) / p.splits;
  first += split * per;
  last = min(first + per, last);
  __syncthreads();
  if (warp == 0) {
    const int n = r16_plan(steps, last - first, lane, [&](int t, int e) {
      const int at = (first + t) * R16_T + e * 64;
      return (uint32_t)(rule_see<true>(tiles[0], at, 1) | rule_see<true>(tiles[1], at, 1) << 2);
    });
    if (lane == 0) steps[2 * R16_PLAN] = (uint32_t)n;
  }
  __syncthreads();
  const int walk = (int)steps[2 * R16_PLAN];

  const int g = (warp >> 3) & 1, half = (warp >> 2) & 1, quad = warp & 3, row = quad * 32 + lane;
  float m = -INFINITY, l = 0.f;
  uint32_t count = 0;
  bool ok = true;
  if (warp == R16_ROW_WARPS + 1) {
    if (lane == 0) {
      if (p.packed) {
        mbar_expect_tx(bar_q, (uint32_t)(DP / 64) * (uint32_t)(group * r.lq) * 128u);
        r16_load_tile<DP>(slot_q, &map_q, 0, hi, bi, bar_q);
      } else {
        mbar_expect_tx(bar_q, (uint32_t)W::TILE * (both ? 2u : 1u));
        r16_load_tile<DP>(slot_q, &map_q, i0, hi, bi, bar_q);
        if (both) r16_load_tile<DP>(slot_q + W::TILE, &map_q, i0 + R16_T, hi, bi, bar_q);
      }
      int s = 0;
      uint32_t phase = 0;
      bool again = false;
      for (int n = 0; ok && n < walk; n++) {
        const uint32_t step = steps[n];
        if (!(step & R16_OPENS)) continue;
        for (int kv = 0; kv < 2 && ok; kv++) {
          if (again) ok = r16_bar(&bar_empty[s], phase ^ 1u, abort_flag, p.status, 61);
          if (!ok) break;
          mbar_expect_tx(&bar_full[s], W::TILE);
          r16_load_tile<DP>(ring + s * W::TILE, kv ? &map_v : &map_k, (first + r16_tile_of(step)) * R16_T, hk, bi, &bar_full[s]);
          if (++s == W::STAGES) {
            s = 0;
            phase ^= 1u;
            again = true;
          }
        }
      }
    }
  } else if (warp == R16_ROW_WARPS) {
    if (lane == 0) {
      ok = r16_bar(bar_q, 0, abort_flag, p.status, 62);
      int s = 0, ks = 0, vs = 0;                          // the ring's next tile, and those of the steps at hand
      uint32_t phase = 0, scored[2] = {0, 0}, summed[2] = {0, 0};
      auto take = [&]() {
        const int at = s;
        ok = ok && r16_bar(&bar_full[s], phase, abort_flag, p.status, 63);
        if (++s == W::STAGES) {
          s = 0;
          phase ^= 1u;
        }
        return at;
      };
      // The scores of a step for every query tile that sees something of it.
      auto scores = [&](uint32_t step) {
        if (step & R16_OPENS) ks = take();
#pragma unroll
        for (int t = 0; t < 2; t++) {
          if (!ok || !r16_sees_of(step, t)) continue;
          // The rows have taken the scores before to registers.
          if (scored[t] > 0) ok = r16_bar(&bar_read[t], (scored[t] - 1) & 1u, abort_flag, p.status, 64);
          if (!ok) break;
          tc_fence_after();
          r16_scores<DP>(tmem + COL_S + 64u * t, r16_desc_k(slot_q + t * W::TILE), r16_desc_k(ring + ks * W::TILE) + r16_half_of(step) * R16_HALF_K);
          umma_commit(&bar_s[t]);
          scored[t]++;
        }
        if (ok && (step & R16_CLOSES)) umma_commit(&bar_empty[ks]);
      };
      uint32_t step = walk > 0 ? steps[0] : 0u;
      if (ok && walk > 0) scores(step);
      for (int n = 0; ok && n < walk; n++) {
        const uint32_t ahead = n + 1 < walk ? steps[n + 1] : 0u;
        if (step & R16_OPENS) vs = take();
        if (ok && n + 1 < walk) scores(ahead);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          if (!ok || !r16_sees_of(step, t)) continue;
          const uint32_t place = summed[t] & 1u;
          ok = r16_bar(&bar_p[t * 2 + place], (summed[t] >> 1) & 1u, abort_flag, p.status, 65);
          if (!ok) break;
          tc_fence_after();
          r16_gather<DP>(tmem + COL_O + 128u * t, tmem + COL_P + 64u * t + 32u * place, r16_desc_mn(ring + vs * W::TILE) + r16_half_of(step) * R16_HALF_MN,
                         summed[t] > 0 ? 1u : 0u);
          umma_commit(&bar_o[t * 2 + place]);
          summed[t]++;
        }
        if (ok && (step & R16_CLOSES)) umma_commit(&bar_empty[vs]);
        step = ahead;
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    int i = i0 + g * R16_T + row, head = hi;
    if (p.packed) {
      const int gi = row / r.lq;
      i = g == 0 && gi < group ? row - gi * r.lq : 0;
      head = g == 0 && gi < group ? hi + gi : hi;
    }
    const float slope = EXTRA && r.slopes ? r.slopes[head] : 0.f;
    const R16Row seen = r16_query_row(r, prefix, bi, min(i, r.lq - 1));
    const int32_t* docs = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_s = lane_base + COL_S + 64u * g + 32u * half, t_p = lane_base + COL_P + 64u * g + 16u * half,
                   t_o = lane_base + COL_O + 128u * g + (uint32_t)(DP / 2) * half;
    const float mult = EXTRA ? 1.f : r.scale * R16_LOG2E;
    const uint64_t mult2 = r16_two(mult, mult);
    for (int n = 0; ok && n < walk; n++) {
      const uint32_t step = steps[n];
      const int sees = r16_sees_of(step, g);
      if (!sees) continue;
      if (!(ok = r16_wait(&bar_s[g], count & 1u, abort_flag, p.status, 66))) break;
      tc_fence_after();
      uint32_t x[32];
      tmem_ld_32x32b_x32(t_s, x);
      tmem_ld_wait();
      r16_arrive_warp(&bar_read[g], lane);
      const int j = (first + r16_tile_of(step)) * R16_T + (int)r16_half_of(step) * 64 + half * 32;
      if (EXTRA) {
        const int far = i + r.q_offset - j;
#pragma unroll
        for (int u = 0; u < 32; u++) {
          float dcap;
          x[u] = __float_as_uint(r16_score(r, slope, far - u, __uint_as_float(x[u]), &dcap));
        }
      }
      if (sees == 1) r16_hide(x, r16_bits(seen, j, docs));
      float t[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        t[e] = fmaxf(__uint_as_float(x[8 * e]), __uint_as_float(x[8 * e + 1]));
#pragma unroll
        for (int u = 2; u < 8; u += 2) t[e] = r16_max3(t[e], __uint_as_float(x[8 * e + u]), __uint_as_float(x[8 * e + u + 1]));
      }
      float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      // The other half of the row is with another warp.
      float* slots = maxima + ((count & 1u) * 2 + g) * 256;
      slots[half * 128 + row] = top;
      __syncwarp();
      if (lane == 0) r16_arrive(&bar_max[g * 4 + quad]);
      if (!(ok = r16_wait(&bar_max[g * 4 + quad], count & 1u, abort_flag, p.status, 68))) break;
      top = fmaxf(top, slots[(half ^ 1) * 128 + row]) * mult;
      const bool grown = top > m + 8.f || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, grown)) {
        const float shrink = grown ? r16_ex2(m - top) : 1.f;      // m = -inf: 0
        if (grown) m = top;
        l *= shrink;
        if (count > 0) {
          const uint32_t before = count - 1;
          if (!(ok = r16_wait(&bar_o[g * 2 + (before & 1u)], (before >> 1) & 1u, abort_flag, p.status, 69))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DP / 2; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + (uint32_t)c, o);
            tmem_ld_wait();
#pragma unroll
            for (int u = 0; u < 32; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * shrink);
            r16_st32(t_o + (uint32_t)c, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m;
      const uint64_t base2 = r16_two(-base, -base);
      uint64_t sum[2] = {0ull, 0ull};
      uint32_t w[16];
#pragma unroll
      for (int u = 0; u < 16; u++) {
        float a, b;
        r16_fma2(a, b, x[2 * u], x[2 * u + 1], mult2, base2);
        a = r16_ex2(a);
        b = r16_ex2(b);
        sum[u & 1] = r16_add2(sum[u & 1], a, b);
        w[u] = r16_pack(a, b);
      }
      const float2 s0 = *reinterpret_cast<const float2*>(&sum[0]), s1 = *reinterpret_cast<const float2*>(&sum[1]);
      l += (s0.x + s0.y) + (s1.x + s1.y);
      const uint32_t place = count & 1u;
      // The product before last has read this place.
      if (count >= 2 && !(ok = r16_wait(&bar_o[g * 2 + place], ((count - 2) >> 1) & 1u, abort_flag, p.status, 60))) break;
      tc_fence_after();
      r16_st16(t_p + 32u * place, w);
      r16_st_wait();
      r16_arrive_warp(&bar_p[g * 2 + place], lane);
      count++;
    }
    if (ok && count > 0) ok = r16_wait(&bar_o[g * 2 + ((count - 1) & 1u)], ((count - 1) >> 1) & 1u, abort_flag, p.status, 67);
    tc_fence_after();
    maxima[(g * 2 + half) * 128 + row] = l;
  }
  __syncthreads();
  if (warp < R16_ROW_WARPS && ok && (g == 0 || both)) {
    int i = i0 + g * R16_T + row, head = hi;
    bool valid = i < r.lq;
    if (p.packed) {
      const int gi = row / r.lq;
      i = row - gi * r.lq;
      head = hi + gi;
      valid = gi < group;
    }
    l += maxima[(g * 2 + (half ^ 1)) * 128 + row];
    const uint32_t t_o = tmem + ((uint32_t)(quad * 32) << 16) + COL_O + 128u * g + (uint32_t)(DP / 2) * half;
    const long long at_row = ((long long)bi * p.h + head) * r.lq + i;
    float inv = l == 0.f ? 0.f : 1.f / l;
    float* out = p.out;
    __nv_bfloat16* out16 = p.out16;
    long long at = bi * p.os.batch + head * p.os.head + (long long)i * p.os.row;
    if (p.splits > 1) {
      inv = 1.f;
      out = p.part;
      out16 = nullptr;
      at = ((long long)split * p.rows + at_row) * p.d;
      if (valid && half == 0) p.part_ml[(long long)split * p.rows + at_row] = make_float2(m, l);
    } else if (p.lse && valid && half == 0) {
      p.lse[at_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * R16_LN2;
    }
#pragma unroll 1
    for (int c = 0; c < DP / 2; c += 32) {
      uint32_t o[32];
      __syncwarp();
      if (count > 0) {
        tmem_ld_32x32b_x32(t_o + (uint32_t)c, o);
        tmem_ld_wait();
      }
      if (count == 0 || l == 0.f) {
#pragma unroll
        for (int u = 0; u < 32; u++) o[u] = 0u;
      }
      const int col = half * (DP / 2) + c;
      if (valid) r16_write(o, inv, out, out16, at + col, col, p.d);
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
    const long long bh = row / p.r.lq;
    const int i = (int)(row - bh * p.r.lq), bi = (int)(bh / p.h), hi = (int)(bh - (long long)bi * p.h);
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
  int32_t* status;
};

template <int DP>
struct R16BwdShape {
  static constexpr int TILE = DP / 64 * R16_CHUNK;
  static constexpr int RING = 2;
  static constexpr int ROWS = (2 + 2 * RING) * TILE;     // the queries' log-sum-exps and row dots, 1 KB a stage
  static constexpr int RULES = ROWS + RING * 1024;
  static constexpr int PLAN = RULES + 64;
  static constexpr int BARS = PLAN + 2 * R16_PLAN * 4 + 16;
  static constexpr int SMEM = BARS + 256 + 1024;
};

// Scores of one row (32 of them, a quarter of a tile) to weights: packed as bfloat16 in w where they are wanted, and in x, times the
// cap's derivative, for r16_gradients. Rows are keys (COLUMNS: the log-sum-exps go with the columns) or queries.
template <bool EXTRA, bool COLUMNS>
__device__ __forceinline__ void r16_weights(const RuleArgs& r, uint32_t (&x)[32], uint32_t (&w)[16], const float* lses, float lse, float slope, int far, float mult,
                                            bool partial, const R16Row& seen, int at, const int32_t* docs) {
  float dcap[EXTRA ? 32 : 1];
  if (EXTRA) {
#pragma unroll
    for (int u = 0; u < 32; u++)
      x[u] = __float_as_uint(r16_score(r, slope, COLUMNS ? far + u : far - u, __uint_as_float(x[u]), &dcap[EXTRA ? u : 0]));
  }
  if (partial) r16_hide(x, r16_bits(seen, at, docs));
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
      r16_fma2(p[t], p[t + 1], x[u + t], x[u + t + 1], mult2, r16_two(-e[t], -e[t + 1]));
      p[t] = r16_ex2(p[t]);
      p[t + 1] = r16_ex2(p[t + 1]);
      if (COLUMNS) w[(u + t) / 2] = r16_pack(p[t], p[t + 1]);
    }
#pragma unroll
    for (int t = 0; t < 4; t++) x[u + t] = __float_as_uint(EXTRA ? p[t] == 0.f ? 0.f : p[t] * dcap[EXTRA ? u + t : 0] : p[t]);
  }
}
// dS = weight (dP - dot), 32 of them, packed. partial: some are hidden, and 0 whatever dP is there.
template <bool COLUMNS>
__device__ __forceinline__ void r16_gradients(const uint32_t (&x)[32], const uint32_t (&dp)[32], uint32_t (&w)[16], const float* dots, float dot, bool partial) {
  float v[32];
#pragma unroll
  for (int u = 0; u < 32; u += 4) {
    float d[4] = {dot, dot, dot, dot};
    if (COLUMNS) {
      const float4 f = *reinterpret_cast<const float4*>(dots + u);
      d[0] = f.x; d[1] = f.y; d[2] = f.z; d[3] = f.w;
    }
#pragma unroll
    for (int t = 0; t < 4; t++) v[u + t] = __uint_as_float(x[u + t]) * (__uint_as_float(dp[u + t]) - d[t]);
  }
  if (partial) {
#pragma unroll
    for (int u = 0; u < 32; u++) v[u] = x[u] == 0u ? 0.f : v[u];
  }
#pragma unroll
  for (int u = 0; u < 32; u += 2) w[u / 2] = r16_pack(v[u], v[u + 1]);
}

template <int DP, bool EXTRA>
__global__ void __launch_bounds__(R16_THREADS, 1)
rule16_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ CUtensorMap map_g, const __grid_constant__ R16Bwd p) {
  typedef R16BwdShape<DP> W;
  // Scores, dP; two places each of P and dS (32 columns) that the two sets of rows fill in turn; the sums.
  constexpr uint32_t COL_S = 0, COL_DP = 64, COL_P = 128, COL_DS = 192, COL_DV = 256, COL_DK = 384;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *slot_k = smem, *slot_v = smem + W::TILE, *ring_q = smem + 2 * W::TILE, *ring_g = ring_q + W::RING * W::TILE;
  uint32_t* steps = reinterpret_cast<uint32_t*>(smem + W::PLAN);
  float* ring_rows = reinterpret_cast<float*>(smem + W::ROWS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  // By the step's parity but for the first and the last line: a set of rows waits for its own steps only.
  uint64_t *bar_kv = bars, *bar_done = bars + 1, *bar_s = bars + 2, *bar_dp = bars + 4, *read_s = bars + 6, *read_dp = bars + 8, *bar_p = bars + 10, *bar_ds = bars + 12,
           *bar_dv = bars + 14, *bar_dk = bars + 16, *full_q = bars + 18, *empty_q = bars + 20, *full_g = bars + 22, *empty_g = bars + 24;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 26);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const RuleArgs& r = p.r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j0 = blockIdx.y * R16_T, bi = blockIdx.x / p.hkv, hk = blockIdx.x - bi * p.hkv, group = p.h / p.hkv;   // the longest walks of a causal mask first

  if (threadIdx.x == 0) {
    mbar_init(bar_kv, 1);
    mbar_init(bar_done, 1);
    for (int a = 0; a < 2; a++) {
      mbar_init(&bar_s[a], 1);
      mbar_init(&bar_dp[a], 1);
      mbar_init(&read_s[a], R16_ROW_WARPS / 2);
      mbar_init(&read_dp[a], R16_ROW_WARPS / 2);
      mbar_init(&bar_p[a], R16_ROW_WARPS / 2);
      mbar_init(&bar_ds[a], R16_ROW_WARPS / 2);
      mbar_init(&bar_dv[a], 1);
      mbar_init(&bar_dk[a], 1);
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
    const int n = r16_plan(steps, tiles, lane, [&](int t, int e) { return (uint32_t)rule_see<false>(*tile, (first + t) * R16_T + e * 64, 1); });
    if (lane == 0) steps[2 * R16_PLAN] = (uint32_t)n;
  }
  __syncthreads();
  // The same steps for every head that shares the keys, head by head.
  const int round = (int)steps[2 * R16_PLAN], walk = round * group;
  int gi = 0, k = -1, turn = -1;                         // the head, its step, and the number of its tile in the rings
  auto forth = [&]() {
    if (++k == round) {
      k = 0;
      gi++;
    }
    const uint32_t step = steps[k];
    if (step & R16_OPENS) turn++;
    return step;
  };

  bool ok = true;
  if (warp == R16_ROW_WARPS + 1) {
    if (lane == 0) {
      mbar_expect_tx(bar_kv, 2 * W::TILE);
      r16_load_tile<DP>(slot_k, &map_k, j0, hk, bi, bar_kv);
      r16_load_tile<DP>(slot_v, &map_v, j0, hk, bi, bar_kv);
      for (int n = 0; ok && n < walk; n++) {
        const uint32_t step = forth();
        if (!(step & R16_OPENS)) continue;
        const int a = turn % W::RING, head = hk * group + gi, at = first + r16_tile_of(step);
        const uint32_t before = ((turn / W::RING) & 1u) ^ 1u;
        // The keys' gradient of the tile before in this stage has read it, after the rows were done with its log-sum-exps and dots.
        if (turn >= W::RING) ok = r16_bar(&empty_q[a], before, abort_flag, p.status, 71);
        if (!ok) break;
        mbar_expect_tx(&full_q[a], W::TILE + 1024);
        r16_load_tile<DP>(ring_q + a * W::TILE, &map_q, at * R16_T, head, bi, &full_q[a]);
        r16_load_rows(ring_rows + a * 256, p.rows + (((long long)bi * p.h + head) * p.tiles + at) * 256, &full_q[a]);
        if (turn >= W::RING) ok = r16_bar(&empty_g[a], before, abort_flag, p.status, 72);
        if (!ok) break;
        mbar_expect_tx(&full_g[a], W::TILE);
        r16_load_tile<DP>(ring_g + a * W::TILE, &map_g, at * R16_T, head, bi, &full_g[a]);
      }
    }
  } else if (warp == R16_ROW_WARPS) {
    if (lane == 0) {
      ok = r16_bar(bar_kv, 0, abort_flag, p.status, 73);
      auto scores = [&](int n, uint32_t step, uint64_t* full, uint64_t* read, uint64_t* bar, const uint8_t* keep, const uint8_t* ring, uint32_t col) {
        const int a = turn % W::RING;
        if (step & R16_OPENS) ok = ok && r16_bar(&full[a], (turn / W::RING) & 1u, abort_flag, p.status, 74);
        if (ok && n > 0) ok = r16_bar(&read[(n - 1) & 1], ((n - 1) >> 1) & 1u, abort_flag, p.status, 75);   // the rows have taken the ones before
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP>(tmem + col, r16_desc_k(keep), r16_desc_k(ring + a * W::TILE) + r16_half_of(step) * R16_HALF_K);
        umma_commit(&bar[n & 1]);
      };
      uint32_t step = walk > 0 ? forth() : 0u;
      if (ok && walk > 0) {
        scores(0, step, full_q, read_s, bar_s, slot_k, ring_q, COL_S);
        scores(0, step, full_g, read_dp, bar_dp, slot_v, ring_g, COL_DP);
      }
      for (int n = 0; ok && n < walk; n++) {
        const int a = turn % W::RING;
        const uint32_t set = n & 1, phase = (n >> 1) & 1u, half = r16_half_of(step) * R16_HALF_MN;
        const uint32_t ahead = n + 1 < walk ? forth() : 0u;
        if (n + 1 < walk) scores(n + 1, ahead, full_q, read_s, bar_s, slot_k, ring_q, COL_S);
        // dV += P^T dO
        if (!(ok = ok && r16_bar(&bar_p[set], phase, abort_flag, p.status, 76))) break;
        tc_fence_after();
        r16_gather<DP>(tmem + COL_DV, tmem + COL_P + 32u * set, r16_desc_mn(ring_g + a * W::TILE) + half, n > 0 ? 1u : 0u);
        umma_commit(&bar_dv[set]);
        if (step & R16_CLOSES) umma_commit(&empty_g[a]);
        if (n + 1 < walk) scores(n + 1, ahead, full_g, read_dp, bar_dp, slot_v, ring_g, COL_DP);
        // dK += dS^T Q
        if (!(ok = ok && r16_bar(&bar_ds[set], phase, abort_flag, p.status, 78))) break;
        tc_fence_after();
        r16_gather<DP>(tmem + COL_DK, tmem + COL_DS + 32u * set, r16_desc_mn(ring_q + a * W::TILE) + half, n > 0 ? 1u : 0u);
        umma_commit(&bar_dk[set]);
        if (step & R16_CLOSES) umma_commit(&empty_q[a]);
        step = ahead;
      }
      if (ok) umma_commit(bar_done);
      else *abort_flag = 1;
    }
  } else {
    const int set = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3, row = quad * 32 + lane, j = j0 + row;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_s = lane_base + COL_S + 32u * half, t_dp = lane_base + COL_DP + 32u * half, t_p = lane_base + COL_P + 32u * set + 16u * half,
                   t_ds = lane_base + COL_DS + 32u * set + 16u * half;
    const R16Row seen = r16_key_row(r, prefix, bi, min(j, r.lk - 1));
    const int32_t* docs = r.q_docs ? r.q_docs + (long long)bi * r.lq : nullptr;
    const float mult = EXTRA ? 1.f : r.scale * R16_LOG2E;
    for (int n = 0; ok && n < walk; n++) {
      const uint32_t step = forth();
      if ((n & 1) != set) continue;
      const int a = turn % W::RING, in = (int)r16_half_of(step) * 64 + half * 32, at = (first + r16_tile_of(step)) * R16_T + in;
      const uint32_t phase = (n >> 1) & 1u;
      const bool partial = r16_sees_of(step, 0) == 1;
      const float slope = EXTRA && r.slopes ? r.slopes[hk * group + gi] : 0.f;
      const float* rows = ring_rows + a * 256 + in;
      // The queries' log-sum-exps came with the queries, which the scores have waited for; this wait makes them seen here.
      if (!(ok = r16_wait(&full_q[a], (turn / W::RING) & 1u, abort_flag, p.status, 94) && r16_wait(&bar_s[set], phase, abort_flag, p.status, 80))) break;
      tc_fence_after();
      uint32_t x[32], w[16];
      tmem_ld_32x32b_x32(t_s, x);
      tmem_ld_wait();
      r16_arrive_warp(&read_s[set], lane);
      r16_weights<EXTRA, true>(r, x, w, rows, 0.f, slope, at + r.q_offset - j, mult, partial, seen, at, docs);
      // The products of this set's step before have read the places of P and dS.
      if (n >= 2 && !(ok = r16_wait(&bar_dv[set], phase ^ 1u, abort_flag, p.status, 95))) break;
      tc_fence_after();
      r16_st16(t_p, w);
      r16_st_wait();
      r16_arrive_warp(&bar_p[set], lane);
      if (!(ok = r16_wait(&bar_dp[set], phase, abort_flag, p.status, 81))) break;
      tc_fence_after();
      uint32_t dp[32];
      tmem_ld_32x32b_x32(t_dp, dp);
      tmem_ld_wait();
      r16_arrive_warp(&read_dp[set], lane);
      r16_gradients<true>(x, dp, w, rows + 128, 0.f, partial);
      if (n >= 2 && !(ok = r16_wait(&bar_dk[set], phase ^ 1u, abort_flag, p.status, 96))) break;
      tc_fence_after();
      r16_st16(t_ds, w);
      r16_st_wait();
      r16_arrive_warp(&bar_ds[set], lane);
    }
    if (ok) ok = r16_wait(bar_done, 0, abort_flag, p.status, 82);
    if (ok) {
      tc_fence_after();
      // dV by the first set, dK by the other, half of the columns each.
      float* out = set == 0 ? p.d0 : p.d1;
      __nv_bfloat16* out16 = set == 0 ? p.d0_16 : p.d1_16;
      const R16Strides& s = set == 0 ? p.s0 : p.s1;
      if (out || out16) {
#pragma unroll 1
        for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
          uint32_t o[32];
          __syncwarp();
          if (walk > 0) {
            tmem_ld_32x32b_x32(lane_base + (set == 0 ? COL_DV : COL_DK) + (uint32_t)c, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int u = 0; u < 32; u++) o[u] = 0u;
          }
          if (j < r.lk) r16_write(o, set == 0 ? 1.f : r.scale, out, out16, bi * s.batch + hk * s.head + (long long)j * s.row + c, c, p.d);
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

template <int DP, bool EXTRA>
__global__ void __launch_bounds__(R16_THREADS, 1)
rule16_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_g, const __grid_constant__ R16Bwd p) {
  typedef R16BwdShape<DP> W;
  // Two places each of scores, dP (64 columns) and dS (32): the two sets of rows take the steps in turn.
  constexpr uint32_t COL_S = 0, COL_DP = 128, COL_DS = 256, COL_DQ = 384;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *slot_q = smem, *slot_g = smem + W::TILE, *ring_k = smem + 2 * W::TILE, *ring_v = ring_k + W::RING * W::TILE;
  uint32_t* steps = reinterpret_cast<uint32_t*>(smem + W::PLAN);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  uint64_t *bar_qg = bars, *bar_done = bars + 1, *bar_s = bars + 2, *bar_dp = bars + 4, *read_s = bars + 6, *read_dp = bars + 8, *bar_ds = bars + 10, *bar_dq = bars + 12,
           *full_k = bars + 14, *empty_k = bars + 16, *full_v = bars + 18, *empty_v = bars + 20;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const RuleArgs& r = p.r;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * R16_T, bi = blockIdx.x / p.h, hi = blockIdx.x - bi * p.h, hk = hi / (p.h / p.hkv);

  if (threadIdx.x == 0) {
    mbar_init(bar_qg, 1);
    mbar_init(bar_done, 1);
    for (int a = 0; a < 2; a++) {
      mbar_init(&bar_s[a], 1);
      mbar_init(&bar_dp[a], 1);
      mbar_init(&read_s[a], R16_ROW_WARPS / 2);
      mbar_init(&read_dp[a], R16_ROW_WARPS / 2);
      mbar_init(&bar_ds[a], R16_ROW_WARPS / 2);
      mbar_init(&bar_dq[a], 1);
      mbar_init(&full_v[a], 1);
      mbar_init(&empty_v[a], 1);
      mbar_init(&full_k[a], 1);
      mbar_init(&empty_k[a], 1);
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
    const int n = r16_plan(steps, tiles, lane, [&](int t, int e) { return (uint32_t)rule_see<true>(*tile, (first + t) * R16_T + e * 64, 1); });
    if (lane == 0) steps[2 * R16_PLAN] = (uint32_t)n;
  }
  __syncthreads();
  const int walk = (int)steps[2 * R16_PLAN];
  int turn = -1;                                         // the number of a step's tile in the rings

  bool ok = true;
  if (warp == R16_ROW_WARPS + 1) {
    if (lane == 0) {
      mbar_expect_tx(bar_qg, 2 * W::TILE);
      r16_load_tile<DP>(slot_q, &map_q, i0, hi, bi, bar_qg);
      r16_load_tile<DP>(slot_g, &map_g, i0, hi, bi, bar_qg);
      for (int n = 0; ok && n < walk; n++) {
        const uint32_t step = steps[n];
        if (!(step & R16_OPENS)) continue;
        const int a = ++turn % W::RING, at = (first + r16_tile_of(step)) * R16_T;
        const uint32_t before = ((turn / W::RING) & 1u) ^ 1u;
        if (turn >= W::RING) ok = r16_bar(&empty_k[a], before, abort_flag, p.status, 83);
        if (!ok) break;
        mbar_expect_tx(&full_k[a], W::TILE);
        r16_load_tile<DP>(ring_k + a * W::TILE, &map_k, at, hk, bi, &full_k[a]);
        if (turn >= W::RING) ok = r16_bar(&empty_v[a], before, abort_flag, p.status, 84);
        if (!ok) break;
        mbar_expect_tx(&full_v[a], W::TILE);
        r16_load_tile<DP>(ring_v + a * W::TILE, &map_v, at, hk, bi, &full_v[a]);
      }
    }
  } else if (warp == R16_ROW_WARPS) {
    if (lane == 0) {
      ok = r16_bar(bar_qg, 0, abort_flag, p.status, 85);
      // Scores and dP of a step, into the places that this set's step before has been taken from.
      auto scores = [&](int n, uint32_t step) {
        if (step & R16_OPENS) turn++;
        const int a = turn % W::RING;
        const uint32_t phase = (turn / W::RING) & 1u, set = n & 1, before = ((n >> 1) & 1u) ^ 1u, half = r16_half_of(step) * R16_HALF_K;
        if (step & R16_OPENS) ok = r16_bar(&full_k[a], phase, abort_flag, p.status, 86);
        if (ok && n >= 2) ok = r16_bar(&read_s[set], before, abort_flag, p.status, 87);
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP>(tmem + COL_S + 64u * set, r16_desc_k(slot_q), r16_desc_k(ring_k + a * W::TILE) + half);
        umma_commit(&bar_s[set]);
        if (step & R16_OPENS) ok = r16_bar(&full_v[a], phase, abort_flag, p.status, 88);
        if (ok && n >= 2) ok = r16_bar(&read_dp[set], before, abort_flag, p.status, 89);
        if (!ok) return;
        tc_fence_after();
        r16_scores<DP>(tmem + COL_DP + 64u * set, r16_desc_k(slot_g), r16_desc_k(ring_v + a * W::TILE) + half);
        umma_commit(&bar_dp[set]);
        if (step & R16_CLOSES) umma_commit(&empty_v[a]);
      };
      uint32_t step = walk > 0 ? steps[0] : 0u;
      if (ok && walk > 0) scores(0, step);
      for (int n = 0; ok && n < walk; n++) {
        const int a = turn % W::RING;
        const uint32_t set = n & 1, ahead = n + 1 < walk ? steps[n + 1] : 0u;
        if (n + 1 < walk) scores(n + 1, ahead);
        if (!(ok = ok && r16_bar(&bar_ds[set], (n >> 1) & 1u, abort_flag, p.status, 90))) break;
        tc_fence_after();
        r16_gather<DP>(tmem + COL_DQ, tmem + COL_DS + 32u * set, r16_desc_mn(ring_k + a * W::TILE) + r16_half_of(step) * R16_HALF_MN, n > 0 ? 1u : 0u);
        umma_commit(&bar_dq[set]);
        if (step & R16_CLOSES) umma_commit(&empty_k[a]);
        step = ahead;
      }
      if (ok) umma_commit(bar_done);
      else *abort_flag = 1;
    }
  } else {
    const int set = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3, row = quad * 32 + lane, i = i0 + row;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_s = lane_base + COL_S + 64u * set + 32u * half, t_dp = lane_base + COL_DP + 64u * set + 32u * half, t_ds = lane_base + COL_DS + 32u * set + 16u * half;
    const float slope = EXTRA && r.slopes ? r.slopes[hi] : 0.f;
    const R16Row seen = r16_query_row(r, prefix, bi, min(i, r.lq - 1));
    const int32_t* docs = r.k_docs ? r.k_docs + (long long)bi * r.lk : nullptr;
    const float mult = EXTRA ? 1.f : r.scale * R16_LOG2E;
    const float2 stat = rule_row(p.rows, (long long)bi * p.h + hi, r.lq, i);
    for (int n = set; ok && n < walk; n += 2) {
      const uint32_t step = steps[n];
      const int at = (first + r16_tile_of(step)) * R16_T + (int)r16_half_of(step) * 64 + half * 32;
      const uint32_t phase = (n >> 1) & 1u;
      const bool partial = r16_sees_of(step, 0) == 1;
      if (!(ok = r16_wait(&bar_s[set], phase, abort_flag, p.status, 91))) break;
      tc_fence_after();
      uint32_t x[32], dp[32], w[16];
      tmem_ld_32x32b_x32(t_s, x);
      tmem_ld_wait();
      r16_arrive_warp(&read_s[set], lane);
      r16_weights<EXTRA, false>(r, x, w, nullptr, stat.x, slope, i + r.q_offset - at, mult, partial, seen, at, docs);
      if (!(ok = r16_wait(&bar_dp[set], phase, abort_flag, p.status, 92))) break;
      tc_fence_after();
      tmem_ld_32x32b_x32(t_dp, dp);
      tmem_ld_wait();
      r16_arrive_warp(&read_dp[set], lane);
      r16_gradients<false>(x, dp, w, nullptr, stat.y, partial);
      if (n >= 2 && !(ok = r16_wait(&bar_dq[set], phase ^ 1u, abort_flag, p.status, 97))) break;    // the product has read the gradients before
      tc_fence_after();
      r16_st16(t_ds, w);
      r16_st_wait();
      r16_arrive_warp(&bar_ds[set], lane);
    }
    if (ok) ok = r16_wait(bar_done, 0, abort_flag, p.status, 93);
    if (ok) {
      tc_fence_after();
      // A quarter of dQ's columns by each four warps.
#pragma unroll 1
      for (int c = (set * 2 + half) * 32; c < DP; c += 128) {
        uint32_t o[32];
        __syncwarp();
        if (walk > 0) {
          tmem_ld_32x32b_x32(lane_base + COL_DQ + (uint32_t)c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int u = 0; u < 32; u++) o[u] = 0u;
        }
        if (i < r.lq) r16_write(o, r.scale, p.d0, p.d0_16, bi * p.s0.batch + hi * p.s0.head + (long long)i * p.s0.row + c, c, p.d);
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

template <int DP, bool EXTRA>
static int32_t r16_fwd(om_ctx* ctx, dim3 grid, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const R16Fwd& p) {
  OM_TRY(r16_room(ctx, rule16_fwd_kernel<DP, EXTRA>, R16FwdShape<DP>::SMEM));
  launch_chained(ctx, rule16_fwd_kernel<DP, EXTRA>, grid, R16_THREADS, R16FwdShape<DP>::SMEM, mq, mk, mv, p);
  return OM_OK;
}

int32_t rule16_fwd(om_ctx* ctx, const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                   const om_head_strides* vs, float* out, void* out16, const om_head_strides* os, float* lse) {
  const int group = c.h / c.hkv, lq = c.r.lq, lk = c.r.lk;
  R16Fwd p = {};
  p.r = c.r; p.h = c.h; p.hkv = c.hkv; p.d = c.d;
  p.out = out; p.out16 = reinterpret_cast<__nv_bfloat16*>(out16); p.os = r16_strides(os); p.lse = lse;
  p.rows = (long long)c.b * c.h * lq;
  p.status = ctx->status_dev;
  // Heads that share keys as rows of one tile where they fit it: keys and values are read once for all of them.
  p.packed = (long long)group * lq <= R16_T && (group > 1);
  dim3 grid((unsigned)(c.b * (p.packed ? c.hkv : c.h)), p.packed ? 1u : (unsigned)ceil_div(lq, 2 * R16_T), 1);
  // A walk is split where the CTAs leave SMs without one, four tiles of keys a part at least: a part costs its CTA's start and a
  // row of O per query in memory, twice.
  const int64_t ctas = (int64_t)grid.x * grid.y;
  const int64_t span = c.r.window && !c.r.prefix ? std::min<int64_t>(lk, 2ll * c.r.window + lq) : lk;
  const int64_t tiles = ceil_div(span, R16_T);
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(ctx->sm_count / std::max<int64_t>(ctas, 1), tiles / 4));
  p.splits = (int)std::max<int64_t>(p.splits, ceil_div(ceil_div(lk, R16_T) + 1, R16_PLAN));   // a part is at most a plan long
  grid.z = (unsigned)p.splits;
  CUtensorMap mq, mk, mv;
  if (!r16_map(&mq, q, c.d, lq, c.h, c.b, qs, p.packed ? lq : R16_T, p.packed ? group : 1) || !r16_map(&mk, k, c.d, lk, c.hkv, c.b, ks, R16_T, 1) ||
      !r16_map(&mv, v, c.d, lk, c.hkv, c.b, vs, R16_T, 1))
    return fail(ctx, OM_ERR_CUDA, "cuTensorMapEncodeTiled failed for the operands of om_rule_attention_fwd_bf16");
  char* part = nullptr;
  if (p.splits > 1) {
    const size_t ml = ((size_t)p.splits * p.rows * sizeof(float2) + 255) & ~(size_t)255;
    OM_TRY(pool_alloc(ctx, ml + (size_t)p.splits * p.rows * c.d * sizeof(float), false, (void**)&part));
    p.part_ml = reinterpret_cast<float2*>(part);
    p.part = reinterpret_cast<float*>(part + ml);
  }
  const bool extra = c.r.softcap > 0.f || c.r.slopes;
  int32_t st;
  if (c.d <= 64) st = extra ? r16_fwd<64, true>(ctx, grid, mq, mk, mv, p) : r16_fwd<64, false>(ctx, grid, mq, mk, mv, p);
  else st = extra ? r16_fwd<128, true>(ctx, grid, mq, mk, mv, p) : r16_fwd<128, false>(ctx, grid, mq, mk, mv, p);
  if (p.splits > 1) {
    if (st == OM_OK) launch_chained(ctx, rule16_join_kernel, grid_for(ctx, p.rows, 8), 256, 0, p);
    pool_free(ctx, part);
  }
  OM_TRY(st);
  OM_LAUNCH_CHECK(ctx, "om_rule_attention_fwd_bf16");
  return OM_OK;
}

template <int DP, bool EXTRA>
static int32_t r16_bwd(om_ctx* ctx, const RuleCall& c, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mg,
                       const R16Bwd& kv, const R16Bwd& q) {
  const int smem = R16BwdShape<DP>::SMEM;
  if (kv.d0 || kv.d0_16 || kv.d1 || kv.d1_16) {
    OM_TRY(r16_room(ctx, rule16_dkv_kernel<DP, EXTRA>, smem));
    launch_chained(ctx, rule16_dkv_kernel<DP, EXTRA>, dim3((unsigned)(c.b * c.hkv), (unsigned)ceil_div(c.r.lk, R16_T)), R16_THREADS, smem, mq, mk, mv, mg, kv);
  }
  if (q.d0 || q.d0_16) {
    OM_TRY(r16_room(ctx, rule16_dq_kernel<DP, EXTRA>, smem));
    launch_chained(ctx, rule16_dq_kernel<DP, EXTRA>, dim3((unsigned)(c.b * c.h), (unsigned)ceil_div(c.r.lq, R16_T)), R16_THREADS, smem, mq, mk, mv, mg, q);
  }
  return OM_OK;
}

int32_t rule16_bwd(om_ctx* ctx, const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                   const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* rows, float* dq, void* dq16,
                   const om_head_strides* dqs, float* dk, void* dk16, const om_head_strides* dks, float* dv, void* dv16, const om_head_strides* dvs) {
  const int lq = c.r.lq, lk = c.r.lk;
  CUtensorMap mq, mk, mv, mg;
  if (!r16_map(&mq, q, c.d, lq, c.h, c.b, qs, R16_T, 1) || !r16_map(&mk, k, c.d, lk, c.hkv, c.b, ks, R16_T, 1) ||
      !r16_map(&mv, v, c.d, lk, c.hkv, c.b, vs, R16_T, 1) || !r16_map(&mg, g, c.d, lq, c.h, c.b, gs, R16_T, 1))
    return fail(ctx, OM_ERR_CUDA, "cuTensorMapEncodeTiled failed for the operands of om_rule_attention_bwd_bf16");
  R16Bwd kv = {};
  kv.r = c.r; kv.h = c.h; kv.hkv = c.hkv; kv.d = c.d; kv.rows = rows; kv.tiles = rule_row_tiles(lq); kv.status = ctx->status_dev;
  R16Bwd one = kv;
  kv.d0 = dv; kv.d1 = dk; kv.d0_16 = reinterpret_cast<__nv_bfloat16*>(dv16); kv.d1_16 = reinterpret_cast<__nv_bfloat16*>(dk16);
  if (dv || dv16) kv.s0 = r16_strides(dvs);
  if (dk || dk16) kv.s1 = r16_strides(dks);
  one.d0 = dq; one.d0_16 = reinterpret_cast<__nv_bfloat16*>(dq16);
  if (dq || dq16) one.s0 = r16_strides(dqs);
  const bool extra = c.r.softcap > 0.f || c.r.slopes;
  int32_t st;
  if (c.d <= 64) st = extra ? r16_bwd<64, true>(ctx, c, mq, mk, mv, mg, kv, one) : r16_bwd<64, false>(ctx, c, mq, mk, mv, mg, kv, one);
  else st = extra ? r16_bwd<128, true>(ctx, c, mq, mk, mv, mg, kv, one) : r16_bwd<128, false>(ctx, c, mq, mk, mv, mg, kv, one);
  OM_TRY(st);
  OM_LAUNCH_CHECK(ctx, "om_rule_attention_bwd_bf16");
  return OM_OK;
}

}  // namespace om
