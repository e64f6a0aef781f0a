// The mask rule of om_rule_attention_*: which keys a query sees, which tiles of keys (or of queries) a tile has to visit, and
// which tiles are visible as a whole. Shared by the fp32 and the bfloat16 kernels.
#pragma once
#include "om_common.cuh"

namespace om {

constexpr int RULE_GRAIN = 64;   // rows per entry of the document ranges: every tile is a whole number of these

struct RuleArgs {
  int causal, window, q_offset;
  float softcap, inv_softcap, scale;
  const float* slopes;
  const int32_t* prefix;
  const int32_t *q_docs, *k_docs;
  const int4 *q_ranges, *k_ranges;   // [b][ceil(l / 64)]: lowest and highest document (padding left out), the document if it is one only else -1
  int lq, lk, nq64, nk64;
};

// The keys that queries [i0, i1) of a sequence may see by position: [0, prefix) and [lo, hi).
struct RuleSpan {
  int prefix, lo, hi;
};
__device__ __forceinline__ RuleSpan rule_keys(const RuleArgs& r, int prefix, int i0, int i1) {
  RuleSpan s;
  s.prefix = min(max(prefix, 0), r.lk);
  const long long p0 = (long long)i0 + r.q_offset, p1 = (long long)i1 - 1 + r.q_offset;
  long long lo = 0, hi = r.lk;
  if (r.causal) hi = min(hi, p1 + 1);
  if (r.window) {
    lo = max(lo, p0 - r.window + 1);
    hi = min(hi, p1 + r.window);
  }
  s.lo = (int)min(lo, (long long)r.lk);
  s.hi = (int)max(hi, 0ll);
  return s;
}
// The queries that may see keys [j0, j1): [lo, hi), all of them where the prefix reaches into the keys.
__device__ __forceinline__ void rule_queries(const RuleArgs& r, int prefix, int j0, int j1, int* lo, int* hi) {
  long long a = 0, b = r.lq;
  if (j0 >= prefix) {
    if (r.causal) a = max(a, (long long)j0 - r.q_offset);
    if (r.window) {
      a = max(a, (long long)j0 - r.window + 1 - r.q_offset);
      b = min(b, (long long)j1 - 1 + r.window - r.q_offset);
    }
  }
  *lo = (int)min(a, (long long)r.lq);
  *hi = (int)max(b, 0ll);
}
// Documents of queries [i0, i0 + 64 nq) and keys [j0, j0 + 64 nk): 0 none in common, 1 perhaps some, 2 one and the same throughout.
__device__ __forceinline__ int rule_documents(const RuleArgs& r, int b, int i0, int nq, int j0, int nk) {
  if (!r.q_docs) return 2;
  int qlo = INT32_MAX, qhi = -1, klo = INT32_MAX, khi = -1, one = -2;
  bool whole = true;
  for (int t = i0 / RULE_GRAIN; t < min(i0 / RULE_GRAIN + nq, r.nq64); t++) {
    const int4 v = r.q_ranges[(long long)b * r.nq64 + t];
    qlo = min(qlo, v.x);
    qhi = max(qhi, v.y);
    if (one == -2) one = v.z;
    whole = whole && v.z >= 0 && v.z == one;
  }
  for (int t = j0 / RULE_GRAIN; t < min(j0 / RULE_GRAIN + nk, r.nk64); t++) {
    const int4 v = r.k_ranges[(long long)b * r.nk64 + t];
    klo = min(klo, v.x);
    khi = max(khi, v.y);
    whole = whole && v.z == one;
  }
  if (qhi < 0 || khi < 0 || qlo > khi || klo > qhi) return 0;
  return whole ? 2 : 1;
}
// 0: nothing of the tile is visible; 1: some may be; 2: every query of the sequence in it sees all of its keys, none of them beyond
// the last.
__device__ __forceinline__ int rule_tile(const RuleArgs& r, int prefix, int b, int i0, int nq, int j0, int nk) {
  const int i1 = min(i0 + nq * RULE_GRAIN, r.lq), j1 = min(j0 + nk * RULE_GRAIN, r.lk);
  if (i0 >= i1 || j0 >= j1) return 0;
  const RuleSpan s = rule_keys(r, prefix, i0, i1);
  if (!(j0 < s.prefix || (j0 < s.hi && j1 > s.lo))) return 0;
  const int docs = rule_documents(r, b, i0, nq, j0, nk);
  if (docs != 2) return docs;
  if (j1 - j0 != nk * RULE_GRAIN) return 1;
  if (j1 <= s.prefix) return 2;
  const long long p0 = (long long)i0 + r.q_offset, p1 = (long long)i1 - 1 + r.q_offset;
  if (r.causal && j1 - 1 > p0) return 1;
  if (r.window && (p1 - j0 >= r.window || j1 - 1 - p0 >= r.window)) return 1;
  return 2;
}
// One pair, both inside the matrix; doc: the query's document (any value where there are none).
__device__ __forceinline__ bool rule_visible(const RuleArgs& r, int prefix, int i, int j, int q_doc, int k_doc) {
  const int far = i + r.q_offset - j;   // lengths and offset are below 2^30: no overflow
  const bool near = (!r.causal || far >= 0) && (!r.window || abs(far) < r.window);
  return (near || j < prefix) && (!r.q_docs || (q_doc == k_doc && q_doc >= 0));
}
// The score of a visible pair from the plain product, and the derivative of the cap.
__device__ __forceinline__ float rule_score(const RuleArgs& r, float slope, int i, int j, float dot, float* dcap) {
  float s = dot * r.scale;
  *dcap = 1.f;
  if (r.softcap > 0.f) {
    const float t = tanhf(s / r.softcap);
    *dcap = fmaf(-t, t, 1.f);
    s = r.softcap * t;
  }
  if (r.slopes) s = fmaf(-slope, (float)abs(i + r.q_offset - j), s);
  return s;
}

// What both precisions do around their kernels (om_rule_attention.cu).
struct RuleCall {
  RuleArgs r;
  int b, h, hkv, d;
  int4* ranges;   // pooled; freed by rule_end
};
int32_t rule_check(om_ctx* ctx, const char* who, const om_attention_rule* rule, int b, int h, int hkv, int lq, int lk, int d, float scale);
int32_t rule_operand(om_ctx* ctx, const char* who, const void* p, const om_head_strides* s, int d);
int32_t rule_result(om_ctx* ctx, const char* who, const om_head_strides* s, int b, int h, int l, int d);
// What the backward kernels read of the queries: per (batch, head) and 128 queries, the log-sum-exps times a unit and behind them the
// row dots rowsum(dO o O), 256 floats.
__host__ __device__ constexpr int rule_row_tiles(int lq) { return (lq + 127) / 128; }
__device__ __forceinline__ float2 rule_row(const float* rows, long long bh, int lq, int i) {
  const float* t = rows + (bh * rule_row_tiles(lq) + i / 128) * 256 + i % 128;
  return make_float2(t[0], t[128]);
}
int32_t rule_begin(om_ctx* ctx, const om_attention_rule* rule, int b, int h, int hkv, int lq, int lk, int d, float scale, RuleCall* call);
void rule_end(om_ctx* ctx, RuleCall* call);
// The tensor-pipe kernels for bfloat16 operands (om_rule_attention16.cu): whether they take a call, and the call. Pointers to
// operands and bfloat16 results are to 2-byte elements; `rows` as above with log2 e for the unit.
bool rule16_fwd_takes(const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                      const om_head_strides* vs, const float* out, const void* out16, const om_head_strides* os);
int32_t rule16_fwd(om_ctx* ctx, const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                   const om_head_strides* vs, float* out, void* out16, const om_head_strides* os, float* lse);
bool rule16_bwd_takes(const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                      const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* dq, const void* dq16, const om_head_strides* dqs,
                      const float* dk, const void* dk16, const om_head_strides* dks, const float* dv, const void* dv16, const om_head_strides* dvs);
int32_t rule16_bwd(om_ctx* ctx, const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                   const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* rows, float* dq, void* dq16,
                   const om_head_strides* dqs, float* dk, void* dk16, const om_head_strides* dks, float* dv, void* dv16, const om_head_strides* dvs);

}  // namespace om
