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
  const int4 *q_ranges, *k_ranges;   // [b][ceil(l / 64)]: lowest and highest document (padding left out), the document if it is one only else -1, padding
  const uint2 *q_pads, *k_pads;      // [b][ceil(l / 64)]: a bit for each row that is padding
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
// What a fixed tile of queries (or of keys) sees of the other axis, as whole numbers that a walk over that axis compares with: the
// indices below `pre` and those in [lo, hi) are seen by some of its rows, those below `all_pre` and those in [all_lo, all_hi) by all.
struct RuleTile {
  int pre, lo, hi, all_pre, all_lo, all_hi, end;
  int doc_lo, doc_hi, doc;               // documents of its rows; `doc` where they are one and the same, else -1
  const int4* other;                     // the other axis's documents, per 64 indices (null: no documents)
  int n64;
};
__device__ __forceinline__ int rule_clamp(long long v, int end) { return (int)max(0ll, min(v, (long long)end)); }
__device__ __forceinline__ void rule_tile_documents(RuleTile& t, const int4* mine, int m64, int first, int n, const int4* other, int n64) {
  t.other = other;
  t.n64 = n64;
  t.doc_lo = INT32_MAX;
  t.doc_hi = t.doc = -1;
  if (!other) return;
  for (int e = first / RULE_GRAIN; e < min(first / RULE_GRAIN + n, m64); e++) {
    const int4 v = mine[e];
    t.doc_lo = min(t.doc_lo, v.x);
    t.doc_hi = max(t.doc_hi, v.y);
    t.doc = e == first / RULE_GRAIN || v.z == t.doc ? v.z : -1;
  }
}
// Queries [i0, i0 + 64 n).
__device__ __forceinline__ RuleTile rule_query_tile(const RuleArgs& r, int prefix, int b, int i0, int n) {
  RuleTile t;
  const int i1 = min(i0 + n * RULE_GRAIN, r.lq);
  const RuleSpan s = rule_keys(r, prefix, i0, i1);
  t.end = r.lk;
  t.pre = t.all_pre = s.prefix;
  t.lo = s.lo;
  t.hi = i0 < i1 ? s.hi : 0;
  const long long p0 = (long long)i0 + r.q_offset, p1 = (long long)i1 - 1 + r.q_offset;
  long long lo = 0, hi = r.lk;
  if (r.causal) hi = min(hi, p0 + 1);
  if (r.window) {
    lo = max(lo, p1 - r.window + 1);
    hi = min(hi, p0 + r.window);
  }
  t.all_lo = rule_clamp(lo, r.lk);
  t.all_hi = rule_clamp(hi, r.lk);
  if (i0 >= i1) t.pre = 0;
  rule_tile_documents(t, r.q_docs ? r.q_ranges + (long long)b * r.nq64 : nullptr, r.nq64, i0, n, r.q_docs ? r.k_ranges + (long long)b * r.nk64 : nullptr, r.nk64);
  return t;
}
// Keys [j0, j0 + 64 n).
__device__ __forceinline__ RuleTile rule_key_tile(const RuleArgs& r, int prefix, int b, int j0, int n) {
  RuleTile t;
  const int j1 = min(j0 + n * RULE_GRAIN, r.lk);
  t.end = r.lq;
  t.pre = t.all_pre = 0;
  rule_queries(r, prefix, j0, j1, &t.lo, &t.hi);
  long long lo = 0, hi = r.lq;
  if (j1 > prefix) {
    if (r.causal) lo = max(lo, (long long)j1 - 1 - r.q_offset);
    if (r.window) {
      lo = max(lo, (long long)j1 - r.window - r.q_offset);
      hi = min(hi, (long long)j0 + r.window - r.q_offset);
    }
  }
  t.all_lo = rule_clamp(lo, r.lq);
  t.all_hi = rule_clamp(hi, r.lq);
  rule_tile_documents(t, r.q_docs ? r.k_ranges + (long long)b * r.nk64 : nullptr, r.nk64, j0, n, r.q_docs ? r.q_ranges + (long long)b * r.nq64 : nullptr, r.nq64);
  return t;
}
// What the tile sees of indices [at, at + 64 n): 0 nothing, 1 perhaps some, 2 all of its rows see all of those in range (FULL: and
// all of them are in range).
template <bool FULL>
__device__ __forceinline__ int rule_see(const RuleTile& t, int at, int n) {
  const int to = min(at + n * RULE_GRAIN, t.end);
  if (at >= to || !(at < t.pre || (at < t.hi && to > t.lo))) return 0;
  const bool all = (to <= t.all_pre || (at >= t.all_lo && to <= t.all_hi)) && (!FULL || to == at + n * RULE_GRAIN);
  if (!t.other) return all ? 2 : 1;
  int lo = INT32_MAX, hi = -1;
  bool same = t.doc >= 0;
  for (int e = at / RULE_GRAIN; e < min(at / RULE_GRAIN + n, t.n64); e++) {
    const int4 v = t.other[e];
    lo = min(lo, v.x);
    hi = max(hi, v.y);
    same = same && v.z == t.doc;
  }
  if (hi < 0 || t.doc_hi < 0 || lo > t.doc_hi || hi < t.doc_lo) return 0;
  return all && same ? 2 : 1;
}
// Whether any of indices [at, at + 64 n) is padding.
__device__ __forceinline__ bool rule_padding(const RuleTile& t, int at, int n) {
  int pad = 0;
  if (t.other)
    for (int e = at / RULE_GRAIN; e < min(at / RULE_GRAIN + n, t.n64); e++) pad |= t.other[e].w;
  return pad != 0;
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
struct RulePlanes {
  const void* p[4];               // q, k, v, g
  om_head_strides q, k;           // of q and g, of k and v
  const float* units;
  const int32_t* plain;           // [b * hkv]
  void *small, *large;
};
// The tensor-pipe kernels for bfloat16 operands (om_rule_attention16.cu): whether they take a call, and the call. Pointers to
// operands and bfloat16 results are to 2-byte elements; `rows` as above with log2 e for the unit.
bool rule16_fwd_takes(const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                      const om_head_strides* vs, const float* out, const void* out16, const om_head_strides* os);
int32_t rule16_fwd(om_ctx* ctx, const RuleCall& c, const void* q, const om_head_strides* qs, const void* k, const om_head_strides* ks, const void* v,
                   const om_head_strides* vs, float* out, void* out16, const om_head_strides* os, float* lse, const RulePlanes* planes);
bool rule16_bwd_takes(const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                      const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* dq, const void* dq16, const om_head_strides* dqs,
                      const float* dk, const void* dk16, const om_head_strides* dks, const float* dv, const void* dv16, const om_head_strides* dvs);
int32_t rule16_bwd(om_ctx* ctx, const RuleCall& c, const void* g, const om_head_strides* gs, const void* q, const om_head_strides* qs, const void* k,
                   const om_head_strides* ks, const void* v, const om_head_strides* vs, const float* rows, float* dq, void* dq16,
                   const om_head_strides* dqs, float* dk, void* dk16, const om_head_strides* dks, float* dv, void* dv16, const om_head_strides* dvs,
                   const RulePlanes* planes);
// fp32 operands as two planes of halves for the same kernels: whether a call is taken, the planes (freed by rule16_planes_end once
// what reads them is queued), and whether a result can be written. Where the flag of a head of k and v gets set in `plain` on the device,
// the kernels leave the heads that share it to the fp32 ones, which have to be queued behind them with the flags.
bool rule16_planes_take(const RuleCall& c, bool backward);
bool rule16_result_fits(const float* p, const om_head_strides* s);
int32_t rule16_planes(om_ctx* ctx, const RuleCall& c, const float* q, const om_head_strides* qs, const float* k, const om_head_strides* ks, const float* v,
                      const om_head_strides* vs, const float* g, const om_head_strides* gs, RulePlanes* out);
void rule16_planes_end(om_ctx* ctx, RulePlanes* planes);

}  // namespace om
