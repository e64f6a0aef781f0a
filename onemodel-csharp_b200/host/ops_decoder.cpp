// The operators a decoder needs beside the reference's: rotary positions and attention by rule, forward and backward.
// Each takes activations as [B, H, L, D] or, in its *Heads form, still packed as [B, L, H * D], and addresses strided views
// (a slice of a packed projection) in place.
#include <math.h>

#include "omh.hpp"

namespace omh {

static om_ctx* C() { return Device::Current(); }

static Tensor NewOut(const Shape& s) {
  Tensor r = Tensor::Create(DType::F32, s);
  ActivationScope::Track(r);
  return r;
}

// A [B, H, L, D] or [B, L, W] activation with its columns adjacent, its rows apart and no negative stride, as it is or cloned.
static Tensor InPlace(const Tensor& t) {
  const int rank = t.Rank();
  const auto& st = t.Strides();
  if (t.Length() == 0) return t.Contiguous();
  if (st[rank - 1] != 1 && t.GetShape()[rank - 1] != 1) return t.Contiguous();
  for (int i = 0; i < rank; i++)
    if (st[i] < 0) return t.Contiguous();
  return st[rank - 2] >= t.GetShape()[rank - 1] ? t : t.Contiguous();
}
// heads == 0: [B, H, L, D]; else [B, L, heads * d].
static om_head_strides StridesOf(const Tensor& t, int heads) {
  const auto& st = t.Strides();
  if (heads == 0) return om_head_strides{st[0], st[1], st[2]};
  return om_head_strides{st[0], (int64_t)(t.GetShape()[2] / heads), st[1]};
}
static void RequireFloat32(const Tensor& t) {
  if (t.IsEmpty() || t.GetDType() != DType::F32) throw TensorShapeException("A float32 tensor is required.");
}
static void RequireInt32(const Tensor& t, const char* what) {
  if (!t.IsEmpty() && t.GetDType() != DType::I32) throw TensorShapeException(std::string(what) + " must be an int32 tensor.");
}
// All three strides on the grid that the bfloat16 kernels address (those of axes with one entry do not matter).
static bool Bf16InPlace(const Tensor& t) {
  for (int i = 0; i + 1 < t.Rank(); i++)
    if (t.GetShape()[i] > 1 && t.Strides()[i] % 8 != 0) return false;
  return Bf16Operand(t, 0);
}

// ---- rotary positions -------------------------------------------------------------------------------------------------------

static void Turn(const Tensor& x, const Tensor& positions, const RotarySpec& spec, int heads, bool inverse, const Tensor& y) {
  const int b = x.GetShape()[0];
  const int h = heads ? heads : x.GetShape()[1], l = heads ? x.GetShape()[1] : x.GetShape()[2];
  const int d = heads ? x.GetShape()[2] / heads : x.GetShape()[3];
  double f[128];
  om_rotary_spec s{spec.columns ? spec.columns : d, spec.scaling, spec.base, spec.factor, spec.originalContext, spec.lowTurns, spec.highTurns};
  if (s.columns > d) throw TensorShapeException("Heads of " + std::to_string(d) + " columns have no " + std::to_string(s.columns) + " to turn.");
  Check(om_rotary_frequencies(C(), &s, f));
  const om_head_strides xs = StridesOf(x, heads), ys = StridesOf(y, heads);
  Check(om_rotary(C(), x.Data(), &xs, positions.IsEmpty() ? nullptr : (const int32_t*)positions.RawData(), positions.Rank() == 2 ? l : 0,
                  spec.firstPosition, b, h, l, d, f, s.columns / 2, spec.adjacent, spec.magnitude, inverse, y.Data(), &ys));
}

static Tensor RotaryOver(const Tensor& x, const Tensor& positions, const RotarySpec& spec, int heads) {
  RequireFloat32(x);
  RequireInt32(positions, "Positions");
  if (heads == 0 ? x.Rank() != 4 : (x.Rank() != 3 || heads < 1 || x.GetShape()[2] % heads != 0))
    throw TensorShapeException("Rotary positions need [B,H,L,D], or [B,L,H*D] and the number of heads, not " + x.GetShape().ToString() + ".");
  const int b = x.GetShape()[0], l = heads ? x.GetShape()[1] : x.GetShape()[2];
  if (!positions.IsEmpty()) {
    const Shape& p = positions.GetShape();
    if (!((p.rank == 1 && p[0] == l) || (p.rank == 2 && p[0] == b && p[1] == l)))
      throw TensorShapeException("Positions must be [" + std::to_string(l) + "] or [" + std::to_string(b) + "," + std::to_string(l) + "], not " + p.ToString() + ".");
  }
  const Tensor pc = positions.IsEmpty() ? Tensor() : positions.Contiguous().Detach();
  Tensor y = NewOut(x.GetShape());
  Turn(InPlace(x), pc, spec, heads, false, y);
  if (!Ops::Recording({&x})) return y;
  auto rec = BackwardRecord::Create(OpKind::Rotary, 1, {&x});
  if (!pc.IsEmpty()) rec->Save(0, pc);
  rec->Ints = {heads, spec.columns, spec.adjacent ? 1 : 0, spec.firstPosition, spec.scaling};
  rec->Floats = {spec.base, spec.factor, spec.originalContext, spec.lowTurns, spec.highTurns, spec.magnitude};
  return rec->Attach(y);
}
Tensor Ops::Rotary(const Tensor& x, const Tensor& positions, const RotarySpec& spec) { return RotaryOver(x, positions, spec, 0); }
Tensor Ops::RotaryHeads(const Tensor& x, int heads, const Tensor& positions, const RotarySpec& spec) {
  if (heads < 1) throw TensorShapeException("Rotary positions over heads need at least one head.");
  return RotaryOver(x, positions, spec, heads);
}

// A turn is a rotation times the magnitude: its gradient is the turn back, times the magnitude.
void RotaryBackward(BackwardRecord& r, const Tensor& g) {
  if (!r.NeedsInputGrad(0)) return;
  RotarySpec spec;
  spec.columns = (int)r.Ints[1]; spec.adjacent = r.Ints[2] != 0; spec.firstPosition = (int)r.Ints[3]; spec.scaling = (int)r.Ints[4];
  spec.base = r.Floats[0]; spec.factor = r.Floats[1]; spec.originalContext = r.Floats[2]; spec.lowTurns = r.Floats[3]; spec.highTurns = r.Floats[4];
  spec.magnitude = (float)r.Floats[5];
  Tensor dx = Tensor::Create(DType::F32, r.InputShapes[0]);
  Turn(InPlace(g), r.Saved(0), spec, (int)r.Ints[0], true, dx);
  Engine::Emit(r, 0, dx, true);
}

// ---- attention by rule ---------------------------------------------------------------------------------------------------------

struct RuleSizes {
  int b, h, hkv, lq, lk, d;
};

static om_attention_rule RuleOf(const AttentionRule& a, const Tensor& prefix, const Tensor& qd, const Tensor& kd, const Tensor& slopes) {
  om_attention_rule r{};
  r.causal = a.causal; r.window = a.window; r.q_offset = a.qOffset; r.softcap = a.softcap;
  r.slopes = slopes.IsEmpty() ? nullptr : slopes.Data();
  r.prefix = prefix.IsEmpty() ? nullptr : (const int32_t*)prefix.RawData();
  r.q_documents = qd.IsEmpty() ? nullptr : (const int32_t*)qd.RawData();
  r.k_documents = kd.IsEmpty() ? nullptr : (const int32_t*)kd.RawData();
  return r;
}

static Tensor RuleOver(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionRule& a, float scale, int heads, int keyHeads) {
  RequireFloat32(q);
  RequireFloat32(k);
  RequireFloat32(v);
  const std::string shapes = q.GetShape().ToString() + ", " + k.GetShape().ToString() + ", " + v.GetShape().ToString() + ".";
  RuleSizes s{};
  if (heads == 0) {
    if (q.Rank() != 4 || k.Rank() != 4 || k.GetShape() != v.GetShape() || q.GetShape()[0] != k.GetShape()[0] || q.GetShape()[3] != k.GetShape()[3])
      throw TensorShapeException("Attention by rule needs [B,H,L,D] tensors with matching batch and D, not " + shapes);
    s = RuleSizes{q.GetShape()[0], q.GetShape()[1], k.GetShape()[1], q.GetShape()[2], k.GetShape()[2], q.GetShape()[3]};
  } else {
    if (q.Rank() != 3 || k.Rank() != 3 || k.GetShape() != v.GetShape() || q.GetShape()[0] != k.GetShape()[0] || keyHeads < 1 ||
        q.GetShape()[2] % heads != 0 || k.GetShape()[2] % keyHeads != 0 || q.GetShape()[2] / heads != k.GetShape()[2] / keyHeads)
      throw TensorShapeException("Attention by rule over heads needs [B,L,H*D] tensors with matching batch and D, not " + shapes);
    s = RuleSizes{q.GetShape()[0], heads, keyHeads, q.GetShape()[1], k.GetShape()[1], q.GetShape()[2] / heads};
  }
  if (s.hkv == 0 ? s.h != 0 : s.h % s.hkv != 0)
    throw TensorShapeException(std::to_string(s.h) + " query heads do not share " + std::to_string(s.hkv) + " key heads evenly.");
  RequireInt32(a.prefix, "Prefix lengths");
  RequireInt32(a.qDocuments, "Documents");
  RequireInt32(a.kDocuments, "Documents");
  auto shaped = [](const Tensor& t, const Shape& want, const char* what) {
    if (!t.IsEmpty() && t.GetShape() != want)
      throw TensorShapeException(std::string(what) + " must be " + want.ToString() + ", not " + t.GetShape().ToString() + ".");
    return t.IsEmpty() ? Tensor() : t.Contiguous().Detach();
  };
  const Tensor prefix = shaped(a.prefix, Shape{s.b}, "Prefix lengths"), qd = shaped(a.qDocuments, Shape{s.b, s.lq}, "The queries' documents"),
               kd = shaped(a.kDocuments, Shape{s.b, s.lk}, "The keys' documents"), slopes = shaped(a.slopes, Shape{s.h}, "Slopes");
  if (!slopes.IsEmpty()) RequireFloat32(slopes);
  if (scale == 0.f || isnan(scale)) scale = 1.0f / sqrtf((float)s.d);
  const om_attention_rule rule = RuleOf(a, prefix, qd, kd, slopes);
  const Tensor qc = InPlace(q), kc = InPlace(k), vc = InPlace(v);
  const om_head_strides qs = StridesOf(qc, heads), ks = StridesOf(kc, heads ? keyHeads : 0), vs = StridesOf(vc, heads ? keyHeads : 0);
  Tensor out = NewOut(q.GetShape());
  const om_head_strides os = StridesOf(out, heads);
  const bool recording = Ops::Recording({&q, &k, &v});
  Tensor lse = recording ? Tensor::Create(DType::F32, Shape{s.b, s.h, s.lq}) : Tensor();
  float* lp = lse.IsEmpty() ? nullptr : lse.Data();
  const bool half = Bf16Products() && s.d % 8 == 0 && Bf16InPlace(qc) && Bf16InPlace(kc) && Bf16InPlace(vc) && q.Length() > 0 && k.Length() > 0;
  if (half) {
    uint16_t* o16 = out.Bf16ForWrite();
    Check(om_rule_attention_fwd_bf16(C(), &rule, qc.Bf16(), &qs, kc.Bf16(), &ks, vc.Bf16(), &vs, s.b, s.h, s.hkv, s.lq, s.lk, s.d, scale, out.Data(),
                                     o16, &os, lp));
    out.Bf16Written();
  } else {
    Check(om_rule_attention_fwd(C(), &rule, qc.Data(), &qs, kc.Data(), &ks, vc.Data(), &vs, s.b, s.h, s.hkv, s.lq, s.lk, s.d, scale, out.Data(), &os, lp));
  }
  if (!recording) return out;
  auto rec = BackwardRecord::Create(OpKind::RuleAttention, 9, {&q, &k, &v});
  rec->Save(0, qc.Detach());
  rec->Save(1, kc.Detach());
  rec->Save(2, vc.Detach());
  rec->Save(3, out.Detach());
  rec->Save(4, lse);
  if (!prefix.IsEmpty()) rec->Save(5, prefix);
  if (!qd.IsEmpty()) {
    rec->Save(6, qd);
    rec->Save(7, kd);
  }
  if (!slopes.IsEmpty()) rec->Save(8, slopes);
  rec->Ints = {heads, keyHeads, a.causal ? 1 : 0, a.window, a.qOffset, half ? 1 : 0, s.b, s.h, s.hkv, s.lq, s.lk, s.d};
  rec->Floats = {a.softcap, scale};
  return rec->Attach(out);
}
Tensor Ops::RuleAttention(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionRule& rule, float scale) {
  return RuleOver(q, k, v, rule, scale, 0, 0);
}
Tensor Ops::RuleAttentionHeads(const Tensor& q, const Tensor& k, const Tensor& v, int heads, int keyHeads, const AttentionRule& rule, float scale) {
  if (heads < 1 || keyHeads < 1) throw TensorShapeException("Attention by rule over heads needs at least one head.");
  return RuleOver(q, k, v, rule, scale, heads, keyHeads);
}

void RuleAttentionBackward(BackwardRecord& r, const Tensor& g) {
  const Tensor &q = r.Saved(0), &k = r.Saved(1), &v = r.Saved(2), &out = r.Saved(3), &lse = r.Saved(4);
  const int heads = (int)r.Ints[0], keyHeads = heads ? (int)r.Ints[1] : 0;
  AttentionRule a;
  a.causal = r.Ints[2] != 0; a.window = (int)r.Ints[3]; a.qOffset = (int)r.Ints[4]; a.softcap = (float)r.Floats[0];
  const om_attention_rule rule = RuleOf(a, r.Saved(5), r.Saved(6), r.Saved(7), r.Saved(8));
  const RuleSizes s{(int)r.Ints[6], (int)r.Ints[7], (int)r.Ints[8], (int)r.Ints[9], (int)r.Ints[10], (int)r.Ints[11]};
  const float scale = (float)r.Floats[1];
  const Tensor gc = g.Contiguous();
  Tensor dq, dk, dv;
  if (r.NeedsInputGrad(0)) dq = Tensor::Create(DType::F32, r.InputShapes[0]);
  if (r.NeedsInputGrad(1)) dk = Tensor::Create(DType::F32, r.InputShapes[1]);
  if (r.NeedsInputGrad(2)) dv = Tensor::Create(DType::F32, r.InputShapes[2]);
  const om_head_strides gs = StridesOf(gc, heads), qs = StridesOf(q, heads), ks = StridesOf(k, keyHeads), vs = StridesOf(v, keyHeads),
                        os = StridesOf(out, heads);
  om_head_strides dqs{}, dks{}, dvs{};
  if (!dq.IsEmpty()) dqs = StridesOf(dq, heads);
  if (!dk.IsEmpty()) dks = StridesOf(dk, keyHeads);
  if (!dv.IsEmpty()) dvs = StridesOf(dv, keyHeads);
  float *dqp = dq.IsEmpty() ? nullptr : dq.Data(), *dkp = dk.IsEmpty() ? nullptr : dk.Data(), *dvp = dv.IsEmpty() ? nullptr : dv.Data();
  if (r.Ints[5]) {
    Check(om_rule_attention_bwd_bf16_out32(C(), &rule, gc.Bf16(), &gs, q.Bf16(), &qs, k.Bf16(), &ks, v.Bf16(), &vs, out.Data(), &os, lse.Data(), s.b, s.h,
                                           s.hkv, s.lq, s.lk, s.d, scale, dqp, nullptr, &dqs, dkp, nullptr, &dks, dvp, nullptr, &dvs));
  } else {
    Check(om_rule_attention_bwd(C(), &rule, gc.Data(), &gs, q.Data(), &qs, k.Data(), &ks, v.Data(), &vs, out.Data(), &os, lse.Data(), s.b, s.h, s.hkv, s.lq,
                                s.lk, s.d, scale, dqp, &dqs, dkp, &dks, dvp, &dvs));
  }
  if (!dq.IsEmpty()) Engine::Emit(r, 0, dq, true);
  if (!dk.IsEmpty()) Engine::Emit(r, 1, dk, true);
  if (!dv.IsEmpty()) Engine::Emit(r, 2, dv, true);
}

}  // namespace omh
