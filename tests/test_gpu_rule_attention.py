"""Attention by rule through the C ABI and the tensor API against the formulas in 64 bits: masks, heads, lengths and layouts where it
can go wrong, in both precisions, with each element's error bounded by the roundings on its way (rule_reference.attention)."""
import ctypes as C

import numpy as np
import pytest

import om_binding as omb
import rule_reference as ref
from om_binding import f32, i32

pytestmark = pytest.mark.gpu
BF16 = omb.OM_TF32 | omb.OM_BF16_OPERANDS


def documents(r, b, l, most, padded):
    out = np.full((b, l), -1, np.int32)
    for n in range(b):
        at, doc = 0, int(r.integers(0, 3))
        while at < l - padded:
            size = int(r.integers(1, most + 1))
            out[n, at:min(at + size, l - padded)] = doc
            at, doc = at + size, doc + 1
    return out


class Call:
    """One problem on the device. layout 'heads': [B, H, L, D]; 'rows': [B, L, H, D]; 'packed': q | k | v in one [B, L, (H + 2 Hkv) D]."""

    def __init__(self, ctx, r, b, h, hk, lq, lk, d, half=False, layout="rows", causal=False, window=0, q_offset=None, prefix=False, softcap=0.0,
                 slopes=False, docs=0, padded=0, scale=None, size=1.0):
        self.ctx, self.half, self.dims = ctx, half, (b, h, hk, lq, lk, d)
        self.q_offset = lk - lq if q_offset is None else q_offset
        self.scale = d ** -0.5 if scale is None else scale
        self.prefix = r.integers(0, lk + 1, b).astype(np.int32) if prefix else None
        kd = documents(r, b, lk, docs, padded) if docs else None
        qd = (kd[:, -lq:] if lq <= lk else documents(r, b, lq, docs, padded)).copy() if docs else None
        self.kd, self.qd = kd, qd
        self.slopes = (2.0 ** -(1.0 + np.arange(h))).astype(np.float32) if slopes else None
        self.causal, self.window, self.softcap = causal, window, softcap
        self.layout = layout
        self.value, self.dev = {}, {}
        for n, heads, l in (("q", h, lq), ("k", hk, lk), ("v", hk, lk), ("g", h, lq)):
            a = (size * r.standard_normal((b, heads, l, d))).astype(np.float32)
            self.value[n] = ref.from_bf16(ref.to_bf16(a)) if half else a
        if layout == "packed":
            assert lq == lk
            both = np.concatenate([self.value[n].transpose(0, 2, 1, 3) for n in ("q", "k", "v")], axis=2)
            self.packed = self.put(both)
            self.dpacked = self.poison(both.size)
        for n in ("q", "k", "v", "g"):
            if layout != "packed" or n == "g":
                self.dev[n] = self.put(self.value[n] if layout == "heads" else self.value[n].transpose(0, 2, 1, 3))

    def put(self, a):
        return self.ctx.to_device(ref.to_bf16(a) if self.half else np.ascontiguousarray(a, np.float32))

    def poison(self, n):
        a = self.ctx.empty((max(n, 1),), np.uint16 if self.half else np.float32)
        self.ctx.call("om_memset", self.ctx.handle, a.ptr, i32(0xFF), C.c_size_t(a.nbytes))
        return a

    def where(self, n):
        """(pointer, strides) of a tensor, of its gradient with a leading d."""
        b, h, hk, lq, lk, d = self.dims
        name = n[-1]
        heads, l = (h, lq) if name in "qgo" else (hk, lk)
        if self.layout == "packed" and name in "qkv":
            base = self.dpacked if n[0] == "d" else self.packed
            at = {"q": 0, "k": h, "v": h + hk}[name] * d * base.dtype.itemsize
            return C.c_void_p(base.ptr.value + at), omb.HeadStrides(l * (h + 2 * hk) * d, d, (h + 2 * hk) * d)
        if n not in self.dev:
            self.dev[n] = self.poison(b * heads * l * d)
        s = omb.HeadStrides(heads * l * d, l * d, d) if self.layout == "heads" else omb.HeadStrides(l * heads * d, d, heads * d)
        return self.dev[n].ptr, s

    def get(self, n):
        b, h, hk, lq, lk, d = self.dims
        name = n[-1]
        heads, l = (h, lq) if name in "qgo" else (hk, lk)
        if self.layout == "packed" and name in "qkv":
            a = self.dpacked.numpy().reshape(b, l, h + 2 * hk, d)
            a = a[:, :, {"q": slice(0, h), "k": slice(h, h + hk), "v": slice(h + hk, None)}[name]]
        else:
            a = self.dev[n].numpy()[: b * heads * l * d].reshape((b, heads, l, d) if self.layout == "heads" else (b, l, heads, d))
        a = ref.from_bf16(a) if self.half else a
        return a if self.layout == "heads" else a.transpose(0, 2, 1, 3)

    def rule(self):
        self.keep = {n: self.ctx.to_device(a) for n, a in (("slopes", self.slopes), ("prefix", self.prefix), ("q_documents", self.qd),
                                                           ("k_documents", self.kd)) if a is not None}
        return omb.AttentionRule(causal=self.causal, window=self.window, q_offset=self.q_offset, softcap=self.softcap,
                                 **{n: a.ptr.value for n, a in self.keep.items()})

    def run(self, backward=True):
        b, h, hk, lq, lk, d = self.dims
        self.the_rule, self.lse = self.rule(), self.ctx.empty((b, h, lq))
        self.queue(backward)
        self.ctx.sync()
        return self

    def queue(self, backward=True):
        b, h, hk, lq, lk, d = self.dims
        ctx, rule = self.ctx, self.the_rule
        sizes = [i32(n) for n in self.dims] + [f32(self.scale)]
        w = lambda n: (self.where(n)[0], C.byref(self.where(n)[1]))   # noqa: E731
        o, os = w("o")
        qkv = [*w("q"), *w("k"), *w("v")]
        ctx.call("om_rule_attention_fwd" + ("_bf16" if self.half else ""), ctx.handle, C.byref(rule), *qkv, *sizes, *([None, o] if self.half else [o]), os,
                 self.lse.ptr)
        if backward:
            grads = []
            for n in ("dq", "dk", "dv"):
                p, s = w(n)
                grads += ([None] if self.half else []) + [p, s]
            ctx.call("om_rule_attention_bwd" + ("_bf16" if self.half else ""), ctx.handle, C.byref(rule), *w("g"), *qkv, o, os, self.lse.ptr, *sizes, *grads)

    def check(self, backward=True, planes=None):
        b, h, hk, lq, lk, d = self.dims
        seen = ref.visible(b, lq, lk, self.causal, self.window, self.q_offset, self.prefix, self.qd, self.kd)
        v = self.value
        if planes is None:
            planes = not self.half and d <= 64 and d % 8 == 0 and max(lq, lk) >= 96
        want, tol = ref.attention(v["q"], v["k"], v["v"], v["g"], seen, self.scale, self.softcap, self.slopes, self.q_offset, self.half, planes)
        names = (("o", "out"),) + ((("dq", "dq"), ("dk", "dk"), ("dv", "dv")) if backward else ())
        for n, full in names:
            got = self.get(n).astype(np.float64)
            assert np.isfinite(got).all(), full
            over = np.abs(got - want[full]) - tol[full]
            assert over.max(initial=-1) <= 0, (full, over.max(), np.unravel_index(over.argmax(), over.shape))
        lse = self.lse.numpy()
        none = ~np.isfinite(want["lse"])
        assert np.array_equal(np.isneginf(lse), none)
        assert (np.abs(self.get("o"))[none] == 0).all()
        assert np.allclose(lse[~none], want["lse"][~none], rtol=1e-5, atol=1e-4)
        return self


MASKS = {
    "all": {},
    "causal": dict(causal=True),
    "window": dict(window=17),
    "causal-window": dict(causal=True, window=40),
    "window-of-one": dict(causal=True, window=1),
    "prefix": dict(causal=True, prefix=True),
    "window-prefix": dict(causal=True, window=9, prefix=True),
    "documents": dict(causal=True, docs=50, padded=11),
    "documents-both-ways": dict(docs=90, padded=70),
    "documents-prefix": dict(causal=True, docs=60, padded=3, prefix=True),
    "cap": dict(causal=True, softcap=5.0, size=2.0),
    "slopes": dict(slopes=True),
    "everything": dict(causal=True, window=60, prefix=True, softcap=8.0, slopes=True, docs=80, padded=20),
    "before-all-keys": dict(causal=True, q_offset=-70),
    "behind-all-keys": dict(causal=True, window=30, q_offset=500),
}


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("mask", list(MASKS))
def test_masks(ctx, mask, half):
    r = np.random.default_rng(list(MASKS).index(mask))
    Call(ctx, r, 2, 2, 2, 197, 197, 64, half=half, **MASKS[mask]).run().check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 2), (2, 1), (1, 64), (1, 1000), (63, 65), (64, 64), (65, 63), (127, 129), (128, 128), (129, 127), (256, 256),
                                   (257, 300), (300, 257), (40, 700), (385, 513)])
def test_lengths(ctx, lq, lk, half):
    r = np.random.default_rng(lq * 1000 + lk)
    Call(ctx, r, 1, 2, 1, lq, lk, 64, half=half, causal=True).run().check()
    Call(ctx, r, 2, 1, 1, lq, lk, 64, half=half, window=33, q_offset=0).run().check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d", [1, 2, 7, 8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 100, 120, 128, 136, 192, 256])
def test_widths(ctx, d, half):
    r = np.random.default_rng(d)
    Call(ctx, r, 1, 4, 2, 150, 150, d, half=half, causal=True, window=90).run().check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("h,hk", [(1, 1), (3, 1), (6, 2), (8, 1), (5, 5)])
@pytest.mark.parametrize("layout", ["heads", "rows", "packed"])
def test_shared_heads_and_layouts(ctx, h, hk, layout, half):
    r = np.random.default_rng(10 * h + hk)
    Call(ctx, r, 2, h, hk, 140, 140, 64, half=half, layout=layout, causal=True, docs=50, padded=5).run().check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("mask", ["all", "causal", "cap", "slopes", "everything", "documents-prefix"])
@pytest.mark.parametrize("layout,d", [("packed", 64), ("heads", 40)])
def test_calls_large_enough_for_the_tensor_pipe_in_both_precisions(ctx, layout, d, mask, half):
    r = np.random.default_rng(50 + d)
    m = dict(MASKS[mask])
    m.update({k: v * 6 for k, v in m.items() if k in ("window", "docs", "padded")})
    Call(ctx, r, 2, 8, 4, 750, 750, d, half=half, layout=layout, **m).run().check()


def test_large_fp32_call_with_few_queries_and_a_split_walk(ctx):
    r = np.random.default_rng(60)
    Call(ctx, r, 2, 8, 2, 30, 20011, 64, causal=True).run(False).check(False)


@pytest.mark.parametrize("half,b,h,hk,lq,lk,d,kw", [
    (True, 75, 4, 2, 1, 1100, 128, {}),                                           # more heads than SMs, not split
    (True, 75, 4, 2, 1, 1100, 64, dict(softcap=5.0, slopes=True)),
    (False, 75, 4, 2, 1, 1100, 64, {}),
    (True, 80, 2, 2, 100, 1300, 128, dict(causal=True)),                          # one tile of queries with its own keys
    (True, 1, 2, 2, 100, 1300, 128, dict(causal=True, window=20)),                # two or three tiles in sight
    (True, 2, 8, 1, 5, 3000, 64, dict(docs=40, padded=200, causal=True)),         # tiles in sight next to hidden ones
    (False, 2, 8, 1, 5, 3000, 64, dict(docs=40, padded=200, causal=True)),
    (True, 2, 4, 2, 3, 1200, 128, dict(causal=True, q_offset=5)),                 # one tile in sight: half the rows' warps have none
    (False, 2, 4, 2, 3, 1200, 64, dict(causal=True, q_offset=5)),
    (True, 2, 4, 2, 3, 1200, 96, dict(causal=True, q_offset=-10)),                # none
])
def test_few_queries_and_many_keys(ctx, half, b, h, hk, lq, lk, d, kw):
    r = np.random.default_rng(63)
    Call(ctx, r, b, h, hk, lq, lk, d, half=half, **kw).run(False).check(False)


def test_values_far_apart_keep_their_precision(ctx):
    """One value row 1e20 times the others: the rows that do not see it keep fp32 accuracy, in a call of the size that is otherwise done
    with two half-precision numbers a value. The same for tiny rows of k and of the output's gradient."""
    r = np.random.default_rng(61)
    for name, at, factor in (("v", 700, 1e20), ("k", 3, 1e-9), ("g", 5, 1e-9), ("q", 8, 1e-8)):
        c = Call(ctx, r, 2, 8, 4, 750, 750, 64, causal=True)
        c.value[name][:, :, at] *= np.float32(factor)
        c.dev[name] = c.put(c.value[name].transpose(0, 2, 1, 3))
        c.run().check(planes=False)


def test_more_keys_than_one_plan(ctx):
    r = np.random.default_rng(62)
    Call(ctx, r, 1, 2, 1, 2, 140003, 64, half=True, causal=True).run(False).check(False)
    Call(ctx, r, 1, 1, 1, 3, 131200, 64, half=True, causal=True, window=700).run().check()


@pytest.mark.parametrize("half", [False, True])
def test_strides_off_the_vector_grid(ctx, half):
    r = np.random.default_rng(3)
    b, h, l, d = 2, 3, 70, 64
    c = Call(ctx, r, b, h, h, l, l, d, half=half, layout="heads", causal=True)
    for n in ("q", "k", "v", "g"):          # rows d + 1 apart, starting one element in
        a = np.full((b * h * l, d + 1), np.nan, np.float32)
        a[:, 1:] = c.value[n].reshape(-1, d)
        c.dev[n] = c.put(a)
    plain = c.where
    c.where = lambda n: ((C.c_void_p(c.dev[n].ptr.value + c.dev[n].dtype.itemsize), omb.HeadStrides(h * l * (d + 1), l * (d + 1), d + 1))
                         if n in ("q", "k", "v", "g") else plain(n))
    c.run().check()


@pytest.mark.parametrize("half", [False, True])
def test_long_rows_and_many_keys(ctx, half):
    r = np.random.default_rng(8)
    Call(ctx, r, 1, 1, 1, 1, 20011, 64, half=half, causal=True).run(False).check(False)
    Call(ctx, r, 2, 4, 2, 3, 9001, 128, half=half, causal=True, window=5000).run(False).check(False)


def test_large_scores_do_not_overflow(ctx):
    r = np.random.default_rng(9)
    for half in (False, True):
        c = Call(ctx, r, 1, 2, 2, 130, 130, 64, half=half, causal=True, size=30.0).run()
        for n in ("o", "dq", "dk", "dv"):
            assert np.isfinite(c.get(n)).all()


def test_hidden_scores_may_be_infinite(ctx):
    """A hidden key's huge row makes its scores overflow; no visible one changes by a bit."""
    r = np.random.default_rng(12)
    for half in (False, True):
        c = Call(ctx, r, 1, 1, 1, 100, 100, 64, half=half, docs=100, padded=0)
        c.kd = c.qd = np.zeros((1, 100), np.int32)
        c.kd[:, 60:] = -1
        first = c.run().get("o").copy()
        c.value["k"][:, :, 60:] = 3e38
        c.dev["k"] = c.put(c.value["k"].transpose(0, 2, 1, 3))
        second = c.run()
        assert np.array_equal(first, second.get("o"))
        assert np.isfinite(second.get("dq")).all() and (second.get("dk")[:, :, 60:] == 0).all()


def test_same_bits_twice_and_gradients_one_by_one(ctx):
    r = np.random.default_rng(21)
    for half in (False, True):
        c = Call(ctx, r, 2, 4, 2, 200, 200, 64, half=half, causal=True, softcap=10.0).run()
        first = {n: c.get(n).copy() for n in ("o", "dq", "dk", "dv")}
        c.run()
        for n, a in first.items():
            assert np.array_equal(a, c.get(n)), n
        rule, sizes = c.rule(), [i32(n) for n in c.dims] + [f32(c.scale)]
        w = lambda n: (c.where(n)[0], C.byref(c.where(n)[1]))   # noqa: E731
        for only in ("dq", "dk", "dv"):
            c.dev[only] = c.poison(c.value[only[1]].size)
            args = []
            for n in ("dq", "dk", "dv"):
                p, s = w(n)
                args += ([None] if half else []) + [p if n == only else None, s]
            ctx.call("om_rule_attention_bwd" + ("_bf16" if half else ""), ctx.handle, C.byref(rule), *w("g"), *w("q"), *w("k"), *w("v"), *w("o"), c.lse.ptr,
                     *sizes, *args)
            ctx.sync()
            assert np.array_equal(first[only], c.get(only)), only


def test_a_sequence_does_not_depend_on_its_neighbours(ctx):
    """One sequence of an fp32 batch is made to hold values far apart (another kind of kernel does it): the others keep every bit. So do
    all when rows of no document are filled with what is not a number."""
    r = np.random.default_rng(23)
    c = Call(ctx, r, 3, 4, 2, 200, 200, 64, causal=True, docs=200, padded=0)
    c.qd[:, 180:] = -1
    c.kd[:, 180:] = -1
    first = {n: c.run().get(n).copy() for n in ("o", "dq", "dk", "dv")}
    for n in ("q", "k", "v", "g"):
        c.value[n][:, :, 180:] = np.nan
        c.value[n][1, :, 7] *= np.float32(1e-9)
        c.dev[n] = c.put(c.value[n].transpose(0, 2, 1, 3))
    c.run()
    for n, a in first.items():
        assert np.array_equal(a[[0, 2]], c.get(n)[[0, 2]]), n
        assert np.isfinite(c.get(n)).all(), n


def test_large_fp32_call_in_a_graph(ctx):
    """Captured once, replayed over other values: the units and the choice of kernels follow the values, not the capture."""
    r = np.random.default_rng(24)
    c = Call(ctx, r, 2, 4, 2, 300, 300, 64, causal=True).run()
    graph = C.c_void_p()
    ctx.call("om_graph_begin", ctx.handle)
    c.queue()
    ctx.call("om_graph_end", ctx.handle, C.byref(graph))
    try:
        for n, factor, planes in (("q", 1.0, True), ("v", 300.0, True), ("k", 1e-12, False)):
            c.value[n][:, :, 5:9] = (c.value[n][:, :, 5:9] * np.float32(factor)).astype(np.float32)
            host = np.ascontiguousarray(c.value[n].transpose(0, 2, 1, 3))
            ctx.call("om_memcpy_h2d", ctx.handle, c.dev[n].ptr, host.ctypes.data_as(C.c_void_p), C.c_size_t(host.nbytes))
            ctx.call("om_graph_launch", ctx.handle, graph)
            ctx.sync()
            c.check(planes=planes)
    finally:
        ctx.call("om_graph_destroy", ctx.handle, graph)


def test_workspaces_under_the_checked_flag(ctx):
    """Poisoned workspaces with guard bytes behind them: nothing is read that was not written, nothing written behind an end."""
    ctx.set_flags(omb.OM_CHECKED)
    try:
        r = np.random.default_rng(25)
        for half in (False, True):
            for lq, lk, d, kw in ((130, 130, 64, dict(causal=True, docs=50, padded=9)), (1, 2050, 64, {}), (77, 300, 40, dict(softcap=4.0, slopes=True)), (5, 7, 33, {})):
                Call(ctx, r, 2, 4, 2, lq, lk, d, half=half, **kw).run().check()
    finally:
        ctx.set_flags(0)


def test_both_forms_of_a_result(ctx):
    """The bfloat16 entry points write fp32, bfloat16 or both; the bfloat16 values are the fp32 ones rounded."""
    r = np.random.default_rng(22)
    c = Call(ctx, r, 1, 2, 2, 150, 150, 64, half=True, causal=True).run()
    rule, sizes = c.rule(), [i32(n) for n in c.dims] + [f32(c.scale)]
    w = lambda n: (c.where(n)[0], C.byref(c.where(n)[1]))   # noqa: E731
    n = c.value["q"].size
    f = {k: ctx.empty((n,)) for k in ("o", "dq", "dk", "dv")}
    ctx.call("om_rule_attention_fwd_bf16", ctx.handle, C.byref(rule), *w("q"), *w("k"), *w("v"), *sizes, f["o"].ptr, *w("o"), c.lse.ptr)
    grads = [a for k in ("dq", "dk", "dv") for a in (f[k].ptr, *w(k))]
    ctx.call("om_rule_attention_bwd_bf16", ctx.handle, C.byref(rule), *w("g"), *w("q"), *w("k"), *w("v"), *w("o"), c.lse.ptr, *sizes, *grads)
    ctx.sync()
    c.check()
    for k in f:
        assert np.array_equal(ref.to_bf16(f[k].numpy()), c.dev[k].numpy()), k


@pytest.mark.parametrize("half", [False, True])
def test_no_keys_and_no_queries(ctx, half):
    r = np.random.default_rng(1)
    c = Call(ctx, r, 2, 2, 1, 5, 0, 16, half=half).run()
    assert (c.get("o") == 0).all() and np.isneginf(c.lse.numpy()).all() and (c.get("dq") == 0).all()
    c = Call(ctx, r, 2, 2, 1, 0, 5, 16, half=half).run()
    assert (c.get("dk") == 0).all() and (c.get("dv") == 0).all()


def test_refusals(ctx):
    r = np.random.default_rng(2)
    c = Call(ctx, r, 1, 2, 1, 8, 8, 64, causal=True, docs=4).run()

    def forward(status, rule=None, **change):
        dims = dict(zip(("b", "h", "hk", "lq", "lk", "d"), c.dims)) | {k: v for k, v in change.items() if k in ("b", "h", "hk", "lq", "lk", "d")}
        q, qs = c.where("q")
        if "row" in change:
            qs = omb.HeadStrides(qs.batch, qs.head, change["row"])
        o, os = c.where("o")
        if "out_head" in change:
            os = omb.HeadStrides(os.batch, change["out_head"], os.row)
        args = [C.byref(rule if rule is not None else c.rule()), None if "no_q" in change else q, C.byref(qs)]
        for n in ("k", "v"):
            p, s = c.where(n)
            args += [p, C.byref(s)]
        args += [i32(dims[n]) for n in ("b", "h", "hk", "lq", "lk", "d")] + [f32(change.get("scale", 0.1)), None if "no_out" in change else o, C.byref(os), None]
        with pytest.raises(omb.OmError) as e:
            ctx.call("om_rule_attention_fwd", ctx.handle, *args)
        assert e.value.status == status, (change, e.value)

    def changed(**fields):
        rule = c.rule()
        for n, v in fields.items():
            setattr(rule, n, v)
        return rule

    forward(1, h=3, hk=2)
    forward(1, lq=-1)
    forward(1, row=63)
    forward(1, out_head=0)
    forward(7, d=257)
    forward(7, d=0)
    forward(7, b=70000)
    forward(8, scale=float("nan"))
    forward(8, no_q=1)
    forward(8, no_out=1)
    forward(8, changed(window=-1))
    forward(8, changed(softcap=-1.0))
    forward(8, changed(softcap=float("inf")))
    forward(8, changed(q_offset=(1 << 30) + 1))
    forward(8, changed(k_documents=None))
    with pytest.raises(omb.OmError):
        ctx.call("om_rule_attention_fwd", ctx.handle, None, *[None] * 6, *[i32(1)] * 6, f32(1), None, None, None)
    q, qs = c.where("q")
    with pytest.raises(omb.OmError) as e:    # no log-sum-exp
        ctx.call("om_rule_attention_bwd", ctx.handle, C.byref(c.rule()), q, C.byref(qs), q, C.byref(qs), q, C.byref(qs), q, C.byref(qs), q, C.byref(qs), None,
                 *[i32(n) for n in c.dims], f32(0.1), q, C.byref(qs), None, None, None, None)
    assert e.value.status == 8


# ---- through the tensor API --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("flags", [0, BF16])
@pytest.mark.parametrize("heads_form", [False, True])
def test_tensor_api_gradients(ctx, flags, heads_form):
    ctx.set_flags(flags)
    try:
        r = np.random.default_rng(31)
        b, h, hk, l, d = 2, 4, 2, 77, 32
        half = flags != 0
        a = {n: r.standard_normal((b, heads, l, d)).astype(np.float32) for n, heads in (("q", h), ("k", hk), ("v", hk), ("g", h))}
        a = {n: ref.from_bf16(ref.to_bf16(x)) for n, x in a.items()}
        docs = documents(r, b, l, 30, 4)
        slopes = np.array([0.5, 0.25, 0.125, 0.0625], np.float32)
        shaped = lambda x: np.ascontiguousarray(x.transpose(0, 2, 1, 3).reshape(b, l, -1)) if heads_form else x   # noqa: E731
        q, k, v = (omb.Tensor.from_numpy(shaped(a[n]), requires_grad=True) for n in ("q", "k", "v"))
        extra = [None, omb.Tensor.from_numpy(docs), omb.Tensor.from_numpy(docs), omb.Tensor.from_numpy(slopes)]
        ints = [1, 40, 0] + ([h, hk] if heads_form else [])
        out = omb.call("rule_attention_heads" if heads_form else "rule_attention", [q, k, v, *extra], ints=ints, floats=[6.0, 0.0])
        out.backward(omb.Tensor.from_numpy(shaped(a["g"])))
        seen = ref.visible(b, l, l, True, 40, 0, None, docs, docs)
        want, tol = ref.attention(a["q"], a["k"], a["v"], a["g"], seen, d ** -0.5, 6.0, slopes, 0, half)
        for n, t in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
            got = t.numpy().astype(np.float64)
            if heads_form:
                got = got.reshape(b, l, -1, d).transpose(0, 2, 1, 3)
            assert (np.abs(got - want[n]) <= tol[n]).all(), (n, np.abs(got - want[n]).max())
    finally:
        ctx.set_flags(0)


def test_gradients_against_differences(ctx):
    """The loss sum(w * out) moves by the gradients' inner product with a small step: central differences, whose rounding is
    2^-24 of the loss's terms over the step and whose curvature term is the step squared."""
    ctx.set_flags(0)
    r = np.random.default_rng(33)
    b, h, hk, l, d = 1, 2, 1, 19, 16
    a = {n: r.standard_normal((b, heads, l, d)).astype(np.float32) for n, heads in (("q", h), ("k", hk), ("v", hk))}
    w = r.standard_normal((b, h, l, d)).astype(np.float32)
    step = {n: r.standard_normal(x.shape).astype(np.float32) for n, x in a.items()}

    def out(at):
        ts = [omb.Tensor.from_numpy((a[n] + at * step[n]).astype(np.float32), requires_grad=True) for n in ("q", "k", "v")]
        return ts, omb.call("rule_attention", ts, ints=[1, 12, 0], floats=[4.0, 0.0])

    ts, o = out(0.0)
    o.backward(omb.Tensor.from_numpy(w))
    slope = sum(float((t.grad.numpy().astype(np.float64) * step[n]).sum()) for t, n in zip(ts, ("q", "k", "v")))
    eps = 2.0 ** -8
    up, down = (float((w.astype(np.float64) * out(s)[1].numpy()).sum()) for s in (eps, -eps))
    assert abs((up - down) / (2 * eps) - slope) <= 0.02 * max(1.0, abs(slope))


def test_tensor_api_refusals(ctx):
    t = lambda *s: omb.Tensor.from_numpy(np.zeros(s, np.float32))   # noqa: E731
    with pytest.raises(omb.ShapeError):
        omb.call("rule_attention", [t(1, 3, 4, 8), t(1, 2, 4, 8), t(1, 2, 4, 8)], ints=[1])
    with pytest.raises(omb.ShapeError):
        omb.call("rule_attention", [t(1, 2, 4, 8), t(1, 2, 4, 16), t(1, 2, 4, 16)], ints=[1])
    with pytest.raises(omb.ShapeError):
        omb.call("rule_attention_heads", [t(1, 4, 16), t(1, 4, 16), t(1, 4, 16)], ints=[1, 0, 0, 3, 3])
    with pytest.raises(omb.ShapeError):      # documents of another length
        omb.call("rule_attention", [t(1, 2, 4, 8)] * 3 + [None, omb.Tensor.from_numpy(np.zeros((1, 5), np.int32))] * 1, ints=[1])
    with pytest.raises(omb.ShapeError):      # prefix lengths that are not integers
        omb.call("rule_attention", [t(1, 2, 4, 8)] * 3 + [t(1)], ints=[1])


# ---- captured into a graph -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("half", [False, True])
def test_captured_and_replayed(ctx, half):
    r = np.random.default_rng(41)
    c = Call(ctx, r, 1, 4, 2, 160, 160, 64, half=half, causal=True, docs=70).run().check()
    first = {n: c.get(n).copy() for n in ("o", "dq", "dk", "dv")}
    graph = C.c_void_p()
    rule = c.rule()
    c.rule = lambda: rule
    ctx.sync()
    ctx.call("om_graph_begin", ctx.handle)
    sync, ctx.sync = ctx.sync, lambda: None
    empty, lse = ctx.empty, c.lse
    ctx.empty = lambda *a, **k: lse
    try:
        c.run()
    finally:
        ctx.sync, ctx.empty = sync, empty
        ctx.call("om_graph_end", ctx.handle, C.byref(graph))
    for n in ("dq", "dk", "dv", "o"):
        a = c.dev[n]
        ctx.call("om_memset", ctx.handle, a.ptr, i32(0xFF), C.c_size_t(a.nbytes))
    other = Call(ctx, r, 1, 4, 4, 300, 300, 64, half=half).run()      # takes pool memory between capture and replay
    for _ in range(2):
        ctx.call("om_graph_launch", ctx.handle, graph)
    ctx.sync()
    for n, a in first.items():
        assert np.array_equal(a, c.get(n)), n
    other.check()
    ctx.call("om_graph_destroy", ctx.handle, graph)
