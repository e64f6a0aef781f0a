"""Attention by rule where values are far apart, huge or tiny, caps large and padding not a number: against the formulas in 64 bits, with
bounds that follow from the precision promised and not from how a kernel gets there."""
import ctypes as C

import numpy as np
import pytest

import om_binding as omb
import rule_reference as ref
from om_binding import f32, i32
from test_gpu_rule_attention import Call

pytestmark = pytest.mark.gpu


def put(c, name, value):
    """Another value of one operand of a call in the layout of rows."""
    c.value[name] = ref.from_bf16(ref.to_bf16(value)) if c.half else value.astype(np.float32)
    c.dev[name] = c.put(c.value[name].transpose(0, 2, 1, 3))


def wanted(c):
    b, h, hk, lq, lk, d = c.dims
    seen = ref.visible(b, lq, lk, c.causal, c.window, c.q_offset, c.prefix, c.qd, c.kd)
    v = c.value
    return ref.attention(v["q"], v["k"], v["v"], v["g"], seen, c.scale, c.softcap, c.slopes, c.q_offset, c.half)


def row_errors(got, want):
    """Each row's error over the row, in the Euclidean norm."""
    return np.linalg.norm(got - want, axis=-1) / np.maximum(np.linalg.norm(want, axis=-1), 1e-300)


@pytest.mark.parametrize("names,size", [("v", 1e19), ("g", 1e20), ("v", 1e22), ("q", 1e19), ("vg", 3e17)])
def test_huge_values_in_every_row(ctx, names, size):
    """All rows alike, so nothing is far apart, in a call long enough for two half-precision numbers a value."""
    r = np.random.default_rng(70)
    c = Call(ctx, r, 1, 4, 2, 300, 300, 64, causal=True)
    for n in names:
        put(c, n, c.value[n] * np.float32(size))
    if names == "q":
        put(c, "k", c.value["k"] * np.float32(1 / size))
    c.run().check(planes=False)


# What fp32 arithmetic does to a row of a gradient whose terms are of like size: a product of two pairs of half-precision numbers is within
# 12 * 2^-24, there are two in a row (dP, dS k), a weight is within 16 * 2^-24 for scores up to 4, and the row dot that is taken from dP has the
# error of a sum of 64 products once more. 64 * 2^-24 holds them, in norm, whatever the size of the row.
LIKE_FP32 = 64 * ref.U32


@pytest.mark.parametrize("power", [-6, -10, -13])
def test_a_small_gradient_row_keeps_its_digits(ctx, power):
    r = np.random.default_rng(71)
    c = Call(ctx, r, 1, 2, 1, 1024, 1024, 64)
    rows = [5, 300, 1023]
    g = c.value["g"].copy()
    g[:, :, rows] *= np.float32(2.0 ** power)
    put(c, "g", g)
    c.run()
    want, _ = wanted(c)
    err = row_errors(c.get("dq"), want["dq"])
    assert err.max() <= LIKE_FP32, (err.max(), err[:, :, rows])


@pytest.mark.parametrize("name", ["g", "v"])
@pytest.mark.parametrize("power", [-8, -13])
def test_a_document_of_small_values_keeps_its_digits(ctx, name, power):
    """The second of two documents has small values: its rows of every gradient are as exact as the first one's."""
    r = np.random.default_rng(72)
    c = Call(ctx, r, 1, 2, 1, 700, 700, 64, docs=700)
    c.kd = c.qd = (np.arange(700)[None] >= 350).astype(np.int32)
    a = c.value[name].copy()
    a[:, :, 350:] *= np.float32(2.0 ** power)
    put(c, name, a)
    c.run()
    want, _ = wanted(c)
    for n in ("dq", "dk", "dv"):
        err = row_errors(c.get(n), want[n])
        assert err.max() <= LIKE_FP32, (n, err.max(), err[:, :, :350].max())


def test_gradients_of_hardly_seen_keys(ctx):
    """Keys whose weights are about 2^-36 in every row. A weight's relative error is its score's absolute one: 25 here, four roundings of 2^-24
    of it each, so 100 * 2^-24 more than above.

    All queries lie in nearly one direction, so the terms of dK = sum dS q, whose signs differ, can cancel: a row's error is that of its terms,
    independent of one another, and so is taken over the root of the sum of their squares (which is the row's norm where they do not cancel)."""
    r = np.random.default_rng(73)
    c = Call(ctx, r, 1, 2, 2, 500, 500, 64, scale=1.0)
    q, k = 0.05 * c.value["q"], c.value["k"].copy()
    q[..., 0], k[..., 0] = 5.0, 0.0
    k[:, :, 200:210, 0] = -5.0
    put(c, "q", q)
    put(c, "k", k)
    c.run()
    want, _ = wanted(c)
    q, k, v, g = (c.value[n].astype(np.float64) for n in "qkvg")
    p = np.exp(np.einsum("bhid,bhjd->bhij", q, k) - want["lse"][..., None])
    ds = p * (np.einsum("bhid,bhjd->bhij", g, v) - (g * want["out"]).sum(-1, keepdims=True))
    for n, weight, rows in (("dv", p, g), ("dk", ds, q)):
        terms = np.sqrt(np.einsum("bhij,bhi->bhj", weight ** 2, (rows ** 2).sum(-1)))
        err = np.linalg.norm(c.get(n) - want[n], axis=-1) / terms
        assert err.max() <= LIKE_FP32 + 100 * ref.U32, (n, err.max(), err[:, :, 200:210])


def test_many_small_weights_add_up(ctx):
    """One key has all but 2^-21 of the weight and a value of zero: the output is what the thousands of others add up to."""
    r = np.random.default_rng(74)
    c = Call(ctx, r, 1, 2, 2, 200, 5000, 64, scale=1.0, q_offset=0)
    q, k, v = 0.05 * c.value["q"], 0.05 * c.value["k"], c.value["v"].copy()
    q[..., 0], k[..., 0] = 5.0, 0.0
    k[:, :, 17, 0] = 4.6                    # 23 above the others: 2^-33 each
    v[:, :, :128] = 0.0
    v[:, :, 128:, 0] = 1.0
    put(c, "q", q)
    put(c, "k", k)
    put(c, "v", v)
    c.run(False)
    want, _ = wanted(c)
    got = c.get("o").astype(np.float64)
    err = np.abs(got[..., 0] - want["out"][..., 0]) / want["out"][..., 0]
    assert err.max() <= LIKE_FP32 + 100 * ref.U32, err.max()


@pytest.mark.parametrize("half,d", [(False, 64), (True, 64), (True, 128), (False, 80)])
@pytest.mark.parametrize("softcap", [0.5, 50.0, 1e3, 1e6, 1e30, 3e38])
def test_caps_of_every_size(ctx, half, d, softcap):
    """A score's error is relative to the score. Where the cap is far above them it changes nothing: the scores are those of no cap."""
    r = np.random.default_rng(75)
    c = Call(ctx, r, 1, 2, 1, 260, 260, d, half=half, causal=True, softcap=softcap).run()
    b, h, hk, lq, lk, _ = c.dims
    v = {n: a.astype(np.float64) for n, a in c.value.items()}
    s = c.scale * np.einsum("bhid,bhjd->bhij", v["q"], np.repeat(v["k"], h // hk, 1))
    s = softcap * np.tanh(s / softcap)
    s = np.where(np.arange(lk)[None] <= np.arange(lq)[:, None], s, -np.inf)
    lse = np.log(np.exp(s - s.max(-1, keepdims=True)).sum(-1)) + s.max(-1)
    # A score: d products as a random walk of four deviations of 2^-24 each times sqrt(d), the cap and its scale sixteen roundings, of scores below 8;
    # the log-sum-exp is a mean of scores beside its own four roundings.
    allowed = 8 * ref.U32 * (4 * np.sqrt(d) + 16 + 4)
    assert np.abs(c.lse.numpy() - lse).max() <= allowed, np.abs(c.lse.numpy() - lse).max()
    want, tol = (ref.attention(v["q"], v["k"], v["v"], v["g"], ref.visible(b, lq, lk, True), c.scale, 0.0, None, 0, half) if softcap >= 1e6 else (None, None))
    if want:
        for n, full in (("o", "out"), ("dq", "dq"), ("dk", "dk"), ("dv", "dv")):
            assert (np.abs(c.get(n) - want[full]) <= tol[full]).all(), full


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("d,lq,lk,docs,padded", [(64, 200, 200, 90, 20), (128, 300, 300, 200, 130), (64, 1, 700, 400, 90), (40, 130, 130, 130, 1), (120, 5, 600, 50, 60)])
def test_padding_of_bfloat16_calls_may_hold_anything(ctx, d, lq, lk, docs, padded, what):
    r = np.random.default_rng(76)
    c = Call(ctx, r, 2, 4, 2, lq, lk, d, half=True, causal=True, docs=docs, padded=padded)
    if lk > 400:                             # padding between documents as well
        c.kd[:, 130:150] = -1
    c.qd = c.kd[:, -lq:].copy()
    if lq == 1 or lq == 5:
        c.qd[:] = c.kd[:, 100:101]
        c.q_offset = lk
    first = {n: c.run().get(n).copy() for n in ("o", "dq", "dk", "dv")}
    c.check()
    for n, ids in (("q", c.qd), ("k", c.kd), ("v", c.kd), ("g", c.qd)):
        a = c.value[n].copy()
        a.transpose(0, 2, 1, 3)[ids < 0] = what
        put(c, n, a)
    c.run()
    for n, a in first.items():
        assert np.array_equal(a, c.get(n)), n


@pytest.mark.parametrize("half", [False, True])
def test_large_scores_against_64_bits(ctx, half):
    """Scores of several hundred: almost all of a row's weight on one key."""
    r = np.random.default_rng(77)
    Call(ctx, r, 1, 2, 2, 260, 260, 64, half=half, causal=True, size=8.0).run().check(planes=False)


@pytest.mark.parametrize("half", [False, True])
def test_no_query_heads(ctx, half):
    """Key heads that no query head shares get gradients of zero."""
    r = np.random.default_rng(78)
    c = Call(ctx, r, 2, 2, 2, 6, 9, 16, half=half).run()
    rule, sizes = c.rule(), [i32(n) for n in (2, 0, 2, 6, 9, 16)] + [f32(c.scale)]
    w = lambda n: (c.where(n)[0], C.byref(c.where(n)[1]))   # noqa: E731
    for n in ("dk", "dv"):
        c.dev[n] = c.poison(c.value[n[1]].size)
    grads = [a for n in ("dq", "dk", "dv") for a in (([None] if half else []) + list(w(n)))]
    ctx.call("om_rule_attention_bwd" + ("_bf16" if half else ""), ctx.handle, C.byref(rule), *w("g"), *w("q"), *w("k"), *w("v"), *w("o"), c.lse.ptr, *sizes, *grads)
    ctx.sync()
    assert (c.get("dk") == 0).all() and (c.get("dv") == 0).all()


@pytest.mark.parametrize("api", [False, True])
def test_a_row_that_looks_at_one_key_keeps_its_gradient(ctx, api):
    """Scores of tens within one tile: dP and the row dot nearly cancel where a weight is almost 1, and the output's rounding to bfloat16
    (2^-9 of it on average) is many times what is left. With the output in fp32 a row's dQ has only the roundings of its weights in the output,
    which are none for the largest weight (exactly 1), and of its score gradients: half a step of bfloat16 of each term, and with
    the sums' signs at random no more than that of the row's root sum of squares, twice."""
    r = np.random.default_rng(79)
    c = Call(ctx, r, 1, 2, 2, 128, 128, 64, half=True, layout="heads", causal=True, size=3.0)
    put_heads = {n: (c.value[n] if n in "qk" else ref.from_bf16(ref.to_bf16(c.value[n] / np.float32(3)))) for n in "qkvg"}
    c.value = put_heads
    c.dev.update({n: c.put(a) for n, a in put_heads.items()})
    want, _ = wanted(c)
    q, k, v, g = (c.value[n].astype(np.float64) for n in "qkvg")
    s = np.where(np.tril(np.ones((128, 128), bool)), c.scale * np.einsum("bhid,bhjd->bhij", q, k), -np.inf)
    p = np.exp(s - want["lse"][..., None])
    dp = np.einsum("bhid,bhjd->bhij", g, v)
    ds = p * (dp - (g * want["out"]).sum(-1, keepdims=True))
    # The row dot: what the rounding of the weights below the largest leaves in the output, and fp32 sums.
    rounded = np.where(p == p.max(-1, keepdims=True), 0.0, p) * ref.U16
    dot = np.einsum("bhij,bhjd->bhid", rounded, np.abs(v))
    dot = (np.abs(g) * dot).sum(-1, keepdims=True) + 64 * ref.U32 * (np.abs(g) * np.abs(want["out"])).sum(-1, keepdims=True)
    terms = (2 * ref.U16 * np.abs(ds) + p * dot) ** 2
    allowed = c.scale * np.sqrt(np.einsum("bhij,bhj->bhi", terms, (k ** 2).sum(-1)))
    if api:
        ctx.set_flags(omb.OM_TF32 | omb.OM_BF16_OPERANDS)
        try:
            t = {n: omb.Tensor.from_numpy(c.value[n], requires_grad=True) for n in "qkv"}
            out = omb.call("rule_attention", [t["q"], t["k"], t["v"]], ints=[1], floats=[0.0, 0.0])
            out.backward(omb.Tensor.from_numpy(c.value["g"]))
            got = t["q"].grad.numpy()
        finally:
            ctx.set_flags(0)
    else:
        c.run(False)
        n = c.value["q"].size
        rule, sizes = c.rule(), [i32(x) for x in c.dims] + [f32(c.scale)]
        w = lambda x: (c.where(x)[0], C.byref(c.where(x)[1]))   # noqa: E731
        out, dq = ctx.empty((n,)), ctx.empty((n,))
        ctx.call("om_rule_attention_fwd_bf16", ctx.handle, C.byref(rule), *w("q"), *w("k"), *w("v"), *sizes, out.ptr, None, w("o")[1], c.lse.ptr)
        ctx.call("om_rule_attention_bwd_bf16_out32", ctx.handle, C.byref(rule), *w("g"), *w("q"), *w("k"), *w("v"), out.ptr, w("o")[1], c.lse.ptr, *sizes,
                 dq.ptr, None, w("dq")[1], None, None, None, None, None, None)
        ctx.sync()
        got = dq.numpy().reshape(c.value["q"].shape)
    err = np.linalg.norm(got - want["dq"], axis=-1)
    over = err / (allowed + 1e-30)
    assert over[:, :, 1:].max() <= 2, (over[:, :, 1:].max(), over[:, :, 1:].argmax())


def test_results_whose_rows_overlap_are_refused(ctx):
    """Heads in each other's place, also where every stride is large enough by itself; heads between each other's rows are none of it."""
    r = np.random.default_rng(83)
    c = Call(ctx, r, 2, 2, 1, 3, 3, 8).run()
    w = lambda n: (c.where(n)[0], C.byref(c.where(n)[1]))   # noqa: E731
    room = ctx.zeros((4096,))
    freq = (C.c_double * 4)(*[0.5] * 4)

    def calls(strides):
        s, lse = omb.HeadStrides(*strides), c.lse.ptr
        sizes = [i32(n) for n in c.dims] + [f32(c.scale)]
        rule = c.rule()
        yield "om_rule_attention_fwd", [C.byref(rule), *w("q"), *w("k"), *w("v"), *sizes, room.ptr, C.byref(s), None]
        yield "om_rule_attention_bwd", [C.byref(rule), *w("g"), *w("q"), *w("k"), *w("v"), *w("o"), lse, *sizes, room.ptr, C.byref(s), None, None, None, None]
        yield "om_rotary", [*w("q"), None, C.c_int64(0), i32(0), i32(2), i32(2), i32(3), i32(8), freq, i32(4), i32(0), f32(1.0), i32(0), room.ptr, C.byref(s)]

    for strides in ((64, 8, 8), (64, 16, 8), (40, 24, 8), (16, 64, 16), (100, 12, 8), (64, 4, 16)):
        for name, args in calls(strides):
            with pytest.raises(omb.OmError) as e:
                ctx.call(name, ctx.handle, *args)
            assert e.value.status == 1, (name, strides)
    want = None
    for strides in ((48, 24, 8), (48, 8, 16), (8, 64, 16), (200, 24, 16), (24, 8, 64)):     # nested; heads or sequences between rows
        for name, args in calls(strides):
            ctx.call(name, ctx.handle, *args)
        ctx.sync()
        at = sum(np.arange(n).reshape([-1 if a == i else 1 for a in range(4)]) * s for i, (n, s) in enumerate(zip((2, 2, 3, 8), (*strides, 1))))
        got = room.numpy()[at]               # the last call's
        assert want is None or np.array_equal(got, want)
        want = got
