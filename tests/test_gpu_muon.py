"""The Muon update through the C ABI and the optimizer against the formulas in 64 bits.

Tolerance of the orthogonalised update X, in the Frobenius norm: a product of operands of 22 significant bits and fp32 sums is within
2^-20 of its value there (a random walk over the terms of a sum, with room), a step has three of them, and a step multiplies an
error in the direction of a small singular value by at most 3.4445: 3 * 2^-20 * (1 + 3.4445 + ... + 3.4445^4) < 4.5e-4 of |X|.
The weights add their own rounding, two steps of 2^-24 of |p|."""
import ctypes as C

import numpy as np
import pytest

import om_binding as omb
import rule_reference as ref
from om_binding import i32

pytestmark = pytest.mark.gpu
BF16 = omb.OM_TF32 | omb.OM_BF16_OPERANDS
DEFAULT = dict(lr=0.02, momentum=0.95, weight_decay=0.1, eps=1e-7, nesterov=True, steps=5, match_rms=True)


def step(ctx, mats, half=False, device_hyper=False, **change):
    """mats: (p, g, m) arrays; one call for all. Returns the new (p, m, p16)."""
    h = DEFAULT | change
    hyper = omb.MuonHyper(grad_scale=h.get("grad_scale", 1.0), **{k: (int(v) if isinstance(v, bool) else v) for k, v in h.items() if k != "grad_scale"})
    n = len(mats)
    dev = [[ctx.to_device(a) for a in mat] for mat in mats]
    p16 = [ctx.zeros(mat[0].shape, np.uint16) for mat in mats] if half else None
    lists = [(C.c_void_p * n)(*[d[i].ptr.value for d in dev]) for i in range(3)]
    hd = ctx.to_device(np.frombuffer(bytes(hyper), np.uint8).copy()) if device_hyper else None
    if device_hyper:
        hyper = omb.MuonHyper(steps=h["steps"])
    ctx.call("om_optim_muon_step", ctx.handle, i32(n), *lists, (C.c_void_p * n)(*[a.ptr.value for a in p16]) if half else None,
             omb.int_array([mat[0].shape[0] for mat in mats]), omb.int_array([mat[0].shape[1] for mat in mats]), C.byref(hyper), hd.ptr if hd else None)
    ctx.sync()
    return [(d[0].numpy(), d[2].numpy(), p16[i].numpy() if half else None) for i, d in enumerate(dev)]


def make(r, rows, cols, size=1e-3):
    return tuple((s * r.standard_normal((rows, cols))).astype(np.float32) for s in (0.02, size, size))


def check(got, mat, **change):
    h = DEFAULT | change
    p, m, x = ref.muon(*mat, **h)
    rows, cols = mat[0].shape
    rate = h["lr"] * (0.2 * np.sqrt(max(rows, cols)) if h["match_rms"] else np.sqrt(max(1.0, rows / cols)))
    gs = abs(h.get("grad_scale", 1.0))
    assert np.abs(got[1] - m).max() <= 4 * ref.U32 * (np.abs(mat[2]).max() + gs * np.abs(mat[1]).max())
    allowed = rate * 4.5e-4 * np.linalg.norm(x) + 4 * ref.U32 * np.linalg.norm(mat[0])
    assert np.linalg.norm(got[0] - p) <= allowed, (np.linalg.norm(got[0] - p), allowed)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2), (2, 1), (1, 700), (700, 1), (2, 3), (8, 8), (31, 33), (33, 31), (64, 64), (65, 63), (127, 128), (128, 128), (129, 131),
                                       (128, 256), (256, 128), (257, 255), (100, 1000), (1000, 100), (384, 1536), (520, 520), (7, 4099)])
def test_shapes(ctx, rows, cols):
    mat = make(np.random.default_rng(rows * 7 + cols), rows, cols)
    check(step(ctx, [mat])[0], mat)


def test_large(ctx):
    mat = make(np.random.default_rng(1), 2048, 1024)
    check(step(ctx, [mat])[0], mat)


@pytest.mark.parametrize("change", [dict(nesterov=False), dict(momentum=0.0), dict(weight_decay=0.0), dict(steps=1), dict(steps=3), dict(match_rms=False), dict(grad_scale=0.25),
                                    dict(lr=0.0)])
def test_numbers(ctx, change):
    for rows, cols in ((40, 90), (90, 40)):
        mat = make(np.random.default_rng(4), rows, cols)
        check(step(ctx, [mat], **change)[0], mat, **change)
        check(step(ctx, [mat], device_hyper=True, **change)[0], mat, **change)


def test_many_matrices_in_one_call(ctx):
    r = np.random.default_rng(5)
    shapes = [(int(r.integers(1, 200)), int(r.integers(1, 200))) for _ in range(75)] + [(64, 64)] * 5 + [(0, 5), (300, 20)]
    mats = [make(r, *s) for s in shapes]
    got = step(ctx, mats, half=True)
    alone = [step(ctx, [m], half=True)[0] for m in mats[::9]]
    for g, m in zip(got, mats):
        if m[0].size:
            check(g, m)
            assert np.array_equal(g[2], ref.to_bf16(g[0]))
    for a, b in zip(alone, got[::9]):        # a matrix's update does not depend on what else is in the call
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_scale_of_the_gradient_does_not_matter(ctx):
    """X depends on u / |u| only: gradients of 1e-12 and of 1e6 give the same update (as long as |u| is above eps)."""
    r = np.random.default_rng(6)
    p, g, m = make(r, 96, 160, 1.0)
    for size in (1e-6, 1e6):
        mat = (p, (g * size).astype(np.float32), (m * size).astype(np.float32))
        check(step(ctx, [mat], eps=1e-12)[0], mat, eps=1e-12)


def test_zero_and_low_rank_updates(ctx):
    r = np.random.default_rng(7)
    p = make(r, 70, 130)[0]
    zero = np.zeros_like(p)
    got = step(ctx, [(p, zero, zero)])[0]
    assert np.array_equal(got[1], zero) and np.allclose(got[0], p * (1 - 0.02 * 0.1), rtol=1e-6, atol=0)
    u, v = r.standard_normal((70, 2)), r.standard_normal((2, 130))
    mat = (p, (u @ v).astype(np.float32), zero)
    x, want = step(ctx, [mat], weight_decay=0.0)[0][0], ref.muon(*mat, **(DEFAULT | dict(weight_decay=0.0)))[0]
    # Rank two: directions that the matrix does not have hold rounding noise of 2^-22, which five steps raise by at most 3.4445^5.
    rate = 0.02 * 0.2 * np.sqrt(130)
    assert np.linalg.norm(x - want) <= rate * 3.4445 ** 5 * 2.0 ** -20 * np.sqrt(70 * 130)


def test_not_a_number_stays_in_its_matrix(ctx):
    r = np.random.default_rng(8)
    good, bad = make(r, 50, 60), make(r, 50, 60)
    bad[1][3, 4] = np.nan
    got = step(ctx, [good, bad, good])
    check(got[0], good)
    check(got[2], good)
    assert np.isnan(got[1][0]).any()


def test_same_bits_twice(ctx):
    mat = make(np.random.default_rng(9), 300, 500)
    a, b = step(ctx, [mat])[0], step(ctx, [mat])[0]
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_captured_step_follows_its_numbers_on_the_device(ctx):
    r = np.random.default_rng(10)
    p, g, m = make(r, 90, 150)
    P, G, M = (ctx.to_device(a) for a in (p, g, m))
    hyper = omb.MuonHyper(**(DEFAULT | dict(grad_scale=1.0)))
    H = ctx.to_device(np.frombuffer(bytes(hyper), np.uint8).copy())
    one = lambda a: (C.c_void_p * 1)(a.ptr.value)   # noqa: E731
    graph = C.c_void_p()
    ctx.call("om_graph_begin", ctx.handle)
    ctx.call("om_optim_muon_step", ctx.handle, i32(1), one(P), one(G), one(M), None, omb.int_array([90]), omb.int_array([150]), C.byref(hyper), H.ptr)
    ctx.call("om_graph_end", ctx.handle, C.byref(graph))
    for lr in (0.02, 0.005):
        new = omb.MuonHyper(**(DEFAULT | dict(grad_scale=1.0, lr=lr)))
        ctx.call("om_memcpy_h2d", ctx.handle, H.ptr, C.byref(new), C.c_size_t(C.sizeof(new)))
        ctx.call("om_graph_launch", ctx.handle, graph)
        ctx.sync()
        check((P.numpy(), M.numpy()), (p, g, m), lr=lr)
        p, m = P.numpy(), M.numpy()
    ctx.call("om_graph_destroy", ctx.handle, graph)


def test_workspaces_under_the_checked_flag(ctx):
    """Poisoned workspaces with guard bytes behind them: nothing is read that was not written, nothing written behind an end."""
    ctx.set_flags(omb.OM_CHECKED)
    try:
        r = np.random.default_rng(31)
        mats = [make(r, *s) for s in ((33, 65), (129, 31), (257, 130), (1, 5))]
        for got, mat in zip(step(ctx, mats), mats):
            check(got, mat)
    finally:
        ctx.set_flags(0)


def test_refusals(ctx):
    A = ctx.zeros((16,))
    one = (C.c_void_p * 1)(A.ptr.value)
    none = (C.c_void_p * 1)(None)

    def call(status, n=1, p=one, g=one, m=one, rows=4, cols=4, hyper=omb.MuonHyper(**(DEFAULT | dict(grad_scale=1.0)))):
        with pytest.raises(omb.OmError) as e:
            ctx.call("om_optim_muon_step", ctx.handle, i32(n), p, g, m, None, omb.int_array([rows]), omb.int_array([cols]), C.byref(hyper) if hyper else None, None)
        assert e.value.status == status

    call(8, n=-1)
    call(8, p=None)
    call(8, g=none)
    call(8, hyper=None)
    call(8, hyper=omb.MuonHyper(steps=0))
    call(8, hyper=omb.MuonHyper(steps=11))
    call(1, rows=-1)
    call(1, cols=65537)
    call(8)                                                # one memory for everything
    at = lambda *n: (C.c_void_p * len(n))(*[A.ptr.value + 4 * x for x in n])   # noqa: E731
    big = ctx.zeros((64,))
    on = lambda *n: (C.c_void_p * len(n))(*[big.ptr.value + 4 * x for x in n])   # noqa: E731
    for p, g, m in ((on(0, 0), on(16, 16), on(32, 48)), (on(0, 15), on(32, 32), on(40, 48)), (on(0, 16), on(8, 48), on(32, 56))):
        with pytest.raises(omb.OmError) as e:
            ctx.call("om_optim_muon_step", ctx.handle, i32(2), p, g, m, None, omb.int_array([2, 2]), omb.int_array([8, 4]),
                     C.byref(omb.MuonHyper(**(DEFAULT | dict(grad_scale=1.0)))), None)
        assert e.value.status == 8
    ctx.call("om_optim_muon_step", ctx.handle, i32(2), on(0, 16), at(0, 0), on(32, 48), None, omb.int_array([2, 2]), omb.int_array([8, 8]),
             C.byref(omb.MuonHyper(**(DEFAULT | dict(grad_scale=1.0)))), None)                     # one gradient for two matrices
    ctx.sync()
    t = lambda *s: omb.Tensor.from_numpy(np.zeros(s, np.float32), requires_grad=True)   # noqa: E731
    with pytest.raises(omb.ShapeError):
        omb.Optimizer.muon([t(3)])
    with pytest.raises(omb.IndexOutOfRange):
        omb.Optimizer.muon([t(3, 3)], momentum=1.0)
    with pytest.raises(omb.IndexOutOfRange):
        omb.Optimizer.muon([t(3, 3)], steps=0)


@pytest.mark.parametrize("flags", [0, BF16])
def test_a_decoder_layer_trains(ctx, flags):
    """The operators together, as a decoder's training step uses them: packed projections turned by position, attention by rule
    over shared key heads and packed documents, a loss, and the matrices updated by Muon while the vectors go to AdamW. The
    gradients are those of the same composition in 64 bits, and the first update is the formula's on the gradients found."""
    import torch
    ctx.set_flags(flags)
    try:
        r = np.random.default_rng(12)
        b, l, width, h, hk, d = 2, 48, 64, 4, 2, 16
        docs = np.repeat(np.array([[0] * 20 + [1] * 22 + [-1] * 6, [0] * 48], np.int32), 1, axis=0)
        rnd = lambda s: ref.from_bf16(ref.to_bf16(r.standard_normal(s).astype(np.float32) * 0.3))   # noqa: E731
        values = dict(q=rnd((h * d, width)), k=rnd((hk * d, width)), v=rnd((hk * d, width)), o=rnd((width, h * d)), bias=rnd((width,)))
        x = rnd((b, l, width))
        target = r.integers(0, width, (b * l,)).astype(np.int64)
        w = {n: omb.Tensor.from_numpy(a, requires_grad=True) for n, a in values.items()}
        matrices = [w[n] for n in ("q", "k", "v", "o")]
        muon = omb.Optimizer.muon(matrices, lr=0.01)
        adam = omb.Optimizer.adamw([w["bias"]], lr=0.01)
        X, D = omb.Tensor.from_numpy(x), omb.Tensor.from_numpy(docs)

        def loss():
            q = omb.call("rotary_heads", [omb.call("linear", [X, w["q"], None]), None], ints=[0, 0, 0, 0, h])
            k = omb.call("rotary_heads", [omb.call("linear", [X, w["k"], None]), None], ints=[0, 0, 0, 0, hk])
            a = omb.call("rule_attention_heads", [q, k, omb.call("linear", [X, w["v"], None]), None, D, D], ints=[1, 0, 0, h, hk])
            y = omb.call("linear", [a, w["o"], w["bias"]])
            return omb.call("cross_entropy", [y.reshape(b * l, width), omb.Tensor.from_numpy(target)], ints=[1, -100])

        first = loss()
        muon.zero_grad()
        adam.zero_grad()
        first.backward()
        grads = {n: t.grad.numpy() for n, t in w.items()}

        t = {n: torch.tensor(a.astype(np.float64), requires_grad=True) for n, a in values.items()}
        freq = torch.tensor(np.array(omb.rotary_frequencies(d)[: d // 2]))
        ang = torch.arange(l, dtype=torch.float64)[:, None] * freq

        def turn(z, heads):
            z = z.reshape(b, l, heads, d).transpose(1, 2)
            lo, hi = z[..., : d // 2], z[..., d // 2:]
            return torch.cat([lo * ang.cos() - hi * ang.sin(), lo * ang.sin() + hi * ang.cos()], -1)

        xt = torch.tensor(x.astype(np.float64))
        q, k = turn(xt @ t["q"].T, h), turn(xt @ t["k"].T, hk).repeat_interleave(h // hk, 1)
        v = (xt @ t["v"].T).reshape(b, l, hk, d).transpose(1, 2).repeat_interleave(h // hk, 1)
        seen = torch.tensor(ref.visible(b, l, l, True, 0, 0, None, docs, docs))[:, None]
        s = (q @ k.transpose(2, 3) * d ** -0.5).masked_fill(~seen, -1e300)
        a = (torch.softmax(s, -1) * seen) @ v
        y = a.transpose(1, 2).reshape(b, l, h * d) @ t["o"].T + t["bias"]
        want = torch.nn.functional.cross_entropy(y.reshape(b * l, width), torch.tensor(target))
        want.backward()
        # fp32: chains of some hundred roundings of 2^-24. bfloat16: the operands of six products and the weights of the softmax
        # round by 2^-8 each, errors that are independent and so add up as a root: 2^-8 sqrt(10) with a factor of two of room.
        rel = 2.0 ** -8 * np.sqrt(10) * 2 if flags else 1e-5
        assert abs(first.item() - want.item()) <= rel * want.item()
        for n, g in grads.items():
            exact = t[n].grad.numpy()
            assert np.linalg.norm(g - exact) <= rel * np.linalg.norm(exact), (n, np.linalg.norm(g - exact) / np.linalg.norm(exact))

        muon.step()
        adam.step()
        for n in ("q", "k", "v", "o"):
            check((w[n].numpy(), 0.05 * grads[n]), (values[n], grads[n], np.zeros_like(grads[n])), lr=0.01)
        for _ in range(3):
            now = loss()
            muon.zero_grad()
            adam.zero_grad()
            now.backward()
            muon.step()
            adam.step()
        assert np.isfinite(now.item())
    finally:
        ctx.set_flags(0)
