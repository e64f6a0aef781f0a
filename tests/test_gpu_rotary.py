"""Rotary positions through the C ABI and the tensor API against the rotation in 64 bits. An element is two products and a sum of values
whose cosines and sines are within 2^-22 (the angle's rounding to fp32 below an eighth of a turn, the series, the magnitude), so it is
off by at most 2^-21 (|x0| + |x1|) magnitude, and by half a bfloat16 step more in that type."""
import ctypes as C

import numpy as np
import pytest

import om_binding as omb
import rule_reference as ref
from om_binding import f32, i32, i64

pytestmark = pytest.mark.gpu


def check(got, x, positions, freq, adjacent, magnitude=1.0, inverse=False, half=False):
    want = ref.rotary(x, positions, freq, adjacent, magnitude, inverse)
    n = 2 * len(freq)
    pair = np.zeros_like(want)
    a = np.abs(x.astype(np.float64))
    both = (a[..., 0:n:2] + a[..., 1:n:2]) if adjacent else (a[..., : n // 2] + a[..., n // 2: n])
    if adjacent:
        pair[..., 0:n:2] = pair[..., 1:n:2] = both
    else:
        pair[..., : n // 2] = pair[..., n // 2: n] = both
    tol = 2.0 ** -21 * pair * abs(magnitude) + (ref.U16 if half else ref.U32) * np.abs(want) * (np.arange(x.shape[-1]) < n)
    assert (np.abs(got.astype(np.float64) - want) <= tol).all(), (np.abs(got - want) - tol).max()


def run(ctx, x, positions, freq, adjacent, magnitude=1.0, inverse=False, half=False, first=0, pad=0, in_place=False, layout="rows"):
    """x [B, H, L, D]; layout 'rows': [B, L, H, D + pad] on the device."""
    b, h, l, d = x.shape
    put = (lambda a: ctx.to_device(ref.to_bf16(a))) if half else (lambda a: ctx.to_device(np.ascontiguousarray(a, np.float32)))
    if layout == "rows":
        room = np.full((b, l, h, d + pad), 7.5, np.float32)
        room[..., :d] = x.transpose(0, 2, 1, 3)
        s = omb.HeadStrides(l * h * (d + pad), d + pad, h * (d + pad))
    else:
        room = np.full((b, h, l, d + pad), 7.5, np.float32)
        room[..., :d] = x
        s = omb.HeadStrides(h * l * (d + pad), l * (d + pad), d + pad)
    X = put(room)
    Y = X if in_place else put(np.full(room.shape, 7.5, np.float32))
    P = ctx.to_device(np.ascontiguousarray(positions, np.int32)) if positions is not None else None
    f = (C.c_double * len(freq))(*freq)
    ctx.call("om_rotary_bf16" if half else "om_rotary", ctx.handle, X.ptr, C.byref(s), P.ptr if P else None, i64(l if P and positions.ndim == 2 else 0),
             i32(first), i32(b), i32(h), i32(l), i32(d), f, i32(len(freq)), i32(adjacent), f32(magnitude), i32(inverse), Y.ptr, C.byref(s))
    out = Y.numpy()
    out = ref.from_bf16(out) if half else out
    assert (out[..., d:] == 7.5).all()       # what lies between the heads stays
    out = out[..., :d]
    return out.transpose(0, 2, 1, 3) if layout == "rows" else out


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("d,pairs,pad", [(2, 1, 0), (8, 3, 0), (32, 16, 0), (64, 32, 0), (64, 16, 0), (80, 40, 0), (96, 24, 0), (128, 64, 0), (256, 128, 0),
                                         (256, 100, 0), (64, 32, 1), (64, 13, 0), (72, 32, 8), (7, 2, 0)])
def test_widths_and_alignments(ctx, d, pairs, pad, adjacent, half):
    r = np.random.default_rng(d + pairs)
    x = r.standard_normal((2, 3, 5, d)).astype(np.float32)
    x = ref.from_bf16(ref.to_bf16(x)) if half else x
    positions = r.integers(0, 131072, (2, 5))
    freq = np.array(omb.rotary_frequencies(2 * pairs)[:pairs])
    for layout in ("rows", "heads"):
        check(run(ctx, x, positions, freq, adjacent, half=half, pad=pad, layout=layout), x, positions, freq, adjacent, half=half)
    check(run(ctx, x, positions, freq, adjacent, 1.25, True, half, pad=pad, in_place=True), x, positions, freq, adjacent, 1.25, True, half)


@pytest.mark.parametrize("b,h,l", [(1, 1, 1), (8, 12, 1), (1, 1, 3000), (3, 40, 257), (2, 1, 77)])
def test_sizes_and_default_positions(ctx, b, h, l):
    r = np.random.default_rng(l)
    x = r.standard_normal((b, h, l, 64)).astype(np.float32)
    freq = np.array(omb.rotary_frequencies(64)[:32])
    at = np.broadcast_to(np.arange(l) + 1000, (b, l))
    check(run(ctx, x, None, freq, False, first=1000), x, at, freq, False)
    one = np.arange(l)[::-1].copy()
    check(run(ctx, x, one, freq, True), x, np.broadcast_to(one, (b, l)), freq, True)


def test_far_and_negative_positions(ctx):
    r = np.random.default_rng(5)
    x = r.standard_normal((1, 2, 6, 32)).astype(np.float32)
    freq = np.array(omb.rotary_frequencies(32)[:16])
    at = np.array([[2 ** 31 - 1, -2 ** 31, 10 ** 9, -1, 0, 12345678]])
    got = run(ctx, x, at, freq, False)
    want = ref.rotary(x, at, freq, False)
    # A double product of 2^31 radians is off by 2^-22, in the oracle as in the kernel: a tolerance of 2^-20 instead of 2^-21.
    assert np.abs(got - want).max() <= 2.0 ** -20 * 2 * np.abs(x).max()


def test_turning_there_and_back(ctx):
    r = np.random.default_rng(6)
    x = r.standard_normal((2, 2, 50, 64)).astype(np.float32)
    freq = np.array(omb.rotary_frequencies(64)[:32])
    there = run(ctx, x, None, freq, False, 2.0)
    back = run(ctx, there, None, freq, False, 0.5, True)
    assert np.abs(back - x).max() <= 4 * 2.0 ** -21 * 2 * np.abs(x).max()


@pytest.mark.parametrize("flags", [0, omb.OM_TF32 | omb.OM_BF16_OPERANDS])
@pytest.mark.parametrize("heads_form", [False, True])
def test_tensor_api(ctx, flags, heads_form):
    ctx.set_flags(flags)
    try:
        r = np.random.default_rng(7)
        b, h, l, d = 2, 3, 11, 24
        a = r.standard_normal((b, h, l, d)).astype(np.float32)
        g = r.standard_normal((b, h, l, d)).astype(np.float32)
        at = r.integers(0, 5000, (b, l)).astype(np.int32)
        freq = np.array(omb.rotary_frequencies(16, 500.0, "parts", 8.0, 1024.0, 1.0, 4.0)[:8])
        shaped = lambda v: np.ascontiguousarray(v.transpose(0, 2, 1, 3).reshape(b, l, -1)) if heads_form else v   # noqa: E731
        whole = lambda v: v.reshape(b, l, h, d).transpose(0, 2, 1, 3) if heads_form else v                        # noqa: E731
        # A slice of a wider projection: read in place.
        wide = omb.Tensor.from_numpy(np.concatenate([shaped(a), shaped(a)], axis=2 if heads_form else 1), requires_grad=True)
        x = wide.slice(2, 0, h * d) if heads_form else wide.slice(1, 0, h)
        y = omb.call("rotary_heads" if heads_form else "rotary", [x, omb.Tensor.from_numpy(at)], ints=[16, 0, 0, 3, h], floats=[500.0, 8.0, 1024.0, 1.0, 4.0, 1.5])
        check(whole(y.numpy()), a, at, freq, False, 1.5)
        y.backward(omb.Tensor.from_numpy(shaped(g)))
        got = wide.grad.numpy()
        got, rest = (got[..., : h * d], got[..., h * d:]) if heads_form else (got[:, :h], got[:, h:])
        check(whole(got), g, at, freq, False, 1.5, True)
        assert (rest == 0).all()
    finally:
        ctx.set_flags(0)


def test_refusals(ctx):
    X = ctx.zeros((4096,))
    s = omb.HeadStrides(64, 16, 16)
    f = (C.c_double * 8)(*[0.5] * 8)

    def call(status, x=X.ptr, xs=s, ys=s, b=1, h=2, l=3, d=16, freq=f, pairs=8, magnitude=1.0, y=X.ptr):
        with pytest.raises(omb.OmError) as e:
            ctx.call("om_rotary", ctx.handle, x, C.byref(xs), None, i64(0), i32(0), i32(b), i32(h), i32(l), i32(d), freq, i32(pairs), i32(0), f32(magnitude),
                     i32(0), y, C.byref(ys))
        assert e.value.status == status, e.value

    call(1, b=-1)
    call(1, pairs=9)
    call(1, pairs=0)
    call(1, xs=omb.HeadStrides(64, 16, 15))
    call(1, ys=omb.HeadStrides(64, 8, 16), h=2)
    call(1, ys=omb.HeadStrides(128, 32, 16), h=2)          # in place with other strides
    call(8, x=None)
    call(8, freq=None)
    call(8, magnitude=float("inf"))
    call(8, freq=(C.c_double * 8)(*[float("nan")] * 8))
    x = omb.Tensor.from_numpy(np.zeros((1, 2, 3, 8), np.float32))
    with pytest.raises(omb.ShapeError):
        omb.call("rotary", [x, omb.Tensor.from_numpy(np.zeros((4,), np.int32))])
    with pytest.raises(omb.ShapeError):
        omb.call("rotary", [x, None], ints=[16])
    with pytest.raises(omb.ShapeError):
        omb.call("rotary_heads", [x, None], ints=[0, 0, 0, 0, 2])
