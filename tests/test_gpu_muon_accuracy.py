"""The digits of the Muon update: no more than four times what the same steps in fp32 leave off, which is what operands of 22 bits in place
of 24 amount to. fp32 is numpy's here, with the products of a BLAS."""
import numpy as np
import pytest

from test_gpu_muon import check, make, step

pytestmark = pytest.mark.gpu


def update(u, kind, steps=5):
    """X of the update u, everything in one precision."""
    x = u.T if u.shape[0] > u.shape[1] else u
    x = (x / np.linalg.norm(x)).astype(kind)
    a, b, c = (kind(v) for v in (3.4445, -4.7750, 2.0315))
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.T if u.shape[0] > u.shape[1] else x


def digits(got, u):
    """The error of an update and what it may be, both over |X|."""
    x = update(u, np.float64)
    n = np.linalg.norm(x)
    return np.linalg.norm(got - x) / n, 4 * np.linalg.norm(update(u, np.float32) - x) / n


@pytest.mark.parametrize("rows,cols", [(64, 64), (129, 131), (257, 255), (384, 384), (1536, 384), (384, 1536), (700, 1100), (31, 2000), (384, 6144), (64, 16384), (40, 65536)])
def test_digits(ctx, rows, cols):
    """Momentum 0 and no look-ahead: the update is the gradient itself. Sums of up to 65536 terms."""
    _, g, _ = make(np.random.default_rng(rows + cols), rows, cols)
    zero = np.zeros_like(g)
    p, _, _ = step(ctx, [(zero, g, zero)], lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False)[0]
    err, allowed = digits(-p.astype(np.float64) / (0.2 * np.sqrt(max(rows, cols))), g.astype(np.float64))
    assert err <= allowed, (err, allowed)


def test_digits_of_many_large_matrices_in_one_launch(ctx):
    """Every CTA has several tiles, of sums of different lengths, with edges off the tiles' everywhere."""
    r = np.random.default_rng(80)
    shapes = [(601, 777), (640, 650), (777, 601), (640, 1025), (530, 531), (900, 640), (636, 2049), (520, 768)] * 4
    mats = [(np.zeros(s, np.float32), make(r, *s)[1], np.zeros(s, np.float32)) for s in shapes]
    got = step(ctx, mats, lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False)
    for i in list(range(8)) + [31]:
        err, allowed = digits(-got[i][0].astype(np.float64) / (0.2 * np.sqrt(max(shapes[i]))), mats[i][1].astype(np.float64))
        assert err <= allowed, (shapes[i], err, allowed)


@pytest.mark.parametrize("size,eps", [(1e22, 1e-7), (1e35, 1e-7), (2e37, 1e-7), (1e-25, 1e-30), (1e-29, 1e-35)])
def test_updates_of_any_size(ctx, size, eps):
    """X depends on u / |u| alone, however large or small the squares of u are."""
    r = np.random.default_rng(81)
    for rows, cols in ((96, 160), (33, 7)):
        p, g, m = make(r, rows, cols, 1.0)
        mat = (p, (g * np.float32(size)).astype(np.float32), (m * np.float32(size)).astype(np.float32))
        check(step(ctx, [mat], eps=eps)[0], mat, eps=eps)


def test_an_update_of_zero_without_an_eps(ctx):
    """X is zero, not zero over zero: the weights decay and nothing else."""
    p = make(np.random.default_rng(82), 40, 70)[0]
    zero = np.zeros_like(p)
    got = step(ctx, [(p, zero, zero)], eps=0.0, lr=0.5)[0]
    assert np.abs(got[0] - 0.95 * p.astype(np.float64)).max() <= 2.0 ** -23 * np.abs(p).max() and (got[1] == 0).all()
