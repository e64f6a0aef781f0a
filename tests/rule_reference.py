"""The decoder operators in 64 bits on the CPU, for the tests of their kernels: written from the formulas, one (batch, head) at a time."""
import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -8          # half a step of fp32 and of bfloat16, relative


def to_bf16(a):
    """Rounded to nearest even, as uint16."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


def visible(b, lq, lk, causal=False, window=0, q_offset=0, prefix=None, q_docs=None, k_docs=None):
    pos, key = np.arange(lq)[:, None] + q_offset, np.arange(lk)[None, :]
    near = np.ones((lq, lk), bool)
    if causal:
        near &= key <= pos
    if window:
        near &= np.abs(pos - key) < window
    seen = np.broadcast_to(near, (b, lq, lk)).copy()
    if prefix is not None:
        seen |= (key[None] < np.asarray(prefix)[:, None, None])
    if q_docs is not None:
        seen &= (q_docs[:, :, None] == k_docs[:, None, :]) & (q_docs[:, :, None] >= 0)
    return seen


def attention(q, k, v, g, seen, scale, softcap=0.0, slopes=None, q_offset=0, half=False, planes=False):
    """Output, log-sum-exp and gradients of [B, H, L, D] arrays, and how far each may be off: with fp32 arithmetic (half False), or
    with bfloat16 operands, where every weight, every score gradient, the saved output and each result is rounded once.

    planes: fp32 calls that are done with two half-precision numbers a value. Such a pair is within 2^-22 of its value, and the product of
    two pairs leaves out 2^-22 more, 12 * 2^-24 of a product in all: less than the 4 sqrt(d) * 2^-24 that a sum of d products is allowed
    here. What the smallest half, 2^-24, adds: 2^-25 (half a step) of a value's unit, where units put the largest operand of a head group at
    2^14 or more, weights of the forward at 2^7 for the row's largest, weights of the backward at 2^14 for one, and the scores' gradients'
    bound 2 |g| |v| at 2^14 or more (their largest rows' norms)."""
    q, k, v, g = (np.asarray(a, np.float64) for a in (q, k, v, g))
    (b, h, lq, d), (hk, lk) = q.shape, k.shape[1:3]
    r = {n: np.zeros_like(a) for n, a in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: np.zeros_like(a) for n, a in r.items()}
    r["lse"] = np.full((b, h, lq), -np.inf)
    far = np.abs(np.arange(lq)[:, None] + q_offset - np.arange(lk)[None, :])
    for n in range(b):
        for i in range(h):
            j = i // (h // hk)
            s = scale * q[n, i] @ k[n, j].T
            # Rounding of a score: d products summed as a random walk (four deviations), and of what is done to it behind.
            ds_err = 4 * U32 * (np.sqrt(d) * abs(scale) * (np.abs(q[n, i]) @ np.abs(k[n, j]).T) + 4 * np.abs(s) + 4 * softcap)
            cap = np.ones_like(s)
            if softcap:
                t = np.tanh(s / softcap)
                s, cap = softcap * t, 1 - t * t
            if slopes is not None:
                s = s - slopes[i] * far
                ds_err = ds_err + 2 * U32 * slopes[i] * far
            m = seen[n]
            if not m.any():
                continue
            s = np.where(m, s, -np.inf)
            top = np.max(s, axis=1, initial=-np.inf)
            base = np.where(np.isfinite(top), top, 0.0)
            e = np.exp(s - base[:, None])
            total = e.sum(1)
            some = total > 0
            p = e / np.where(some, total, 1.0)[:, None]
            r["lse"][n, i][some] = (base + np.log(np.where(some, total, 1.0)))[some]
            o = p @ v[n, j]
            r["out"][n, i] = o
            dp = g[n, i] @ v[n, j].T
            dot = (g[n, i] * o).sum(1, keepdims=True)
            z = p * (dp - dot) * cap
            r["dq"][n, i] = scale * z @ k[n, j]
            r["dk"][n, j] += scale * z.T @ q[n, i]
            r["dv"][n, j] += p.T @ g[n, i]
            # Relative error of a weight: its score's, the row maximum's share of it, the exponential's and the sum's.
            err = np.where(m, ds_err, 0.0)
            if planes:
                mine = slice(j * (h // hk), (j + 1) * (h // hk))
                top = {x: np.abs(a).max() for x, a in (("q", q[n, mine]), ("k", k[n, j]), ("v", v[n, j]), ("g", g[n, mine]))}
                norm = {x: np.sqrt((a * a).sum(-1).max()) for x, a in (("v", v[n, j]), ("g", g[n, mine]))}
                low = 2.0 ** -39
                err = err + np.where(m, 2 * abs(scale) * low * (np.abs(q[n, i]).sum(1)[:, None] * top["k"] + np.abs(k[n, j]).sum(1)[None, :] * top["q"]), 0.0)
            w = err + err.max(1, keepdims=True) + U32 * (8 + 4 * np.sqrt(lk) + 4 * np.abs(np.where(m, s, 0.0)).max(1, keepdims=True))
            u = U16 if half else 0.0
            pe = p * (w + u)
            tol["out"][n, i] = pe @ np.abs(v[n, j]) + (u + 4 * U32) * np.abs(o)
            # The row dot comes from the output as it was stored.
            dot_err = (np.abs(g[n, i]) * (tol["out"][n, i] + u * np.abs(o))).sum(1, keepdims=True) + 4 * U32 * np.sqrt(d) * (np.abs(g[n, i] * o)).sum(1, keepdims=True)
            dp_err = 4 * U32 * np.sqrt(d) * (np.abs(g[n, i]) @ np.abs(v[n, j]).T)
            ze = np.abs(z) * (w + u + 8 * U32) + p * (dot_err + dp_err) + p * np.abs(dp - dot) * (8 * U32 * (1 + np.abs(cap)))
            tol["dq"][n, i] = abs(scale) * ze @ np.abs(k[n, j]) + 4 * U32 * np.sqrt(lk) * abs(scale) * np.abs(z) @ np.abs(k[n, j])
            tol["dk"][n, j] += abs(scale) * ze.T @ np.abs(q[n, i]) + 4 * U32 * np.sqrt(lq) * abs(scale) * np.abs(z).T @ np.abs(q[n, i])
            tol["dv"][n, j] += pe.T @ np.abs(g[n, i]) + 4 * U32 * np.sqrt(lq) * p.T @ np.abs(g[n, i])
            if planes:
                ds_low = 2.0 ** -38 * norm["g"] * norm["v"]
                dp_low = 2 * low * (np.abs(g[n, i]).sum(1)[:, None] * top["v"] + np.abs(v[n, j]).sum(1)[None, :] * top["g"])
                tol["out"][n, i] += 2.0 ** -32 * p.max(1, keepdims=True) * (m @ np.abs(v[n, j])) + low * top["v"]
                tol["dv"][n, j] += low * (m.T @ np.abs(g[n, i])) + low * top["g"] * p.sum(0)[:, None]
                ze = p * dp_low + ds_low * m
                tol["dq"][n, i] += abs(scale) * (ze @ np.abs(k[n, j]) + low * top["k"] * np.abs(z).sum(1)[:, None])
                tol["dk"][n, j] += abs(scale) * (ze.T @ np.abs(q[n, i]) + low * top["q"] * np.abs(z).sum(0)[:, None])
    for n in ("dq", "dk", "dv"):
        tol[n] += (U16 if half else U32) * np.abs(r[n])
    return r, {n: t + 1e-30 for n, t in tol.items()}


def rotary(x, positions, inv_freq, adjacent, magnitude=1.0, inverse=False):
    """[B, H, L, D] turned; positions [B, L]."""
    x = np.asarray(x, np.float64)
    n = len(inv_freq)
    angle = np.asarray(positions, np.float64)[:, None, :, None] * np.asarray(inv_freq)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if inverse else 1)
    y = x.copy()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if adjacent else (x[..., :n], x[..., n:2 * n])
    if adjacent:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * c - b * s, a * s + b * c
    else:
        y[..., :n], y[..., n:2 * n] = a * c - b * s, a * s + b * c
    return y


def muon(p, g, m, lr, momentum, weight_decay, eps, nesterov, steps, match_rms, grad_scale=1.0):
    """New weights, new momentum, and the orthogonalised update."""
    p, g, m = np.asarray(p, np.float64), np.asarray(g, np.float64) * grad_scale, np.asarray(m, np.float64)
    m = momentum * m + (1 - momentum) * g
    u = momentum * m + (1 - momentum) * g if nesterov else m
    x = u / max(np.linalg.norm(u), eps)
    for _ in range(steps):
        if x.shape[0] <= x.shape[1]:
            a = x @ x.T
            x = 3.4445 * x + (-4.7750 * a + 2.0315 * a @ a) @ x
        else:
            a = x.T @ x
            x = 3.4445 * x + x @ (-4.7750 * a + 2.0315 * a @ a)
    r, c = p.shape
    s = 0.2 * np.sqrt(max(r, c)) if match_rms else np.sqrt(max(1.0, r / c))
    return p * (1 - lr * weight_decay) - lr * s * x, m, x
