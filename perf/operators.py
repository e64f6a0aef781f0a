"""Performance cases of the decoder training operators: rotary positions, attention by rule, and the Muon update.

A *rotary* pass turns the heads of an activation by the angles of their tokens' positions, or a gradient back by them. An
*attention* pass is a forward, alone or with its backward, of attention whose mask, bias and cap follow from a rule
(causal, window, prefix, documents, distance slopes, tanh cap) instead of a stored matrix; query heads may share key heads.
A *muon* pass updates a list of weight matrices by their orthogonalised momentum. Activations are addressed in place inside
the packed projection [batch, length, heads * width] that a program has them in.

Where `own` is false the operators are computed by elementary torch operations in fp32, the angles of positions in fp64.
"""
import ctypes as C
import math
import os
import random
import sys

import torch

own = False
_ctx = None


def _framework():
    """The package and the process's one device context."""
    global _ctx
    package = os.path.join(os.getcwd(), "onemodel-csharp_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import om_binding as omb
    if _ctx is None:
        _ctx = omb.Context(0, omb.OM_TF32 | omb.OM_BF16_OPERANDS)
    return omb, _ctx


def listed():
    return [
        # The smallest call: the query heads of one new token in each of 8 sequences, adjacent pairs, fp32.
        {"name": "rotary-token-fp32", "kind": "rotary", "type": "fp32", "batch": 8, "length": 1, "heads": 12, "others": 24, "width": 64,
         "turned": 64, "adjacent": True, "back": False, "reach": 4096, "factor": 1.0},
        # The gradient of a key projection at an odd length, the first 48 of 96 columns turned, halves paired.
        {"name": "rotary-odd-fp32-back", "kind": "rotary", "type": "fp32", "batch": 3, "length": 1021, "heads": 5, "others": 0, "width": 96,
         "turned": 48, "adjacent": False, "back": True, "reach": 1021, "factor": 1.0},
        # The query and key heads of a packed bfloat16 projection over a long context, frequencies stretched by parts.
        {"name": "rotary-packed-bf16", "kind": "rotary", "type": "bf16", "batch": 8, "length": 4096, "heads": 40, "others": 8, "width": 128,
         "turned": 128, "adjacent": False, "back": False, "reach": 131072, "factor": 16.0},
        # A small model's step in the exact tier: a causal mask and distance slopes.
        {"name": "attention-small-fp32", "kind": "attention", "type": "fp32", "batch": 2, "heads": 4, "shared": 4, "queries": 64, "keys": 64, "width": 32,
         "causal": True, "window": 0, "prefix": 0, "cap": 0.0, "slopes": True, "document": 0, "padded": 0, "back": True},
        # Training in the exact tier at the encoder configuration's heads and a decoder's length.
        {"name": "attention-train-fp32", "kind": "attention", "type": "fp32", "batch": 4, "heads": 12, "shared": 12, "queries": 1024, "keys": 1024, "width": 64,
         "causal": True, "window": 0, "prefix": 0, "cap": 0.0, "slopes": False, "document": 0, "padded": 0, "back": True},
        # Packed documents of uneven length with a padded tail, capped scores, two query heads a key head, bfloat16.
        {"name": "attention-documents-bf16", "kind": "attention", "type": "bf16", "batch": 3, "heads": 10, "shared": 5, "queries": 1531, "keys": 1531, "width": 64,
         "causal": True, "window": 0, "prefix": 0, "cap": 30.0, "slopes": False, "document": 300, "padded": 57, "back": True},
        # The largest attention: long sequences, four query heads a key head, forward and backward.
        {"name": "attention-train-bf16", "kind": "attention", "type": "bf16", "batch": 4, "heads": 16, "shared": 4, "queries": 4096, "keys": 4096, "width": 128,
         "causal": True, "window": 0, "prefix": 0, "cap": 0.0, "slopes": False, "document": 0, "padded": 0, "back": True},
        # Evaluation of long texts: a window, a prefix that everything sees, distance slopes; forward only.
        {"name": "attention-window-bf16", "kind": "attention", "type": "bf16", "batch": 2, "heads": 12, "shared": 12, "queries": 8192, "keys": 8192, "width": 64,
         "causal": True, "window": 1024, "prefix": 200, "cap": 0.0, "slopes": True, "document": 0, "padded": 0, "back": False},
        # One new token of each sequence against a long context: few rows, many keys; forward only.
        {"name": "attention-token-bf16", "kind": "attention", "type": "bf16", "batch": 8, "heads": 32, "shared": 8, "queries": 1, "keys": 8191, "width": 128,
         "causal": True, "window": 0, "prefix": 0, "cap": 0.0, "slopes": False, "document": 0, "padded": 0, "back": False},
        # Two small matrices of odd sizes: launches are what it costs.
        {"name": "muon-small", "kind": "muon", "shapes": "33x65,129x31", "momentum": 0.95, "nesterov": True, "decay": 0.0},
        # The weight matrices of four layers of the encoder of width 384.
        {"name": "muon-encoder", "kind": "muon", "shapes": ",".join(["384x384"] * 16 + ["1536x384"] * 4 + ["384x1536"] * 4), "momentum": 0.95,
         "nesterov": True, "decay": 0.1},
        # The matrices of one wide layer, the largest work of all.
        {"name": "muon-wide", "kind": "muon", "shapes": "4096x4096,1000x4096,4096x1000", "momentum": 0.9, "nesterov": False, "decay": 0.01},
    ]


def _log(rng, low, high):
    """A whole number from [low, high], evenly spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "muon"])
    if kind == "rotary":
        width = rng.choice([32, 64, 80, 96, 128])
        heads = _log(rng, 1, 40)
        length = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(16, 16384 // length)))
        return {"kind": kind, "type": rng.choice(["fp32", "bf16"]), "batch": batch, "length": length, "heads": heads, "others": rng.choice([0, 0, heads, 8]),
                "width": width, "turned": width if rng.random() < 0.6 else 2 * rng.randint(1, width // 2), "adjacent": rng.random() < 0.5,
                "back": rng.random() < 0.4, "reach": _log(rng, max(length, 16), 131072), "factor": rng.choice([1.0, 1.0, 4.0, 16.0])}
    if kind == "attention":
        kind_type = rng.choice(["fp32", "bf16", "bf16"])
        shared = rng.choice([1, 2, 3, 4, 8])
        heads = shared * rng.choice([1, 1, 2, 4])
        keys = _log(rng, 1, 6000)
        queries = rng.choice([keys, keys, keys, 1, rng.randint(1, keys)])
        most = 1_000_000_000 if kind_type == "bf16" else 60_000_000
        batch = _log(rng, 1, max(1, min(16, most // (heads * queries * keys))))
        while batch * heads * queries * keys > most:
            keys = max(1, keys // 2)
            queries = min(queries, keys)
        causal = rng.random() < 0.75
        document = rng.choice([0, 0, _log(rng, 4, 1000)])
        return {"kind": kind, "type": kind_type, "batch": batch, "heads": heads, "shared": shared, "queries": queries, "keys": keys,
                "width": rng.choice([32, 64, 64, 80, 96, 128]), "causal": causal, "window": rng.choice([0, 0, _log(rng, 1, keys)]),
                "prefix": rng.choice([0, 0, rng.randint(1, keys)]) if causal else 0, "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "slopes": rng.random() < 0.3,
                "document": document, "padded": rng.randint(0, keys // 4) if document else 0, "back": rng.random() < 0.7}
    shapes, left = [], 1.0e12
    for _ in range(rng.randint(1, 6)):
        r, c = _log(rng, 8, 4096), _log(rng, 8, 4096)
        while _products((r, c)) > left:
            r, c = max(8, r // 2), max(8, c // 2)
            if r * c <= 64:
                break
        again = rng.choice([1, 1, 2, 4])
        while again > 1 and again * _products((r, c)) > left:
            again -= 1
        left -= again * _products((r, c))
        shapes += ["%dx%d" % (r, c)] * again
    return {"kind": kind, "shapes": ",".join(shapes), "momentum": rng.choice([0.9, 0.95]), "nesterov": rng.random() < 0.5, "decay": rng.choice([0.0, 0.1])}


# ---- what follows from a case alone -------------------------------------------------------------------------------------

A, B, CC = 3.4445, -4.7750, 2.0315   # the quintic of the orthogonalisation
STEPS, EPS, RATE = 5, 1e-7, 2e-3


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _products(shape):
    """Multiplications and additions of one matrix's products over all steps; those of a symmetric result are needed for half of it."""
    m, n = min(shape), max(shape)
    return STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def _frequencies(case):
    """Radians a position of every turned pair; a factor above 1 stretches the slow ones for contexts that much longer than 8192."""
    found = []
    for j in range(case["turned"] // 2):
        f = 10000.0 ** (-2.0 * j / case["turned"])
        if case["factor"] > 1:
            kept = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
            f *= (1 - kept) / case["factor"] + kept
        found.append(f)
    return found


def _magnitude(case):
    return 1.0 if case["factor"] <= 1 else 0.1 * math.log(case["factor"]) + 1.0


def _documents(case, row):
    """The document of every key of one sequence: uneven lengths around the case's, -1 where the tail is padding."""
    r = random.Random(1000 * row + case["document"])
    ids, doc = [], 0
    while len(ids) < case["keys"] - case["padded"]:
        ids += [doc] * max(1, int(case["document"] * r.uniform(0.3, 1.7)))
        doc += 1
    return ids[: case["keys"] - case["padded"]] + [-1] * case["padded"]


def _visible(case, device):
    """Which keys each query sees: [batch or 1, queries, keys]."""
    at = torch.arange(case["queries"], device=device) + case["keys"] - case["queries"]
    far = at[:, None] - torch.arange(case["keys"], device=device)[None, :]
    seen = torch.ones_like(far, dtype=torch.bool)
    if case["causal"]:
        seen = seen & (far >= 0)
    if case["window"]:
        seen = seen & (far.abs() < case["window"])
    if case["prefix"]:
        seen = seen | (torch.arange(case["keys"], device=device) < case["prefix"])[None, :]
    seen = seen[None]
    if case["document"]:
        ids = torch.tensor([_documents(case, r) for r in range(case["batch"])], device=device)
        mine = ids[:, case["keys"] - case["queries"]:]
        seen = seen & (mine[:, :, None] == ids[:, None, :]) & (mine >= 0)[:, :, None]
    return seen


def work(case):
    if case["kind"] == "rotary":
        n = case["batch"] * case["length"] * case["heads"] * case["turned"]
        size = 4 if case["type"] == "fp32" else 2
        whole = case["batch"] * case["length"] * case["heads"] * case["width"]
        return {"bytes": 2 * size * whole + 4 * case["batch"] * case["length"], "flops": 3 * n}
    if case["kind"] == "attention":
        seen = _visible(case, "cuda" if torch.cuda.is_available() else "cpu")
        pairs = int(seen.sum()) * (case["batch"] // seen.shape[0]) * case["heads"]
        size = 4 if case["type"] == "fp32" else 2
        q = case["batch"] * case["heads"] * case["queries"] * case["width"]
        k = case["batch"] * case["shared"] * case["keys"] * case["width"]
        # Forward: q, k, v in, the output out. Backward: those four and the output's gradient in, three gradients out.
        values = (2 * q + 2 * k) + ((4 * q + 4 * k) if case["back"] else 0)
        return {"bytes": size * values, "flops": (4 + (10 if case["back"] else 0)) * pairs * case["width"]}
    n = sum(r * c for r, c in _shapes(case))
    return {"bytes": 20 * n, "flops": sum(_products(s) for s in _shapes(case))}


# ---- what a program has in hand -------------------------------------------------------------------------------------------


def _type(case):
    return torch.float32 if case["type"] == "fp32" else torch.bfloat16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "rotary":
        b, l, h, d = case["batch"], case["length"], case["heads"], case["width"]
        packed = _randn(g, b, l, h + case["others"], d).to(_type(case))
        start = torch.randint(0, case["reach"] - l + 1, (b, 1), generator=g, device="cuda")
        s["x"], s["at"] = packed[:, :, :h], (start + torch.arange(l, device="cuda")[None]).to(torch.int32)
        s["y"] = torch.empty(b, l, h, d, device="cuda", dtype=_type(case))
        s["frequencies"] = (C.c_double * (case["turned"] // 2))(*_frequencies(case))
        s["rates"] = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
        return s
    if case["kind"] == "attention":
        b, h, hk, lq, lk, d = (case[n] for n in ("batch", "heads", "shared", "queries", "keys", "width"))
        t = _type(case)
        if lq == lk:   # one packed projection holds the three, as its gradient does
            packed, grads = _randn(g, b, lq, h + 2 * hk, d).to(t), torch.empty(b, lq, h + 2 * hk, d, device="cuda", dtype=t)
            s["q"], s["k"], s["v"] = packed[:, :, :h], packed[:, :, h:h + hk], packed[:, :, h + hk:]
            s["dq"], s["dk"], s["dv"] = grads[:, :, :h], grads[:, :, h:h + hk], grads[:, :, h + hk:]
        else:
            packed, grads = _randn(g, b, lk, 2 * hk, d).to(t), torch.empty(b, lk, 2 * hk, d, device="cuda", dtype=t)
            s["q"], s["k"], s["v"] = _randn(g, b, lq, h, d).to(t), packed[:, :, :hk], packed[:, :, hk:]
            s["dq"], s["dk"], s["dv"] = torch.empty_like(s["q"]), grads[:, :, :hk], grads[:, :, hk:]
        s["g"] = _randn(g, b, lq, h, d).to(t) if case["back"] else None
        s["out"] = torch.empty(b, lq, h, d, device="cuda", dtype=t)
        s["lse"] = torch.empty(b, h, lq, device="cuda")
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None
        s["prefix"] = torch.full((b,), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
        s["documents"] = torch.tensor([_documents(case, r) for r in range(b)], dtype=torch.int32, device="cuda") if case["document"] else None
        s["mine"] = s["documents"][:, lk - lq:].contiguous() if case["document"] else None
        return s
    shapes = _shapes(case)
    s["shapes"] = shapes
    s["p"] = [0.02 * _randn(g, *shape) for shape in shapes]
    s["g"] = [1e-3 * _randn(g, *shape) for shape in shapes]
    s["m"] = [1e-3 * _randn(g, *shape) for shape in shapes]
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------


def _ptr(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


def _run_own(s):
    omb, ctx = _framework()
    case = s["case"]

    def strides(t):
        return C.byref(omb.HeadStrides(t.stride(0), t.stride(2), t.stride(1)))

    if case["kind"] == "rotary":
        x, y = s["x"], s["y"]
        ctx.call("om_rotary" if case["type"] == "fp32" else "om_rotary_bf16", ctx.handle, _ptr(x), strides(x), _ptr(s["at"]), omb.i64(case["length"]),
                 omb.i32(0), omb.i32(case["batch"]), omb.i32(case["heads"]), omb.i32(case["length"]), omb.i32(case["width"]), s["frequencies"],
                 omb.i32(case["turned"] // 2), omb.i32(case["adjacent"]), omb.f32(_magnitude(case)), omb.i32(case["back"]), _ptr(y), strides(y))
        return {"y": y}
    if case["kind"] == "attention":
        b, h, hk, lq, lk, d = (case[n] for n in ("batch", "heads", "shared", "queries", "keys", "width"))
        rule = omb.AttentionRule(causal=case["causal"], window=case["window"], q_offset=lk - lq, softcap=case["cap"], slopes=_ptr(s["slopes"]),
                                 prefix=_ptr(s["prefix"]), q_documents=_ptr(s["mine"]), k_documents=_ptr(s["documents"]))
        sizes = [omb.i32(n) for n in (b, h, hk, lq, lk, d)] + [omb.f32(d ** -0.5)]
        qkv = [a for n in ("q", "k", "v") for a in (_ptr(s[n]), strides(s[n]))]
        none, half = C.c_void_p(None), case["type"] != "fp32"
        out = [none, _ptr(s["out"])] if half else [_ptr(s["out"])]
        ctx.call("om_rule_attention_fwd" + ("_bf16" if half else ""), ctx.handle, C.byref(rule), *qkv, *sizes, *out, strides(s["out"]),
                 _ptr(s["lse"]) if case["back"] else none)
        if not case["back"]:
            return {"out": s["out"]}
        grads = [a for n in ("dq", "dk", "dv") for a in (([none] if half else []) + [_ptr(s[n]), strides(s[n])])]
        ctx.call("om_rule_attention_bwd" + ("_bf16" if half else ""), ctx.handle, C.byref(rule), _ptr(s["g"]), strides(s["g"]), *qkv, _ptr(s["out"]),
                 strides(s["out"]), _ptr(s["lse"]), *sizes, *grads)
        return {n: s[n] for n in ("out", "dq", "dk", "dv")}
    n = len(s["shapes"])
    hyper = omb.MuonHyper(lr=RATE, momentum=case["momentum"], weight_decay=case["decay"], eps=EPS, grad_scale=1.0, nesterov=case["nesterov"], steps=STEPS, match_rms=1)
    lists = [(C.c_void_p * n)(*[t.data_ptr() for t in s[name]]) for name in ("p", "g", "m")]
    ctx.call("om_optim_muon_step", ctx.handle, omb.i32(n), *lists, None, omb.int_array([r for r, _ in s["shapes"]]),
             omb.int_array([c for _, c in s["shapes"]]), C.byref(hyper), None)
    return {"p": s["p"], "m": s["m"]}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"rotary": _rotary, "attention": _attention, "muon": _muon}[state["case"]["kind"]](state)


def _rotary(s):
    case = s["case"]
    angle = s["at"].to(torch.float64)[:, :, None, None] * s["rates"]
    cos, sin = (angle.cos() * _magnitude(case)).float(), (angle.sin() * _magnitude(case)).float()
    if case["back"]:
        sin = -sin
    x = s["x"].float()
    turned = x[..., : case["turned"]]
    if case["adjacent"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        new = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turned.chunk(2, dim=-1)
        new = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return {"y": torch.cat([new, x[..., case["turned"]:]], dim=-1).to(s["y"].dtype)}


def _attention(s):
    case = s["case"]
    b, h, hk, lq, lk, d = (case[n] for n in ("batch", "heads", "shared", "queries", "keys", "width"))
    t = s["q"].dtype
    # [batch, key heads, query heads of each * queries, width]: the query heads of a key head are rows of one product.
    rows = lambda x: x.float().permute(0, 2, 1, 3).reshape(b, hk, (h // hk) * lq, d)   # noqa: E731
    back = lambda x: x.reshape(b, h, lq, d).permute(0, 2, 1, 3).to(t)                  # noqa: E731
    q, k, v = rows(s["q"]), s["k"].float().permute(0, 2, 1, 3), s["v"].float().permute(0, 2, 1, 3)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(b, h, lq, lk)
    slope = None
    if case["cap"]:
        score.div_(case["cap"]).tanh_()
        slope = 1 - score * score if case["back"] else None
        score.mul_(case["cap"])
    if case["slopes"]:
        far = (torch.arange(lq, device="cuda")[:, None] + (lk - lq) - torch.arange(lk, device="cuda")[None, :]).abs().float()
        score.sub_(s["slopes"][None, :, None, None] * far)
    far = torch.arange(lq, device="cuda")[:, None] + (lk - lq) - torch.arange(lk, device="cuda")[None, :]
    hidden = torch.zeros(1, 1, lq, lk, dtype=torch.bool, device="cuda")
    if case["causal"]:
        hidden = hidden | (far < 0)
    if case["window"]:
        hidden = hidden | (far.abs() >= case["window"])
    if case["prefix"]:
        hidden = hidden & (torch.arange(lk, device="cuda")[None, :] >= s["prefix"][:, None])[:, None, None]
    if case["document"]:
        hidden = hidden | ((s["mine"][:, :, None] != s["documents"][:, None, :]) | (s["mine"] < 0)[:, :, None])[:, None]
    score.masked_fill_(hidden, -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp_(min=-3e38)
    p = score.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p.div_(total.clamp_(min=1e-37))
    grouped = p.view(b, hk, (h // hk) * lq, lk)
    out = torch.matmul(grouped, v)
    if not case["back"]:
        return {"out": back(out)}
    g = rows(s["g"])
    dv = torch.matmul(grouped.transpose(2, 3), g)
    ds = torch.matmul(g, v.transpose(2, 3)).sub_((g * out).sum(dim=-1, keepdim=True)).mul_(grouped)
    if slope is not None:
        ds.mul_(slope.view_as(ds))
    dq = torch.matmul(ds, k).mul_(d ** -0.5)
    dk = torch.matmul(ds.transpose(2, 3), q).mul_(d ** -0.5)
    return {"out": back(out), "dq": back(dq), "dk": dk.permute(0, 2, 1, 3).to(t), "dv": dv.permute(0, 2, 1, 3).to(t)}


def _muon(s):
    case = s["case"]
    together = {}
    for i, shape in enumerate(s["shapes"]):
        together.setdefault(shape, []).append(i)
    for (rows, cols), at in together.items():   # matrices of one shape as one batch
        m, g = torch.stack([s["m"][i] for i in at]), torch.stack([s["g"][i] for i in at])
        m.mul_(case["momentum"]).add_(g, alpha=1 - case["momentum"])
        u = g * (1 - case["momentum"]) + m * case["momentum"] if case["nesterov"] else m
        x = u.transpose(1, 2) if rows > cols else u
        x = x / x.square().sum(dim=(1, 2), keepdim=True).sqrt().clamp(min=EPS)
        for _ in range(STEPS):
            a = torch.bmm(x, x.transpose(1, 2))
            x = torch.baddbmm(x, torch.baddbmm(a, a, a, beta=B, alpha=CC), x, beta=A)
        x = x.transpose(1, 2) if rows > cols else x
        rate = RATE * 0.2 * math.sqrt(max(rows, cols))
        for k, i in enumerate(at):
            s["m"][i].copy_(m[k])
            s["p"][i].mul_(1 - RATE * case["decay"]).sub_(x[k], alpha=rate)
    return {"p": s["p"], "m": s["m"]}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return {"rotary": _exact_rotary, "attention": _exact_attention, "muon": _exact_muon}[case["kind"]](case, prepare(case, seed))


def _exact_rotary(case, s):
    x = s["x"].double()
    turn = s["at"].double()[..., None] * s["rates"] * (-1.0 if case["back"] else 1.0)
    unit = torch.polar(torch.full_like(turn, _magnitude(case)), turn)[:, :, None]
    n = case["turned"]
    first, second = (x[..., 0:n:2], x[..., 1:n:2]) if case["adjacent"] else (x[..., : n // 2], x[..., n // 2: n])
    z = torch.complex(first, second) * unit
    y = x.clone()
    if case["adjacent"]:
        y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
    else:
        y[..., : n // 2], y[..., n // 2: n] = z.real, z.imag
    return {"y": y}


def _exact_attention(case, s):
    h, hk, lq, lk, d = (case[n] for n in ("heads", "shared", "queries", "keys", "width"))
    seen = _visible(case, "cuda")
    found = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in (("out", "dq", "dk", "dv") if case["back"] else ("out",))}
    far = (torch.arange(lq, device="cuda", dtype=torch.float64)[:, None] + (lk - lq) - torch.arange(lk, device="cuda", dtype=torch.float64)[None, :]).abs()
    for n in range(case["batch"]):
        mask = seen[n if seen.shape[0] > 1 else 0]
        for i in range(h):
            j = i // (h // hk)
            q, k, v = s["q"][n, :, i].double(), s["k"][n, :, j].double(), s["v"][n, :, j].double()
            z = q @ k.t() / math.sqrt(d)
            if case["cap"]:
                th = torch.tanh(z / case["cap"])
                z = case["cap"] * th
            if case["slopes"]:
                z = z - 2.0 ** (-8.0 * (i + 1) / h) * far
            weight = torch.softmax(torch.where(mask, z, -1e300), dim=-1) * mask
            found["out"][n, :, i] = weight @ v
            if case["back"]:
                g = s["g"][n, :, i].double()
                inner = g @ v.t()
                dz = weight * (inner - (weight * inner).sum(dim=-1, keepdim=True))
                if case["cap"]:
                    dz = dz * (1 - th ** 2)
                found["dq"][n, :, i] = dz @ k / math.sqrt(d)
                found["dk"][n, :, j] += dz.t() @ q / math.sqrt(d)
                found["dv"][n, :, j] += weight.t() @ g
    return found


def _exact_muon(case, s):
    ps, ms = [], []
    mu = case["momentum"]
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        p, g = p.double(), g.double()
        m = mu * m.double() + (1 - mu) * g
        u = (1 - mu) * g + mu * m if case["nesterov"] else m
        x = u / max(float(torch.linalg.norm(u)), EPS)
        for _ in range(STEPS):   # by the smaller of the two Gram matrices
            if x.shape[0] <= x.shape[1]:
                w = x @ x.t()
                x = A * x + B * (w @ x) + CC * (w @ (w @ x))
            else:
                w = x.t() @ x
                x = A * x + B * (x @ w) + CC * ((x @ w) @ w)
        ms.append(m)
        ps.append(p * (1 - RATE * case["decay"]) - RATE * 0.2 * math.sqrt(max(p.shape)) * x)
    return {"p": ps, "m": ms}
