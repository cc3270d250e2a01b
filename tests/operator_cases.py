"""Programs over the transformer operators, their formulas in float64 and the error a correct fp32 evaluation may make.

Tolerances count roundings of u = 2^-24 (fp32, to nearest): a sum of n terms is off by at most n u of the sum of their
magnitudes, whatever its order; a product on the tensor cores is assembled from halves of 11 bits, which leaves 2^-21 of
each term, and added with truncation, which leaves at most 2^-23 for each of the 3 D / 16 instructions.  Halves are fp16: the
smallest step is 2^-24, so whatever the size of a value, half a step, 2^-25 of the operand's unit, is left.  The unit is
chosen so that the largest value of a tile lies in [2^14, 2^15): 2^-39 of that value; weights are kept in units of 2^-10:
2^-35.  FLOOR_* are those, doubled for the second operand of a product.
"""
from __future__ import annotations

import importlib

import numpy as np

adb = importlib.import_module("autodiff-ir-rust_b200")
ad, nn = adb.autodiff, adb.nn
U = 2.0 ** -24
FLOOR_VALUE, FLOOR_WEIGHT = 2.0 ** -38, 2.0 ** -34


def close(name, got, want, tol):
    """every element within its own tolerance; NaN only where NaN is wanted"""
    got, want, tol = (np.asarray(x, np.float64) for x in (got, want, tol))
    assert got.shape == want.shape, f"{name}: {got.shape} != {want.shape}"
    bad = ~(np.abs(got - want) <= tol + 1e-37) & ~(got == want) & ~(np.isnan(got) & np.isnan(want))
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want) / (tol + 1e-37), 0)), got.shape) if got.ndim else ()
        raise AssertionError(f"{name}: {bad.sum()} of {got.size} beyond tolerance, worst at {i}: {got[i]!r} instead of {want[i]!r} +- {np.broadcast_to(tol, got.shape)[i]:.3g}")


def start(dev):
    ad.set_device(dev)
    ad.eager_dep_opt()


def leaf(x):
    return ad.tensor(np.ascontiguousarray(x, np.float32).reshape(-1), list(x.shape))


def data(x):
    return None if x is None else leaf(x).val().to_node()


def finish(kept):
    for v in kept.values():
        v.keep()
    ad.execute()
    return {n: np.asarray(v.get().data, np.float32).reshape(v.get().dim) for n, v in kept.items()}


# ---------------------------------------------------------------------------------------------------- norm
def norm_case(shape, seed=0, residual=True):
    rng = np.random.default_rng(seed)
    x = {k: rng.standard_normal(shape).astype(np.float32) * s for k, s in (("x", 0.7), ("r", 2.0), ("dy", 0.1), ("dh", 0.1))}
    x["g"] = (1 + 0.2 * rng.standard_normal(shape[-1])).astype(np.float32)
    if not residual:
        x["r"] = x["dh"] = None
    return x


def norm_run(dev, x, eps=1e-6, grad=True):
    start(dev)
    a, g = leaf(x["x"]), leaf(x["g"])
    kept = {}
    if x["r"] is None:
        y = ad.rms_norm(a, g, eps=eps)
        loss = y * data(x["dy"])
        kept["y"] = y.forward()
    else:
        r = leaf(x["r"])
        y, h = ad.rms_norm(a, g, r, eps)
        loss = y * data(x["dy"]) + h * data(x["dh"])
        kept["y"], kept["h"] = y.forward(), h.forward()
    if grad:
        loss.forward()
        loss.backward()
        kept["dx"], kept["dg"] = a.grad(), g.grad()
        if x["r"] is not None:
            kept["dr"] = r.grad()
    return finish(kept)


def norm_reference(x, eps=1e-6):
    f = {k: None if v is None else v.astype(np.float64) for k, v in x.items()}
    h = f["x"] if f["r"] is None else f["x"] + f["r"]
    big = np.abs(f["x"]) + (0 if f["r"] is None else np.abs(f["r"]))   # what h's rounding is relative to
    width = h.shape[-1]
    inv = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n, y = h * inv, h * inv * f["g"]
    dn = f["dy"] * f["g"]
    dx = inv * (dn - n * (dn * n).mean(-1, keepdims=True)) + (0 if f["dh"] is None else f["dh"])
    axes = tuple(range(h.ndim - 1))
    rows = h.size // width
    # a thread adds at most 32 products in turn, the rest is a tree of at most 10 levels (a walk of width / 1024 beyond it)
    s = (48 + width / 1024) * U
    ref = {"y": (y, s * np.abs(y) + 2 * U * inv * np.abs(f["g"]) * big), "h": (h, U * np.abs(h))}
    away = np.abs(dn) + np.abs(n) * (np.abs(dn * n)).mean(-1, keepdims=True)
    ref["dx"] = ref["dr"] = (dx, 4 * s * inv * away + 2 * U * np.abs(dx) + 4 * U * inv * inv * big * np.abs(dn).max(-1, keepdims=True))
    # h is rounded once more in the gradient's own operand; sums over rows: at most rows / blocks in turn, then the blocks
    ref["dg"] = ((f["dy"] * n).sum(axes), (s + (rows + 8) * U) * np.abs(f["dy"] * inv * big).sum(axes))
    return ref


def norm_check(got, x, eps=1e-6):
    ref = norm_reference(x, eps)
    for k, v in got.items():
        close(k, v, *ref[k])


# ---------------------------------------------------------------------------------------------------- rotary
def rotary_run(dev, x, dy, rot, positions=None, offset=0, grad=True, **kw):
    start(dev)
    a = leaf(x)
    turn = nn.Rotary(rot, **kw)
    y = turn.f(a, data(positions), offset)
    kept = {"y": y.forward()}
    if grad:
        loss = y * data(dy)
        loss.forward()
        loss.backward()
        kept["dx"] = a.grad()
    return finish(kept)


def rotary_reference(x, dy, rot, positions=None, offset=0, base=10000.0, stretch=1.0, interleaved=False, gain=1.0):
    b, t, h, d = x.shape
    freq = base ** (-np.arange(0, rot, 2) / rot) / stretch
    at = offset + np.arange(t, dtype=np.float64) if positions is None else positions.astype(np.float64)
    angle = np.broadcast_to(at, (b, t))[..., None, None] * freq
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2, rot))
    out = {}
    for name, v, sign in (("y", x, 1), ("dx", dy, -1)):
        v = v.astype(np.float64)
        r = v.copy()
        c, s = np.cos(angle), sign * np.sin(angle)
        r[..., i] = gain * (v[..., i] * c - v[..., j] * s)
        r[..., j] = gain * (v[..., j] * c + v[..., i] * s)
        # the angle: 3 roundings of less than a turn (2 pi u each, doubled for sine and cosine) and the table's own
        # 2^-48 of position * frequency; then two products and a sum
        tol = np.zeros_like(r)
        size = abs(gain) * (np.abs(v[..., i]) + np.abs(v[..., j]))
        err = 48 * U + 2 * np.abs(angle) * 2.0 ** -48
        tol[..., i] = tol[..., j] = err * size
        out[name] = (r, tol)
    return out


# ---------------------------------------------------------------------------------------------------- attention
def attention_case(b, tq, tk, h, g, d, seed=0, slopes=False, docs=None, prefix=None, lengths=None, causal=True, cap=0.0,
                   scale=None):
    rng = np.random.default_rng(seed)
    c = dict(causal=causal, cap=cap, scale=scale)
    for name, shape in (("q", (b, tq, h, d)), ("k", (b, tk, g, d)), ("v", (b, tk, g, d)), ("do", (b, tq, h, d))):
        c[name] = rng.standard_normal(shape).astype(np.float32)
    c["slopes"] = (2.0 ** -np.arange(1, h + 1)).astype(np.float32) if slopes else None
    for name, v in (("docs", docs), ("prefix", prefix), ("lengths", lengths)):
        c[name] = None if v is None else np.asarray(v, np.float32)
    return c


def attention_run(dev, c, grad=True, views=lambda t: t):
    start(dev)
    q, k, v = leaf(c["q"]), leaf(c["k"]), leaf(c["v"])
    out = ad.attention(views(q), views(k), views(v), c["scale"], c["causal"], c["cap"],
                       *(data(c[n]) for n in ("slopes", "docs", "prefix", "lengths")))
    kept = {"out": out.forward()}
    if grad:
        loss = out * data(c["do"])
        loss.forward()
        loss.backward()
        kept.update(dq=q.grad(), dk=k.grad(), dv=v.grad())
    return finish(kept)


def attention_sees(c):
    """[b, tq, tk] which keys a query sees, and the positions [b, tq]"""
    b, tq = c["q"].shape[:2]
    tk = c["k"].shape[1]
    n = np.full(b, tk) if c["lengths"] is None else np.clip(np.nan_to_num(c["lengths"], nan=0.0), 0, tk).astype(np.int64)
    pos = np.arange(tq)[None] + (n - tq)[:, None]
    j = np.arange(tk)[None, None]
    see = np.broadcast_to(j < n[:, None, None], (b, tq, tk)).copy()
    if c["causal"] or c["lengths"] is not None:
        see &= (pos >= 0)[..., None]
    if c["causal"]:
        first = np.zeros(b) if c["prefix"] is None else np.clip(np.nan_to_num(c["prefix"], nan=0.0), 0, tk).astype(np.int64)
        see &= (j <= pos[..., None]) | (j < first[:, None, None])
    if c["docs"] is not None:
        mine = np.take_along_axis(c["docs"], np.maximum(pos, 0), 1)
        see &= (mine[..., None] == c["docs"][:, None]) & (c["docs"][:, None] >= 0)
    return see, pos


def attention_reference(c):
    """results with their tolerances; rows that no pair reaches enter as zeros"""
    see, pos = attention_sees(c)
    b, tq, h, d = c["q"].shape
    tk, g = c["k"].shape[1:3]
    scale = 1 / np.sqrt(d) if c["scale"] is None else c["scale"]
    res = {n: (np.zeros(c[m].shape), np.zeros(c[m].shape)) for n, m in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    dot = (d + 16) * U + 2.0 ** -21 + 3 * d / 16 * 2.0 ** -23     # of sum |a_i b_i|
    sums = (128 + tk / 16 + tq * (h // g) / 16) * U               # of the sums over keys and over queries
    j = np.arange(tk)
    for n in range(b):
        used_k, used_q = see[n].any(0), see[n].any(1)
        most = {x: np.abs(np.where((used_k if x in "kv" else used_q)[:, None, None], c[x][n].astype(np.float64), 0)).max(initial=0) for x in ("q", "k", "v", "do")}
        for m in range(h):
            at = m // (h // g)
            q, do = (np.where(used_q[:, None], x[n, :, m].astype(np.float64), 0) for x in (c["q"], c["do"]))
            k, v = (np.where(used_k[:, None], x[n, :, at].astype(np.float64), 0) for x in (c["k"], c["v"]))
            s = q @ k.T * scale
            err = dot * np.abs(scale) * (np.abs(q) @ np.abs(k).T) + 4 * U * np.abs(s) + FLOOR_VALUE * d * np.abs(scale) * most["q"] * most["k"]
            bend = np.ones_like(s)
            if c["cap"]:
                t = np.tanh(s / c["cap"])
                s, bend, err = t * c["cap"], 1 - t * t, err + 8 * U * c["cap"]
            if c["slopes"] is not None:
                far = c["slopes"][m].astype(np.float64) * np.abs(pos[n][:, None] - j)
                s, err = s - far, err + 4 * U * (far + np.abs(s))
            s = np.where(see[n], s, -np.inf)
            top = np.where(used_q, s.max(1, initial=-np.inf), 0)[:, None]
            e = np.where(see[n], np.exp(np.where(see[n], s - top, 0)), 0)
            p = e / np.where(used_q, e.sum(1), 1)[:, None]
            o = p @ v
            # a weight's relative error: its score's, its row's sum's, the exponential's (argument of up to |s - top|)
            rel = 2 * np.where(see[n], err + 4 * U * np.abs(np.where(see[n], s - top, 0)), 0).max(1, initial=0)[:, None] + 16 * U
            res["out"][0][n, :, m] = o
            seen = see[n].astype(np.float64)
            res["out"][1][n, :, m] = (rel + sums + 2.0 ** -21) * (p @ np.abs(v)) + FLOOR_WEIGHT * seen.sum(1, keepdims=True) * most["v"]
            dp = do @ v.T
            delta = (do * o).sum(1, keepdims=True)
            size = FLOOR_VALUE / U * d * most["do"] * most["v"] + np.abs(do) @ np.abs(v).T + (np.abs(do) * (p @ np.abs(v))).sum(1, keepdims=True)
            ds = p * (dp - delta) * bend * scale
            # the bend's own error is at most 4 err / cap <= 4 u-sized terms already in rel when the cap is at least 1
            worst = p * size * np.abs(scale) * (2 * rel + dot + sums + 2.0 ** -20) + (p * size * np.abs(scale) * 4 * err / c["cap"] if c["cap"] else 0)
            worst = worst + FLOOR_VALUE * seen * np.abs(scale) * 2 * d * most["do"] * most["v"]     # ds in units of its bound
            res["dq"][0][n, :, m] = ds @ k
            res["dq"][1][n, :, m] = worst @ np.abs(k) + FLOOR_VALUE * worst.sum(1, keepdims=True) / U * most["k"]
            res["dk"][0][n, :, at] += ds.T @ q
            res["dk"][1][n, :, at] += worst.T @ np.abs(q) + FLOOR_VALUE * worst.sum(0)[:, None] / U * most["q"]
            res["dv"][0][n, :, at] += p.T @ do
            res["dv"][1][n, :, at] += (p * (rel + sums + 2.0 ** -21)).T @ np.abs(do) + FLOOR_WEIGHT * seen.sum(0)[:, None] * most["do"]
    return res


def attention_check(got, c):
    ref = attention_reference(c)
    for k, v in got.items():
        close(k, v, *ref[k])
