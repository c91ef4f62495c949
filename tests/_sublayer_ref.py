"""Plain float64 evaluations of the 16-bit product with its epilogue and of the
gated residual norms, with the error bounds that their tests use."""
import math

import numpy as np

import _experts_ref as R

U = 2.0 ** -24


def _erfc(x):
    return np.vectorize(math.erfc, otypes=[float])(x)


def act(z, name):
    """(value, slope) of an activation in float64; NaN where z is."""
    z = np.asarray(z, dtype=np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if name is None:
            return z, np.ones_like(z)
        if name == "relu":
            return np.where(z < 0, 0.0, z), np.where(z > 0, 1.0, 0.0)
        c = np.clip(z, -745.0, 745.0)  # NaN stays
        if name == "silu":
            s = 1.0 / (1.0 + np.exp(-c))
            return np.where(z == -np.inf, 0.0, z * s), s * (1.0 + c * (1.0 - s))
        phi = 0.5 * _erfc(-np.clip(z, -50, 50) / math.sqrt(2.0))
        density = np.exp(-0.5 * np.clip(z, -50, 50) ** 2) / math.sqrt(2 * math.pi)
        return np.where(z == -np.inf, 0.0, z * phi), phi + np.clip(z, -50, 50) * density


# The f32 activations (csrc/linear16.cuh).  gelu = max(z, 0) - a Q(a) and its
# slope take e^(-a^2/2) of an argument below 103 (Q(14.4) leaves f32) with three
# roundings: 103 * 3 * 2^-24 = 1.9e-5 relative, a polynomial within 6e-7 and four
# more roundings: 2^-15 of a Q(a) (at most 0.17) and of Q + a phi (at most 0.63).
# silu takes e^-z, |z| < 89, with two: 89 * 2 * 2^-24 = 1.1e-5, 2^-15 again, of |y|
# and of a slope's terms (at most 1.3); below z = -128 ln 2 = -88.7, where e^-z leaves
# f32, it is 0 in place of at most 88.8 e^-88.7 = 2.6e-37 < 2^-121.  Slopes are at most
# 1.13.
ACT_REL = 2.0 ** -15
STEEP = {None: 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}


def act_error(z, name):
    if name in (None, "relu"):
        return np.zeros_like(z)
    y = act(z, name)[0]
    if name == "silu":
        return ACT_REL * np.abs(y) + 2.0 ** -121
    return ACT_REL * np.abs(np.maximum(z, 0) - y) + 2 * U * np.abs(y) + 2.0 ** -120


def slope_error(z, name):
    return np.zeros_like(z) if name in (None, "relu") else np.full_like(z, ACT_REL * 1.3)


def product(a, b):
    """(a . b, its error): the tensor core's f32 sums, (k + 2) 2^-23 of the sum
    of magnitudes (it may truncate where IEEE rounds)."""
    return a @ b, (a.shape[1] + 2) * 2.0 ** -23 * (np.abs(a) @ np.abs(b))


def linear(a, b, bias=None, activation=None, residual=None):
    """(y, its bound, z, its bound)."""
    z, e = product(a, b)
    if bias is not None:
        z = z + bias
        e = e + U * np.abs(z)
    y = act(z, activation)[0]
    bound = STEEP[activation] * e + act_error(z, activation)
    if residual is not None:
        y = y + residual
        bound = bound + U * np.abs(y)
    return y, bound * (1 + 2.0 ** -10), z, e


def linear_through(a, b, z, activation):
    g, e = product(a, b)
    slope = act(z, activation)[1]
    return g * slope, e * STEEP[activation] + np.abs(g) * (slope_error(z, activation) + 2 * U * STEEP[activation])


# ------------------------------------------------------------------- norms

# Sums over a row: at most 32 values a thread one after another, five steps of a
# warp, four of the warps, each rounding once; means, roots and products a few
# more: 64 roundings cover each of a norm's two sums with room.
ROW = 64 * U


def stats(v, kind, eps):
    """(n, r): the normalised rows and what they were multiplied by."""
    if kind == "layer":
        v = v - v.mean(-1, keepdims=True)
    r = 1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    return v * r, r


def stats_error(v, kind, eps):
    """Bound of n: the mean's error ROW mean|v|, the root's relative ROW."""
    n, r = stats(v, kind, eps)
    shift = np.abs(v).mean(-1, keepdims=True) + np.abs(v) if kind == "layer" else 0.0
    return ROW * (2 * np.abs(n) + r * shift)


def join(x, branch, p):
    """residual_norm in float64: (y, its bound, h, its bound); p has post_gamma,
    post_beta, gate, scale, pre_gamma, pre_beta, eps and kind."""
    rows, hidden = x.shape
    gate = p.get("gate")
    g = 1.0 if gate is None else np.repeat(gate.reshape(-1, hidden), rows // max(1, gate.size // hidden), 0)
    if branch is None:
        y, ey = x, np.zeros_like(x)
    else:
        u, eu = branch, np.zeros_like(x)
        if p.get("post_gamma") is not None:
            n = stats(branch, p["kind"], p["eps"])[0]
            u = n * p["post_gamma"]
            eu = stats_error(branch, p["kind"], p["eps"]) * np.abs(p["post_gamma"]) + 2 * U * np.abs(u)
            if p.get("post_beta") is not None:
                u = u + p["post_beta"]
                eu = eu + 2 * U * np.abs(p["post_beta"])
        y = p["scale"] * x + g * u
        ey = np.abs(g) * (eu + 3 * U * (np.abs(u) + np.abs(p.get("post_beta", 0.0) if p.get("post_beta") is not None else 0.0))) \
            + 2 * U * (np.abs(p["scale"] * x) + np.abs(y))
    if p.get("pre_gamma") is None:
        return y, ey, None, None
    n, r = stats(y, p["kind"], p["eps"])
    # an error of y moves n directly, through the mean and through the root
    moved = r * (ey + ey.mean(-1, keepdims=True) + np.abs(n) * np.sqrt((ey * ey).mean(-1, keepdims=True)))
    en = stats_error(y, p["kind"], p["eps"]) + moved
    h = n * p["pre_gamma"]
    eh = en * np.abs(p["pre_gamma"]) + 2 * U * np.abs(h)
    if p.get("pre_beta") is not None:
        h = h + p["pre_beta"]
        eh = eh + 2 * U * (np.abs(h) + np.abs(p["pre_beta"]))
    return y, ey, h, eh * (1 + 2.0 ** -10)


def _through_norm(g, eg, n, en, r, kind):
    """(the gradient through a norm, its bound) from that of n."""
    m = (g * n).mean(-1, keepdims=True)
    d = g - n * m
    mean_g = np.abs(g).mean(-1, keepdims=True)
    em = (np.abs(g) * en + eg * np.abs(n)).mean(-1, keepdims=True) + ROW * np.abs(g * n).mean(-1, keepdims=True)
    ed = eg + np.abs(n) * em + en * np.abs(m) + ROW * (np.abs(g) + np.abs(n * m))
    if kind == "layer":
        d = d - g.mean(-1, keepdims=True)
        ed = ed + eg.mean(-1, keepdims=True) + ROW * mean_g
    return d * r, r * (ed + ROW * np.abs(d))


def join_bwd(dy, dh, y, branch, p):
    """residual_norm_bwd in float64: {name: (value, bound)}.  A column's sum over
    R rows takes at most R + 64 roundings of its terms."""
    rows, hidden = y.shape
    kind, eps = p["kind"], p["eps"]
    long = (rows + 64) * U
    out = {}
    dt, edt = (np.zeros_like(y), np.zeros_like(y)) if dy is None else (dy, np.zeros_like(y))
    if dh is not None:
        n, r = stats(y, kind, eps)
        en = stats_error(y, kind, eps)
        out["dpre_gamma"] = (dh * n).sum(0), (np.abs(dh) * en).sum(0) + long * np.abs(dh * n).sum(0)
        if p.get("pre_beta") is not None:
            out["dpre_beta"] = dh.sum(0), long * np.abs(dh).sum(0)
        q = dh * p["pre_gamma"]
        d, ed = _through_norm(q, U * np.abs(q), n, en, r, kind)
        dt, edt = dt + d, ed + 2 * U * (np.abs(dt) + np.abs(d))
    out["dx"] = p["scale"] * dt, np.abs(p["scale"]) * (edt + 2 * U * np.abs(dt))
    if branch is None and dy is not None and p.get("gate") is None and not p.get("has_branch"):
        return out
    gate = p.get("gate")
    groups = 1 if gate is None else max(1, gate.size // hidden)
    g = np.ones((1, hidden)) if gate is None else np.repeat(gate.reshape(-1, hidden), rows // groups, 0)
    w, ew = dt * g, np.abs(g) * (edt + 2 * U * np.abs(dt))
    post = p.get("post_gamma") is not None
    u, eu = branch, 0.0
    if post:
        n, r = stats(branch, kind, eps)
        en = stats_error(branch, kind, eps)
        u = n * p["post_gamma"] + (p["post_beta"] if p.get("post_beta") is not None else 0.0)
        eu = en * np.abs(p["post_gamma"]) + 8 * U * (np.abs(n * p["post_gamma"]) + np.abs(u))
        out["dpost_gamma"] = ((w * n).sum(0), (ew * np.abs(n) + np.abs(w) * en).sum(0) + (long + 8 * U) * np.abs(w * n).sum(0))
        if p.get("post_beta") is not None:
            out["dpost_beta"] = w.sum(0), ew.sum(0) + (long + 8 * U) * np.abs(w).sum(0)
    if gate is not None:
        def by_group(v):
            s = v.reshape(groups, rows // groups, hidden).sum(1)
            return s if gate.ndim == 2 else s[0]
        terms = np.abs(dt) * (np.abs(u) + (2 * np.abs(p["post_beta"]) if post and p.get("post_beta") is not None else 0.0))
        out["dgate"] = by_group(dt * u), by_group(edt * np.abs(u) + np.abs(dt) * eu + (long + 8 * U) * terms
                                                  + edt * (np.abs(p["post_beta"]) if post and p.get("post_beta") is not None else 0.0))
    if post:
        w2 = w * p["post_gamma"]
        w, ew = _through_norm(w2, ew * np.abs(p["post_gamma"]) + U * np.abs(w2), n, en, r, kind)
    out["dbranch"] = w, ew
    return out


def check(got, ref, bound, dtype):
    """Assert that a tensor is within a bound and half an ulp of its type."""
    g = got.double().cpu().numpy()
    bad = R.outside(g, ref, bound, dtype)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(g - ref)[bad])))
