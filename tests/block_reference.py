"""Plain forms of the residual-block operators, in numpy's longdouble (64-bit mantissa) where an
element-wise bound needs a reference without errors of its own, and the bounds themselves.

U is the unit roundoff of f64 (half a step): every operation on doubles is within U of its value.  A
sum of n terms in any order is within (depth) * U * sum|terms|, depth being the longest chain of
additions a term goes through."""
import math

import numpy as np
from scipy.special import erf

U = 2.0 ** -53
LD = np.longdouble
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def row_chain(cols):
    """Longest chain of additions in a row sum: each of at least 8 threads adds its share (at most 16
    values in registers; cols / 1024 + 2 in the walking kernels), then 6 exchanges and 16 wavefronts."""
    return 16 + cols // 1024 + 2 + 6 + 16


def column_chain(rows):
    """... in a column sum: a workgroup's own rows (at least 256 workgroups share long arrays; the strips of
    very wide rows give each at least a sixteenth), up to 128 row groups, 64 + 16 partial sums."""
    return rows // 16 + 1 + 128 + 64 + 16


def norm_forward(x, w, b, eps):
    """(y, mean, rstd, bounds of each)."""
    x64, n, L = x, x.shape[1], row_chain(x.shape[1])
    x = x.astype(LD)
    m = x.mean(1, keepdims=True)
    d = x - m
    v = (d * d).mean(1, keepdims=True)
    r = 1 / np.sqrt(v + LD(eps))
    xh = d * r
    wl = np.ones((1, n), LD) if w is None else w.astype(LD)
    y = xh * wl + (0 if b is None else b.astype(LD))
    mean_bound = (L + 1) * U * np.abs(x).mean(1, keepdims=True)
    # d is off by the mean's error and a rounding; its square's sum only by the second order of the first
    # (the deviations around the true mean cancel) and L + 3 roundings; the root halves that
    rstd_rel = ((L + 3) / 2 + 4) * U + (mean_bound / np.sqrt(v + LD(eps))) ** 2
    y_bound = np.abs(r * wl) * (mean_bound + U * np.abs(d)) + np.abs(xh * wl) * (rstd_rel + 3 * U) + 2 * U * np.abs(y)
    del x64
    return y, m, r, y_bound, mean_bound, r * rstd_rel


def norm_backward(g, x, w, m, r, residual):
    """(dx, dw, db, bounds); m and r are the doubles that the operator is given."""
    rows, n = x.shape
    L, C = row_chain(n), column_chain(rows)
    g, x, m, r = (a.astype(LD) for a in (g, x, m, r))
    xh = (x - m) * r
    u = g if w is None else g * w.astype(LD)
    c1, c2 = u.mean(1, keepdims=True), (u * xh).mean(1, keepdims=True)
    dx = r * (u - c1 - xh * c2)
    e1 = (L + 2) * U * np.abs(u).mean(1, keepdims=True)
    e2 = (L + 5) * U * np.abs(u * xh).mean(1, keepdims=True)
    inner = np.abs(u) + np.abs(c1) + np.abs(xh * c2)
    dx_bound = np.abs(r) * (e1 + np.abs(xh) * e2 + 6 * U * inner) + 2 * U * np.abs(dx)
    if residual is not None:
        dx = dx + residual.astype(LD)
        dx_bound = dx_bound + U * np.abs(dx)
    dw, db = (g * xh).mean(0, keepdims=True), g.mean(0, keepdims=True)
    return (dx, dw, db, dx_bound, (C + 5) * U * np.abs(g * xh).mean(0, keepdims=True),
            (C + 2) * U * np.abs(g).mean(0, keepdims=True))


def act(z, kind):
    """(value, derivative) in f64."""
    if kind == "relu":
        return np.maximum(z, 0.0), np.where(z > 0.0, 1.0, 0.0)
    if kind == "gelu":
        p = 0.5 * (1.0 + erf(z / math.sqrt(2.0)))
        return z * p, p + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if kind == "silu":
        s = 0.5 * (1.0 + np.tanh(0.5 * z))
        return z * s, s + z * s * (1.0 - s)
    return z, np.ones_like(z)


# Evaluating an activation or its derivative at a given z in f64, either side: the formulas have at most a
# dozen operations and library functions within 2 steps each, on intermediate values of at most
# max(1, |z|) (the derivatives' z s (1 - s) t'(z) stays below 4): 32 U max(1, |z|) for the two sides together.
def act_bound(z):
    return 32 * U * np.maximum(1.0, np.abs(z))


# |act'| <= 1.13 and |act''| <= 1.2 (gelu: 2 / sqrt(2 pi) at 0; gelu_tanh within 0.01 of it; silu: 1/2)
ACT_SLOPE, ACT_CURVE = 1.2, 1.2


def product(a, b):
    """a . b^T in f64 with the bound that covers both summation orders: 2 (K + 2) U |a| . |b|^T."""
    return a @ b.T, 2 * (a.shape[1] + 2) * U * (np.abs(a) @ np.abs(b).T)


def linear_forward(x, w, b, residual, kind):
    """(out, z, bound of out, bound of z)."""
    z, ez = product(x, w)
    if b is not None:
        z = z + b
        ez = ez + 2 * U * np.abs(z)
    y = act(z, kind)[0]
    ey = ACT_SLOPE * ez + (act_bound(z) if kind not in ("none", "relu") else 0.0)
    if residual is not None:
        y = y + residual
        ey = ey + 2 * U * np.abs(y)
    return y, z, ey, ez


def linear_backward(g, pre, kind, x, w, input_pre, input_kind, residual):
    """dz, dw, db, dx and their bounds, in f64."""
    n = x.shape[0]
    dz, ez = g, np.zeros_like(g)
    if kind != "none":
        dz = g * act(pre, kind)[1]
        ez = np.abs(g) * act_bound(pre) + 2 * U * np.abs(dz) if kind != "relu" else ez
    dw, ew = product(dz.T, x.T)
    ew = (ew + ez.T @ np.abs(x)) / n + 2 * U * np.abs(dw) / n
    db = dz.sum(0, keepdims=True) / n
    eb = (2 * (n + 2) * U * np.abs(dz).sum(0, keepdims=True) + ez.sum(0, keepdims=True)) / n
    dx, ex = product(dz, w.T)
    ex = ex + ez @ np.abs(w)
    if input_kind != "none":
        slope = act(input_pre, input_kind)[1]
        ex = ex * ACT_SLOPE + (np.abs(dx) * act_bound(input_pre) if input_kind != "relu" else 0.0)
        dx = dx * slope
        ex = ex + 2 * U * np.abs(dx)
    if residual is not None:
        dx = dx + residual
        ex = ex + 2 * U * np.abs(dx)
    return (dz, dw / n, db, dx), (ez, ew, eb, ex)


def within(got, want, bound, what=""):
    """Element-wise |got - want| <= bound, with where and by how much it is worst."""
    got = np.asarray(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.isfinite(got).all(), what
    diff = np.abs(got.astype(LD) - want)
    over = diff - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, "%s at %r: got %r want %r, off by %.3g, bound %.3g" % (
        what, at, got[at], float(want[at]), float(diff[at]), float(np.broadcast_to(bound, diff.shape)[at]))


# ---- device buffers with guards ------------------------------------------------------------------
GUARD = -7.25e300


class Guarded:
    """A device array between guard values, ``shift`` doubles off 256-byte alignment."""

    def __init__(self, engine, host, shift=0, pad=64):
        flat = np.full(host.size + 2 * pad + shift, GUARD)
        self.at, self.shape, self.size = pad + shift, host.shape, host.size
        flat[self.at:self.at + host.size] = host.reshape(-1)
        self.store = engine.from_numpy(flat.reshape(1, -1))
        self.ptr = self.store.ptr + 8 * self.at

    def get(self):
        flat = self.store.to_numpy().reshape(-1)
        assert (flat[:self.at] == GUARD).all() and (flat[self.at + self.size:] == GUARD).all(), "written past an array"
        return flat[self.at:self.at + self.size].reshape(self.shape)


def guarded(engine, host, shift=0):
    return None if host is None else Guarded(engine, host, shift)


def blank(engine, shape, shift=0):
    return Guarded(engine, np.full(shape, np.nan), shift)


def address(a):
    return None if a is None else a.ptr
