"""rst_linear_act_forward / _backward and rst_activation_* through the C ABI, element by element."""
import math

import numpy as np
import pytest
from scipy.special import erfc

from block_reference import (ACT_CURVE, ACTIVATIONS, U, act, act_bound, address, blank, guarded, linear_backward,
                             linear_forward, within)

pytestmark = pytest.mark.gpu

# (batch, in, out): single rows and small batches, the README network, odd extents, each family of tiles
# (32x32, 64x64, 128x128, on K slices and whole), an inner dimension of one
SHAPES = [(1, 1, 1), (1, 5, 3), (1, 784, 100), (1, 4096, 1000), (2, 257, 513), (3, 4095, 129), (4, 1024, 1024), (5, 100, 7),
          (8, 2048, 260), (9, 130, 31), (16, 512, 512), (17, 63, 65), (32, 784, 100), (33, 785, 101), (64, 1, 200),
          (100, 300, 33), (129, 17, 130), (512, 256, 384), (1024, 1024, 512), (2048, 100, 10), (1023, 1025, 511),
          (512, 2048, 4096), (2050, 64, 2046), (2047, 1023, 1025), (2064, 2048, 2046), (1024, 2048, 4608), (8192, 100, 100),
          (1157, 233, 203), (46, 2607, 939), (518, 3, 2177), (1953, 32, 3607), (314, 1467, 790)]
KINDS = list(ACTIVATIONS)


def check(status):
    from rstorch_amd import _ffi
    _ffi.check(status)


def data(batch, k, n):
    rng = np.random.default_rng(batch * 1000003 + k * 1009 + n)
    return (rng, rng.standard_normal((batch, k)), rng.standard_normal((n, k)) / np.sqrt(k), 0.5 * rng.standard_normal((1, n)),
            rng.standard_normal((batch, n)))


def forward(engine, x, w, b, residual, kind, pre=True, shift=0, in_place=False):
    batch, k = x.shape
    n = w.shape[0]
    dev = [guarded(engine, a, shift) for a in (x, w, b, residual)]
    out = dev[3] if in_place else blank(engine, (batch, n), shift)
    z = blank(engine, (batch, n), shift) if pre else None
    check(engine.lib.rst_linear_act_forward(engine.handle, *[address(a) for a in dev], address(z), out.ptr, batch, k, n,
                                            ACTIVATIONS[kind]))
    return (out.get(), z.get()) if pre else out.get()


def backward(engine, g, pre, kind, x, w, input_pre, input_kind, residual, shift=0, bias=True, need_input=True):
    batch, k = x.shape
    n = w.shape[0]
    dg, dpre, dx, dw, dip, dres = (guarded(engine, a, shift) for a in (g, pre, x, w, input_pre, residual))
    gp = blank(engine, (batch, n), shift) if kind != "none" else None
    gw, gb = blank(engine, (n, k), shift), blank(engine, (1, n), shift) if bias else None
    gi = blank(engine, (batch, k), shift) if need_input else None
    check(engine.lib.rst_linear_act_backward(
        engine.handle, dg.ptr, address(dpre), ACTIVATIONS[kind], address(gp), dx.ptr, dw.ptr, gw.ptr, address(gb),
        address(gi), address(dip), ACTIVATIONS[input_kind], address(dres), batch, k, n))
    return tuple(None if a is None else a.get() for a in (gp, gw, gb, gi))


@pytest.mark.parametrize("batch,k,n", SHAPES)
def test_forward(engine, batch, k, n):
    _, x, w, b, res = data(batch, k, n)
    for i, kind in enumerate(KINDS):
        # every kind with and without residual, bias and pre-activation over the shapes, not all in each
        turn = (i + batch + n) % 3
        bias, residual, pre, shift = (b if turn else None), (res if turn != 1 else None), turn != 2, i & 1
        y, z, ey, ez = linear_forward(x, w, bias, residual, kind)
        got = forward(engine, x, w, bias, residual, kind, pre, shift)
        within(got[0] if pre else got, y, ey, "out " + kind)
        if pre:
            within(got[1], z, ez, "pre " + kind)


@pytest.mark.parametrize("batch,k,n", SHAPES)
def test_backward(engine, batch, k, n):
    rng, x, w, _, g = data(batch, k, n)
    pre, input_pre, res = rng.standard_normal((batch, n)), rng.standard_normal((batch, k)), rng.standard_normal((batch, k))
    for i, input_kind in enumerate(KINDS):
        kind = KINDS[(i + batch) % 5]
        residual, shift = (res if (i + n) % 2 else None), i & 1
        want, bound = linear_backward(g, pre, kind, x, w, input_pre, input_kind, residual)
        got = backward(engine, g, pre if kind != "none" else None, kind, x, w, input_pre if input_kind != "none" else None,
                       input_kind, residual, shift)
        for name, a, b, e in zip(("grad_pre", "grad_weight", "grad_bias", "grad_input"), got, want, bound):
            if a is not None:
                within(a, b, e, "%s %s/%s" % (name, kind, input_kind))
    less = backward(engine, g, pre if kind != "none" else None, kind, x, w, None, "gelu", None, shift, bias=False,
                    need_input=False)
    within(less[1], want[1], bound[1], "grad_weight alone")


@pytest.mark.parametrize("kind", KINDS[1:])
def test_backward_against_differences(engine, kind):
    """f = sum(g * (act(x w^T + b) + r)) under a step of one weight, one bias and one input: central differences
    with h = 2^-18 (truncation h^2 / 6 * |act'''| <= h^2 per term for these activations, scaled by the cube of the
    step's effect on z, which is at most 1 here; relu is checked away from its corner)."""
    rng, x, w, b, g = data(7, 11, 5)
    res = rng.standard_normal(g.shape)
    x = np.clip(x, -0.9, 0.9)
    y, z = forward(engine, x, w, b, res, kind)
    gp, gw, gb, gx = backward(engine, g, z, kind, x, w, None, "none", None)
    h = 2.0 ** -18

    def f(xv, wv, bv):
        return forward(engine, xv, wv, bv, res, kind)[0]

    if kind == "relu":
        assert np.abs(z).min() > 4 * h
    for arr, grad, scale in ((w, gw, 7.0), (b, gb, 7.0), (x, gx, 1.0)):
        for _ in range(6):
            at = tuple(int(rng.integers(s)) for s in arr.shape)
            hi, lo = arr.copy(), arr.copy()
            hi[at] += h
            lo[at] -= h
            fh = f(*[hi if a is arr else a for a in (x, w, b)])
            fl = f(*[lo if a is arr else a for a in (x, w, b)])
            diff = (g * (fh - fl)).sum() / (hi[at] - lo[at])
            bound = h * h * np.abs(g).sum() + 256 * U * (np.abs(g) * (1 + np.abs(y))).sum() / h
            assert abs(diff - scale * grad[at]) <= bound, (kind, at, diff, scale * grad[at], bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [1, 2, 127, 128, 1001])
def test_activation_passes(engine, kind, count):
    rng = np.random.default_rng(count)
    z, g, res = (rng.standard_normal((1, count)) * s for s in (3.0, 1.0, 1.0))
    y, slope = act(z, kind)
    for shift in (0, 1):
        for residual in (None, res):
            dz, dg, dr, out = (guarded(engine, a, shift) for a in (z, g, residual, np.zeros_like(z)))
            check(engine.lib.rst_activation_forward(engine.handle, dz.ptr, address(dr), out.ptr, count, ACTIVATIONS[kind]))
            add = 0.0 if residual is None else residual
            within(out.get(), y + add, act_bound(z) + 2 * U * np.abs(y + add), "value")
            check(engine.lib.rst_activation_backward(engine.handle, dg.ptr, dz.ptr, address(dr), out.ptr, count,
                                                     ACTIVATIONS[kind]))
            within(out.get(), g * slope + add, np.abs(g) * act_bound(z) + 2 * U * (np.abs(g * slope) + np.abs(add)), "gradient")


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activations_over_their_range(engine, kind):
    """Values and derivatives from -45 to 45 and around 0, against longdouble arithmetic: the exponential is within 3 U of
    its value times max(1, its argument), which a factor exp(-argument) keeps below 3 U absolutely; the reciprocals and
    polynomials (at most 1/2 in value, slope 1 in an argument of 3 roundings) add 4 U, the cubic argument of the tanh form 4 U
    more: 16 U max(1, |z|)."""
    z = np.concatenate([np.linspace(-45, 45, 20011), np.linspace(-1e-3, 1e-3, 999), -np.logspace(-300, 0, 500)]).reshape(1, -1)
    zl = z.astype(np.longdouble)
    if kind == "gelu":
        p = np.where(z > 0, 1.0 - 0.5 * erfc(z / math.sqrt(2.0)).astype(np.longdouble), 0.5 * erfc(-z / math.sqrt(2.0)))
        want, slope = zl * p, p + zl * np.exp(-zl * zl / 2) / np.sqrt(2 * np.longdouble(math.pi))
    else:
        c = 2 * np.sqrt(2 / np.longdouble(math.pi))
        a = np.longdouble(0.044715)
        t, dt = (zl, 1) if kind == "silu" else (c * (zl + a * zl ** 3), c * (1 + 3 * a * zl * zl))
        s = 1 / (1 + np.exp(-t))
        want, slope = zl * s, s + zl * s * (1 / (1 + np.exp(t))) * dt
    dz, one, out = guarded(engine, z), guarded(engine, np.ones_like(z)), blank(engine, z.shape)
    check(engine.lib.rst_activation_forward(engine.handle, dz.ptr, None, out.ptr, z.size, ACTIVATIONS[kind]))
    within(out.get(), want, 16 * U * np.maximum(1.0, np.abs(z)), "value")
    check(engine.lib.rst_activation_backward(engine.handle, one.ptr, dz.ptr, None, out.ptr, z.size, ACTIVATIONS[kind]))
    within(out.get(), slope, 16 * U * np.maximum(1.0, np.abs(z)), "derivative")


@pytest.mark.parametrize("kind,limits", [("relu", (0.0, np.inf, 0.0)), ("gelu", (0.0, np.inf, np.nan)),
                                         ("gelu_tanh", (0.0, np.inf, np.nan)), ("silu", (0.0, np.inf, np.nan))])
def test_activation_limits(engine, kind, limits):
    z = np.array([[-np.inf, np.inf, np.nan, -1e308, 1e308, -1e3, 1e3, 0.0, -0.0, -5e-324]])
    out = blank(engine, z.shape)
    dz, one = guarded(engine, z), guarded(engine, np.ones_like(z))
    check(engine.lib.rst_activation_forward(engine.handle, dz.ptr, None, out.ptr, z.size, ACTIVATIONS[kind]))
    got = out.get()[0]
    assert np.array_equal(got[:3], np.array(limits), equal_nan=True)
    assert got[3] == 0.0 and got[4] == 1e308 and got[5] == 0.0 and got[6] == 1e3 and got[7] == 0.0 and abs(got[9]) <= 5e-324
    check(engine.lib.rst_activation_backward(engine.handle, one.ptr, dz.ptr, None, out.ptr, z.size, ACTIVATIONS[kind]))
    slope = out.get()[0]
    assert slope[0] == 0.0 and slope[1] == 1.0 and slope[3] == 0.0 and slope[4] == 1.0 and slope[5] == 0.0 and slope[6] == 1.0
    assert slope[2] == 0.0 if kind == "relu" else np.isnan(slope[2])


def test_residual_in_place(engine):
    for batch, k, n in ((1, 300, 77), (40, 130, 70), (300, 2048, 600)):
        _, x, w, b, res = data(batch, k, n)
        want = forward(engine, x, w, b, res, "gelu", pre=False)
        assert np.array_equal(forward(engine, x, w, b, res, "gelu", pre=False, in_place=True), want)


def test_input_gradient_in_place(engine):
    """grad_input written over input_pre or over residual_grad, grad_pre over grad or pre."""
    for batch, k, n in ((1, 300, 77), (40, 130, 70), (300, 2048, 600), (2050, 2046, 130)):
        rng, x, w, _, g = data(batch, k, n)
        pre, ip, res = rng.standard_normal((batch, n)), rng.standard_normal((batch, k)), rng.standard_normal((batch, k))
        want = backward(engine, g, pre, "silu", x, w, ip, "gelu", res)
        for over_input, over_grad in ((0, 0), (1, 1)):
            dg, dpre, dx, dw, dip, dres = (guarded(engine, a) for a in (g, pre, x, w, ip, res))
            gw, gb = blank(engine, (n, k)), blank(engine, (1, n))
            gp, gi = (dg, dpre)[over_grad], (dip, dres)[over_input]
            check(engine.lib.rst_linear_act_backward(
                engine.handle, dg.ptr, dpre.ptr, ACTIVATIONS["silu"], gp.ptr, dx.ptr, dw.ptr, gw.ptr, gb.ptr, gi.ptr, dip.ptr,
                ACTIVATIONS["gelu"], dres.ptr, batch, k, n))
            for a, b in zip((gp, gw, gb, gi), want):
                assert np.array_equal(a.get(), b)


def test_one_gradient_in_three_places(engine):
    """The residual block in place: the gradient that arrives is also the skipped one and where the result goes."""
    for batch, n in ((1, 40), (20, 40), (32, 100), (130, 33), (300, 600)):
        rng, x, w, _, g = data(batch, n, n)
        pre = rng.standard_normal((batch, n))
        want = backward(engine, g, pre, "gelu", x, w, None, "none", g)
        for grad_pre_over_pre in (False, True):
            dg, dpre, dx, dw = (guarded(engine, a) for a in (g, pre, x, w))
            gw, gb, gp = blank(engine, (n, n)), blank(engine, (1, n)), blank(engine, (batch, n))
            gp = dpre if grad_pre_over_pre else gp
            check(engine.lib.rst_linear_act_backward(
                engine.handle, dg.ptr, dpre.ptr, ACTIVATIONS["gelu"], gp.ptr, dx.ptr, dw.ptr, gw.ptr, gb.ptr, dg.ptr, None,
                ACTIVATIONS["none"], dg.ptr, batch, n, n))
            for a, b in zip((gp, gw, gb, dg), want):
                assert np.array_equal(a.get(), b)


def test_special_values_stay_in_their_row(engine):
    """A NaN or an infinity in one row of x reaches that row of the result and no other."""
    for batch, k, n in ((1, 64, 64), (6, 200, 90), (64, 500, 64), (600, 600, 200)):
        _, x, w, b, res = data(batch, k, n)
        clean = forward(engine, x, w, b, res, "silu")
        x[batch // 2, k // 2] = np.nan
        got = forward(engine, x, w, b, res, "silu")
        rest = [i for i in range(batch) if i != batch // 2]
        assert np.isnan(got[0][batch // 2]).all() and np.isnan(got[1][batch // 2]).all()
        assert np.array_equal(got[0][rest], clean[0][rest]) and np.array_equal(got[1][rest], clean[1][rest])


@pytest.mark.parametrize("batch", (1, 3, 40, 300))
def test_no_features_in(engine, batch):
    """Nothing to multiply: out = act(bias) + residual, z = bias."""
    rng = np.random.default_rng(batch)
    b, res = rng.standard_normal((1, 90)), rng.standard_normal((batch, 90))
    db, dres, out, pre = guarded(engine, b), guarded(engine, res), blank(engine, (batch, 90)), blank(engine, (batch, 90))
    check(engine.lib.rst_linear_act_forward(engine.handle, None, None, db.ptr, dres.ptr, pre.ptr, out.ptr, batch, 0, 90,
                                            ACTIVATIONS["silu"]))
    z = np.broadcast_to(b, (batch, 90))
    assert np.array_equal(pre.get(), z)
    want = act(z, "silu")[0] + res
    within(out.get(), want, act_bound(z) + 2 * U * np.abs(want), "act(bias) + residual")
