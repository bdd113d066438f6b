"""rst_layer_norm_forward / _backward through the C ABI, element by element against longdouble."""
import numpy as np
import pytest

from block_reference import U, address, blank, guarded, norm_backward, norm_forward, within

pytestmark = pytest.mark.gpu
EPS = 1e-5

# every edge of the widths that pick a kernel, odd widths, more rows than one workgroup takes
WIDTHS = [1, 2, 3, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 513, 1023, 1024, 1025, 2047, 2049, 4095,
          4096, 4097, 8191, 8193, 16383, 16385]
SHAPES = [(r, c) for c in WIDTHS for r in ((1, 37) if c > 100 else (1, 2, 33, 1030))] + \
         [(2500, 20), (3000, 130), (1500, 1000), (700, 4096), (300, 8190), (5, 32769), (70, 20001), (40000, 3)]


def data(rows, cols, seed=0):
    rng = np.random.default_rng(1000003 * rows + cols + seed)
    x = rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal((rows, 1))) + rng.standard_normal((rows, 1))
    return rng, x, 1.0 + 0.1 * rng.standard_normal((1, cols)), 0.1 * rng.standard_normal((1, cols))


def forward(engine, x, w, b, eps=EPS, shift=0, stats=True):
    rows, cols = x.shape
    dev = [guarded(engine, a, shift) for a in (x, w, b)]
    out = blank(engine, x.shape, shift)
    mean, rstd = (blank(engine, (rows, 1), shift), blank(engine, (rows, 1), shift)) if stats else (None, None)
    check(engine.lib.rst_layer_norm_forward(engine.handle, address(dev[0]), address(dev[1]), address(dev[2]), out.ptr,
                                            address(mean), address(rstd), rows, cols, eps))
    return (out.get(), mean.get(), rstd.get()) if stats else out.get()


def backward(engine, g, x, w, m, r, residual, shift=0, weight_grads=True):
    rows, cols = x.shape
    dev = [guarded(engine, a, shift) for a in (g, x, w, m, r, residual)]
    dx = blank(engine, x.shape, shift)
    dw, db = (blank(engine, (1, cols), shift), blank(engine, (1, cols), shift)) if weight_grads else (None, None)
    check(engine.lib.rst_layer_norm_backward(engine.handle, *[address(a) for a in dev], dx.ptr, address(dw), address(db),
                                             rows, cols))
    return (dx.get(), dw.get(), db.get()) if weight_grads else dx.get()


def check(status):
    from rstorch_amd import _ffi
    _ffi.check(status)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(engine, rows, cols):
    _, x, w, b = data(rows, cols)
    for wv, bv, shift in ((w, b, 0), (w, b, 1), (None, None, 0), (w, None, 0)):
        y, m, r, ey, em, er = norm_forward(x, wv, bv, EPS)
        got = forward(engine, x, wv, bv, shift=shift)
        within(got[0], y, ey, "out")
        within(got[1], m, em, "mean")
        within(got[2], r, er, "rstd")
        if shift == 1:  # the same arithmetic at any alignment, and without the statistics
            assert np.array_equal(forward(engine, x, wv, bv, stats=False), got[0])


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(engine, rows, cols):
    rng, x, w, _ = data(rows, cols)
    g, res = rng.standard_normal(x.shape), rng.standard_normal(x.shape)
    m = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + EPS)
    for wv, rv, shift in ((w, res, 0), (w, None, 1), (None, None, 0)):
        dx, dw, db, ex, ew, eb = norm_backward(g, x, wv, m, r, rv)
        got = backward(engine, g, x, wv, m, r, rv, shift)
        within(got[0], dx, ex, "grad_input")
        within(got[1], dw, ew, "grad_weight")
        within(got[2], db, eb, "grad_bias")
    again = backward(engine, g, x, None, m, r, None)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))  # a fixed order of additions
    assert np.array_equal(backward(engine, g, x, None, m, r, None, weight_grads=False), got[0])


@pytest.mark.parametrize("rows,cols", [(3, 7), (6, 33), (9, 257)])
def test_gradients_against_differences(engine, rows, cols):
    """Central differences of f = sum(g * y) with step h = 2^-17: the truncation is h^2 / 6 times the third
    derivative along one coordinate, at most 30 r^3 |g w| sqrt(cols) here (three factors r, xh bounded by sqrt(cols)
    only in a row with one large value), the rounding 2^-53 * sum|g y| * 16 / h."""
    rng, x, w, b = data(rows, cols, 7)
    g = rng.standard_normal(x.shape)
    h = 2.0 ** -17
    _, m, r = forward(engine, x, w, b)
    dx, dw, db = backward(engine, g, x, w, m, r, None)
    for _ in range(12):
        i, j = int(rng.integers(rows)), int(rng.integers(cols))
        hi, lo = x.copy(), x.copy()
        hi[i, j] += h
        lo[i, j] -= h
        # only row i changes; the difference of the rows' terms avoids the rounding of the others
        diff = (g[i] * (forward(engine, hi, w, b)[0][i] - forward(engine, lo, w, b)[0][i])).sum() / (hi[i, j] - lo[i, j])
        bound = h * h / 6 * 30 * float(r[i, 0]) ** 3 * np.abs(g[i] * w).max() * np.sqrt(cols) + \
            64 * U * np.abs(g[i]).sum() * (1 + np.abs(x[i]).max() * float(r[i, 0])) / h
        assert abs(diff - dx[i, j]) <= bound, (diff, dx[i, j], bound)
    # linear in weight and bias: the difference is exact but for rounding
    j = int(rng.integers(cols))
    hi = w.copy()
    hi[0, j] += 0.5
    diff = (g * (forward(engine, x, hi, b)[0] - forward(engine, x, w, b)[0])).sum() / 0.5 / rows
    assert abs(diff - dw[0, j]) <= 64 * U * np.abs(g).sum() * (1 + np.abs(x).max() * r.max())
    assert abs(g[:, j].mean() - db[0, j]) <= (rows + 256) * U * np.abs(g[:, j]).mean()


@pytest.mark.parametrize("cols", [100, 1000, 5000, 20000])
def test_rows_do_not_touch_each_other(engine, cols):
    """NaN and infinity stay in their row (and in the column sums); a row that is all one value has
    rstd = 1 / sqrt(eps) and normalises to 0."""
    rng, x, w, b = data(9, cols)
    clean = forward(engine, x, w, b)
    bad = x.copy()
    bad[2, cols // 2] = np.nan
    bad[5, 0] = np.inf
    bad[7] = 3.0
    got = forward(engine, bad, w, b)
    keep = [0, 1, 3, 4, 6, 8]
    for a, c in zip(got, clean):
        assert np.array_equal(a[keep], c[keep])
    assert np.isnan(got[0][2]).all() and np.isnan(got[0][5]).any()
    assert np.array_equal(got[0][7], np.broadcast_to(b, x.shape)[7]) and got[2][7, 0] == 1.0 / np.sqrt(EPS)
    g = rng.standard_normal(x.shape)
    a = backward(engine, g, x, w, clean[1], clean[2], None)
    m, r = clean[1].copy(), clean[2].copy()
    m[2] = np.nan
    c = backward(engine, g, x, w, m, r, None)
    rest = [i for i in range(9) if i != 2]
    assert np.array_equal(a[0][rest], c[0][rest]) and np.isnan(c[0][2]).all()
    assert np.isnan(c[1]).all() and np.array_equal(a[2], c[2])


def test_large_offset_keeps_its_digits(engine):
    """Values around 1e8 with unit spread: the variance is taken around the mean, so the result is as good
    as the inputs allow (element-wise bound of the forward pass)."""
    for cols in (200, 3000, 30000):
        _, x, w, b = data(4, cols)
        x = x + 1e8
        y, m, r, ey, em, er = norm_forward(x, w, b, EPS)
        got = forward(engine, x, w, b)
        within(got[0], y, ey, "out")
        within(got[2], r, er, "rstd")


@pytest.mark.parametrize("rows,cols", [(5, 60), (40, 1000), (3, 5000), (4, 20000)])
def test_in_place(engine, rows, cols):
    rng, x, w, b = data(rows, cols)
    want, m, r = forward(engine, x, w, b)
    dev = [guarded(engine, a) for a in (x, w, b)]
    check(engine.lib.rst_layer_norm_forward(engine.handle, dev[0].ptr, dev[1].ptr, dev[2].ptr, dev[0].ptr, None, None,
                                            rows, cols, EPS))
    assert np.array_equal(dev[0].get(), want)
    g, res = rng.standard_normal(x.shape), rng.standard_normal(x.shape)
    dx, dw, db = backward(engine, g, x, w, m, r, res)
    for target in range(3):
        d = [guarded(engine, a) for a in (g, x, res)]
        s = [guarded(engine, a) for a in (w, m, r)]
        ow, ob = blank(engine, (1, cols)), blank(engine, (1, cols))
        check(engine.lib.rst_layer_norm_backward(engine.handle, d[0].ptr, d[1].ptr, s[0].ptr, s[1].ptr, s[2].ptr,
                                                 d[2].ptr, d[target].ptr, ow.ptr, ob.ptr, rows, cols))
        assert np.array_equal(d[target].get(), dx) and np.array_equal(ow.get(), dw) and np.array_equal(ob.get(), db)
