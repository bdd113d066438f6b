"""Layer norm where a workgroup takes more than one turn of rows, at widths that do not fill its threads: the next row's
loads are issued ahead (or not, above 4096 columns backward and 8192 forward) and the last pair of a row is loaded from its
last two columns.  Element by element, as in test_gpu_layer_norm.py."""
import numpy as np
import pytest

from block_reference import blank, guarded, norm_backward, norm_forward, within
from test_gpu_layer_norm import EPS, backward, check, data, forward

pytestmark = pytest.mark.gpu

# rows just above what the grid takes in one turn: forward 1280 workgroups of one row up to 2048 columns, 512 up to 4096, 256
# up to 16384; backward 8192 rows up to 64 columns, 4096 up to 128, 2048 up to 512, 1024 up to 1024, 512 up to 2048, 256 above
FORWARD = [(1300, 1025), (1290, 2047), (2570, 1535), (530, 2049), (1030, 3071), (530, 4095), (270, 4097), (520, 8191), (270, 8193),
           (520, 12289), (260, 16383)]
BACKWARD = [(16400, 15), (8300, 17), (8200, 33), (16500, 63), (4200, 65), (8210, 127), (2100, 129), (4100, 511), (1100, 513), (2060, 1023),
            (530, 1025), (1300, 2047), (300, 2049), (530, 4095), (270, 4097), (530, 8191)]


@pytest.mark.parametrize("rows,cols", FORWARD)
def test_forward(engine, rows, cols):
    _, x, w, b = data(rows, cols)
    y, m, r, ey, em, er = norm_forward(x, w, b, EPS)
    for shift in (0, 1):
        got = forward(engine, x, w, b, shift=shift)
        within(got[0], y, ey, "out")
        within(got[1], m, em, "mean")
        within(got[2], r, er, "rstd")
    over = guarded(engine, x, 1)  # in place: a row's loads are ahead of other rows' stores, never behind its own
    dw, db = guarded(engine, w), guarded(engine, b)
    check(engine.lib.rst_layer_norm_forward(engine.handle, over.ptr, dw.ptr, db.ptr, over.ptr, None, None, rows, cols, EPS))
    assert np.array_equal(over.get(), got[0])


@pytest.mark.parametrize("rows,cols", BACKWARD)
def test_backward(engine, rows, cols):
    rng, x, w, _ = data(rows, cols)
    g, res = rng.standard_normal(x.shape), rng.standard_normal(x.shape)
    m = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + EPS)
    dx, dw, db, ex, ew, eb = norm_backward(g, x, w, m, r, res)
    for shift in (0, 1):
        got = backward(engine, g, x, w, m, r, res, shift)
        within(got[0], dx, ex, "grad_input")
        within(got[1], dw, ew, "grad_weight")
        within(got[2], db, eb, "grad_bias")
    for target in range(3):
        d = [guarded(engine, a, 1) for a in (g, x, res)]
        s = [guarded(engine, a, 1) for a in (w, m, r)]
        ow, ob = blank(engine, (1, cols)), blank(engine, (1, cols))
        check(engine.lib.rst_layer_norm_backward(engine.handle, d[0].ptr, d[1].ptr, s[0].ptr, s[1].ptr, s[2].ptr, d[2].ptr,
                                                 d[target].ptr, ow.ptr, ob.ptr, rows, cols))
        for a, want in zip((d[target], ow, ob), got):
            assert np.array_equal(a.get(), want)
