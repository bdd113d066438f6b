"""The residual block's operators where an extent is so large that a launch is cut into several."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def check(status):
    from rstorch_amd import _ffi
    _ffi.check(status)


def window(engine, array, first, count):
    """`count` values from number `first` of an array on, on the host."""
    import rstorch_amd as rs
    return rs.Array2(engine, 1, count, ptr=array.ptr + 8 * first, owner=array).to_numpy()[0]


@pytest.mark.parametrize("batch,features", [(1, (1 << 26) + 5), (3, (1 << 25) + 5), (8, (1 << 25) + 1)])
def test_few_rows_of_very_many_features(engine, batch, features):
    """One value in: out = x w + b in one fused step and one addition, so every element is known to the bit; where one launch
    ends and the next begins (2^25 features), at both ends of every row, and behind the last one."""
    x, w, b = engine.uniform(batch, 1, 5, 1, -1.0, 1.0), engine.uniform(features, 1, 5, 2, -1.0, 1.0), engine.uniform(1, features, 5, 3)
    out = engine.full(1, batch * features + 64, -7.0)
    check(engine.lib.rst_linear_act_forward(engine.handle, x.ptr, w.ptr, b.ptr, None, None, out.ptr, batch, 1, features, 0))
    xs = x.to_numpy()[:, 0]
    for first in (0, 12345, (1 << 25) - 64, (1 << 25), features - 64):
        count = min(64, features - first)
        ws, bs = window(engine, w, first, count), window(engine, b, first, count)
        for row in range(batch):
            assert np.array_equal(window(engine, out, row * features + first, count), ws * xs[row] + bs), (row, first)
    assert np.array_equal(window(engine, out, batch * features, 64), np.full(64, -7.0))
