"""rst_dropout_forward / _backward: every bit follows from value(seed, stream, index) >= p, which the CPU
restatement of the generator gives, so results are compared exactly."""
import numpy as np
import pytest

from block_reference import address, blank, guarded

pytestmark = pytest.mark.gpu


def check(status):
    from rstorch_amd import _ffi
    _ffi.check(status)


def run(engine, x, residual, p, seed, stream, shift=0, back=False):
    dev, res, out = guarded(engine, x, shift), guarded(engine, residual, shift), blank(engine, x.shape, shift)
    if back:
        check(engine.lib.rst_dropout_backward(engine.handle, dev.ptr, out.ptr, x.size, p, seed, stream))
    else:
        check(engine.lib.rst_dropout_forward(engine.handle, dev.ptr, address(res), out.ptr, x.size, p, seed, stream))
    return out.get()


def want(oracle, x, residual, p, seed, stream):
    u = oracle.fill_uniform((1, x.size), seed, stream).reshape(x.shape)
    y = np.where(u >= p, x * (1.0 / (1.0 - p)), 0.0)
    return y if residual is None else y + residual


@pytest.mark.parametrize("count", [1, 2, 3, 63, 64, 65, 127, 128, 129, 1000, 8191, 100003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1e-300])
def test_forward_and_backward_bits(engine, oracle, count, p):
    rng = np.random.default_rng(count)
    x, res = rng.standard_normal((1, count)), rng.standard_normal((1, count))
    for seed, stream, shift in ((0, 0, 0), (0xFFFFFFFFFFFFFFFF, 3, 1), (12345, 0xFFFFFFFFFFFFFFF1, 0)):
        assert np.array_equal(run(engine, x, None, p, seed, stream, shift), want(oracle, x, None, p, seed, stream))
        assert np.array_equal(run(engine, x, res, p, seed, stream, shift), want(oracle, x, res, p, seed, stream))
        assert np.array_equal(run(engine, x, None, p, seed, stream, shift, back=True), want(oracle, x, None, p, seed, stream))


def test_the_threshold_is_the_generator_value_itself(engine, oracle):
    """p equal to a value that is drawn keeps that element (value >= p); the next double above drops it."""
    u = oracle.fill_uniform((1, 64), 9, 4).reshape(-1)
    i = int(np.argsort(u)[32])
    x = np.ones((1, 64))
    assert run(engine, x, None, float(u[i]), 9, 4)[0, i] != 0.0
    assert run(engine, x, None, float(np.nextafter(u[i], 1.0)), 9, 4)[0, i] == 0.0


def test_dropped_values_are_zero_whatever_they_were(engine, oracle):
    x = np.array([[np.nan, np.inf, -np.inf, 1.0] * 50])
    y = run(engine, x, None, 0.5, 1, 2)
    kept = oracle.fill_uniform((1, x.size), 1, 2).reshape(x.shape) >= 0.5
    assert (y[~kept] == 0.0).all() and not np.signbit(y[~kept]).any()
    assert np.array_equal(y[kept], 2.0 * x[kept], equal_nan=True)


def test_share_and_independence_of_calls(engine):
    """2^20 draws at p = 0.3: the share kept is within 5 standard deviations (2.2e-3) of 0.7, and two streams agree
    on a share within 5 deviations (2.5e-3) of 0.7^2 + 0.3^2 = 0.58."""
    x = np.ones((1, 1 << 20))
    a, b = (run(engine, x, None, 0.3, 77, s) != 0.0 for s in (0, 1))
    assert abs(a.mean() - 0.7) <= 5 * np.sqrt(0.21 / x.size)
    assert abs((a == b).mean() - 0.58) <= 5 * np.sqrt(0.58 * 0.42 / x.size)


def test_in_place(engine, oracle):
    rng = np.random.default_rng(3)
    x, res = rng.standard_normal((1, 1001)), rng.standard_normal((1, 1001))
    expect = want(oracle, x, res, 0.4, 5, 6)
    for target in range(2):
        dev = [guarded(engine, a) for a in (x, res)]
        check(engine.lib.rst_dropout_forward(engine.handle, dev[0].ptr, dev[1].ptr, dev[target].ptr, x.size, 0.4, 5, 6))
        assert np.array_equal(dev[target].get(), expect)
