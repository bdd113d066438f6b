"""rst_linear_act_backward where both gradients share a grid: the pairs of 128x128 tiles in either order, and 32x32 tiles of a
thin product beside a wide one.  Element by element, as in test_gpu_linear_act.py."""
import numpy as np
import pytest

from block_reference import ACTIVATIONS, address, blank, guarded, linear_backward, within

pytestmark = pytest.mark.gpu

# (batch, in, out): the input gradient has as many 128x128 tiles or fewer, and comes first ...
INPUT_FIRST = [(1024, 4096, 2000), (1023, 4095, 1111), (1000, 4090, 1025)]
# ... the weight gradient has fewer
WEIGHT_FIRST = [(1111, 4095, 1023)]
THIN = [(7, 4361, 4431), (21, 3858, 2909), (2186, 1794, 62), (13786, 282, 35), (3466, 2176, 7)]


@pytest.mark.parametrize("kind,input_kind,residual", [("none", "gelu", False), ("silu", "none", True)])
@pytest.mark.parametrize("batch,k,n", INPUT_FIRST + WEIGHT_FIRST + THIN)
def test_both_gradients(engine, batch, k, n, kind, input_kind, residual):
    from rstorch_amd import _ffi
    rng = np.random.default_rng(batch * 31 + k * 7 + n)
    g, pre, x, w = (rng.standard_normal(s) for s in ((batch, n), (batch, n), (batch, k), (n, k)))
    ip, res = rng.standard_normal((batch, k)), rng.standard_normal((batch, k))
    shift = k % 2
    dg, dpre, dx, dw, dip, dres = (guarded(engine, a, shift) for a in (g, pre, x, w, ip, res))
    gp, gw, gb, gi = (blank(engine, s, shift) for s in ((batch, n), (n, k), (1, n), (batch, k)))
    _ffi.check(engine.lib.rst_linear_act_backward(
        engine.handle, dg.ptr, dpre.ptr if kind != "none" else None, ACTIVATIONS[kind], gp.ptr if kind != "none" else None, dx.ptr,
        dw.ptr, gw.ptr, gb.ptr, gi.ptr, dip.ptr if input_kind != "none" else None, ACTIVATIONS[input_kind],
        address(dres) if residual else None, batch, k, n))
    want, bound = linear_backward(g, pre, kind, x, w, ip, input_kind, res if residual else None)
    for name, a, b, e in zip(("grad_pre", "grad_weight", "grad_bias", "grad_input"), (gp, gw, gb, gi), want, bound):
        if name != "grad_pre" or kind != "none":
            within(a.get(), b, e, name)
