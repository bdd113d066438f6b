"""The residual-block entry points on the host: their refusals, the launches of accepted shapes, no allocation
or wait inside a stream capture (tests/host_stub/block_ops_driver.cpp, under ASan and UBSan), and what the
Python layers refuse before any call into the library."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_stub")


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs hipcc to compile the host side")
def test_refusals_and_planners_without_a_gpu():
    build = subprocess.run(["make", "-C", HERE, "-j8", "-s"], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    run = subprocess.run([os.path.join(HERE, "build", "block_ops_driver")], capture_output=True, text=True, env=env,
                         timeout=300)
    assert run.returncode == 0, (run.stdout + run.stderr)[-4000:]
    assert "block ops ok" in run.stdout
    assert "ERROR: AddressSanitizer" not in run.stderr and "runtime error" not in run.stderr


@pytest.mark.parametrize("p", [-0.1, 1.0, 2.0, float("nan")])
def test_dropout_refuses_what_is_no_probability(p):
    import rstorch_amd as rs
    with pytest.raises(ValueError):
        rs.Dropout(p)


def test_backward_without_a_forward():
    import rstorch_amd as rs
    for layer in (rs.GELU(), rs.SiLU(), rs.Dropout(0.5), rs.Residual([rs.GELU()])):
        with pytest.raises(rs.StateError):
            layer.backward(None)
        assert len(layer.parameters()) == 0


def test_names():
    import rstorch_amd as rs
    m = rs.Residual([rs.GELU.new(), rs.Dropout.new(0.25), rs.SiLU()])
    assert repr(m) == "Residual(GELU, Dropout(0.25), SiLU)"
    m.eval()
    assert not m.inner.layers[1].training
    m.train()
    assert m.inner.layers[1].training
