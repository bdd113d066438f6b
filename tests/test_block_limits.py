"""The residual-block entry points without a GPU, under ASan and UBSan: the launches' grids and the planners' arithmetic at
the ends of the extents they accept (tests/host_stub/block_limits_driver.cpp), and the addresses of grids that both
gradients of a layer share (block_grids_driver.cpp), and outputs over other arrays (block_overlap_driver.cpp)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_stub")


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs hipcc to compile the host side")
@pytest.mark.parametrize("driver,says", [("block_limits_driver", "block limits ok"), ("block_grids_driver", "block grids ok"),
                                         ("block_overlap_driver", "block overlap ok")])
def test_without_a_gpu(driver, says):
    build = subprocess.run(["make", "-C", HERE, "-j8", "-s"], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    run = subprocess.run([os.path.join(HERE, "build", driver)], capture_output=True, text=True, env=env,
                         timeout=300)
    assert run.returncode == 0, (run.stdout + run.stderr)[-4000:]
    assert says in run.stdout
    assert "ERROR: AddressSanitizer" not in run.stderr and "runtime error" not in run.stderr
