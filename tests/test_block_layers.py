"""Which calls the layers make, without a GPU: an engine that records the library's entry points instead of calling
them, under the Python Sequential and Residual; the C++ ones over a stand-in HIP runtime
(tests/host_stub/mirror_layers_driver.cpp)."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import rstorch_amd as rs

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_stub")


class Recorder:
    """Stands for an Engine: hands out addresses and notes the entry points by name."""

    device = 0

    def __init__(self):
        self.calls, self.handle, self._next = [], 1, 4096
        recorder = self

        class Lib:
            def __getattr__(self, name):
                def call(*args):
                    recorder.calls.append(name)
                    return 0
                return call

        self.lib = Lib()

    def malloc(self, count):
        self._next += 8 * int(count) + 4096
        return self._next

    def free(self, ptr):
        pass

    def empty(self, rows, cols):
        return rs.Array2(self, rows, cols)

    zeros = empty

    def full(self, rows, cols, value):
        return self.empty(rows, cols)

    def normal(self, rows, cols, *args):
        return self.empty(rows, cols)

    def from_numpy(self, host):
        return self.empty(*host.shape)

    def taken(self):
        calls, self.calls = self.calls, []
        return calls


@pytest.fixture
def recorder():
    return Recorder()


def overridden(base):
    """A subclass with passes of its own, which note that they ran."""

    class Own(base):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            self.ran = []

        def forward(self, input):
            self.ran.append("forward")
            return super().forward(input)

        def backward(self, gradient):
            self.ran.append("backward")
            return super().backward(gradient)

    return Own


def neighbours(recorder, layer, where):
    lin = lambda: rs.Linear(6, 6, engine=recorder)
    return {"behind": [lin(), layer], "between": [lin(), layer, lin()], "in front": [layer, lin()],
            "between a Linear and its activation": [lin(), layer, rs.GELU()],
            "between an activation and a Linear": [rs.GELU(), layer, lin()]}[where]


WHERE = ["behind", "between", "in front", "between a Linear and its activation", "between an activation and a Linear"]


@pytest.mark.parametrize("where", WHERE)
@pytest.mark.parametrize("base", [rs.GELU, rs.SiLU, rs.ReLU, rs.Dropout, rs.Identity])
@pytest.mark.parametrize("outer", [rs.Sequential, rs.Residual])
def test_an_overridden_layer_is_called(recorder, base, where, outer):
    layer = overridden(base)()
    model = outer(neighbours(recorder, layer, where))
    x = recorder.empty(4, 6)
    model.forward(x)
    assert layer.ran == ["forward"]
    model.backward(recorder.empty(4, 6))
    assert layer.ran == ["forward", "backward"]


@pytest.mark.parametrize("first", [True, False])
def test_an_overridden_norm_is_called(recorder, first):
    layer = overridden(rs.LayerNorm)(6, engine=recorder)
    inner = [layer, rs.Linear(6, 6, engine=recorder)]
    model = rs.Residual(inner if first else inner[::-1])
    model.forward(recorder.empty(4, 6))
    model.backward(recorder.empty(4, 6))
    assert layer.ran == ["forward", "backward"]


def test_an_overridden_sequential_is_called(recorder):
    inner = overridden(rs.Sequential)([rs.Linear(6, 6, engine=recorder), rs.GELU()])
    for model in (rs.Residual(inner), rs.Residual([inner]), rs.Sequential([inner])):
        model.forward(recorder.empty(4, 6))
        model.backward(recorder.empty(4, 6))
        assert inner.ran == ["forward", "backward"]
        inner.ran = []


@pytest.mark.parametrize("kind", ["gelu", "relu"])
def test_an_overridden_identity_keeps_its_place(recorder, kind):
    """What it is given lies in front of the activation behind it."""
    act = {"gelu": rs.GELU, "relu": rs.ReLU}[kind]()
    name = {"gelu": "rst_activation_", "relu": "rst_relu_"}[kind]
    model = rs.Sequential([rs.Linear(6, 6, engine=recorder), overridden(rs.Identity)(), act, overridden(rs.Identity)(),
                           rs.Linear(6, 6, engine=recorder)])
    recorder.taken()
    model.forward(recorder.empty(4, 6))
    assert recorder.taken() == ["rst_linear_forward", name + "forward", "rst_linear_forward"]
    model.backward(recorder.empty(4, 6))
    assert recorder.taken() == ["rst_linear_backward", name + "backward", "rst_linear_backward"]


def test_a_linear_takes_its_neighbours_work(recorder):
    """The layers themselves (not subclasses) stay joined."""
    model = rs.Residual([rs.Linear(6, 9, engine=recorder), rs.GELU(), rs.Identity(), rs.Linear(9, 6, engine=recorder)])
    recorder.taken()
    model.forward(recorder.empty(4, 6))
    assert recorder.taken() == ["rst_linear_act_forward"] * 2
    model.backward(recorder.empty(4, 6))
    assert recorder.taken() == ["rst_linear_act_backward"] * 2


class Resize(rs.Module):
    """A layer of the caller's own that returns another width than it is given."""

    def __init__(self, size):
        self.size = size

    def forward(self, input):
        self.given = input.cols
        return input.engine.empty(input.rows, self.size)

    def backward(self, gradient):
        return gradient.engine.empty(gradient.rows, self.given)


def test_a_residual_around_layers_that_change_the_width(recorder):
    lin = lambda k, n: rs.Linear(k, n, engine=recorder)
    for inner in ([lin(6, 9), Resize(6)], [Resize(9), lin(9, 6)], [lin(6, 9), Resize(5), lin(5, 7), Resize(6)],
                  [rs.Sequential([lin(6, 9), Resize(6)])], [lin(6, 9), Resize(6), rs.Dropout(0.5)]):
        model = rs.Residual(inner)
        assert model.forward(recorder.empty(4, 6)).shape == (4, 6)
        assert model.backward(recorder.empty(4, 6)).shape == (4, 6)
    # what does not fit is still refused; where the layers tell their width, before any of them runs
    for inner in ([lin(6, 9)], [Resize(6), lin(6, 9)], [Resize(9)], [lin(6, 9), Resize(8)], [lin(6, 9), Resize(8), rs.Dropout(0.5)]):
        recorder.taken()
        with pytest.raises(rs.ShapeError):
            rs.Residual(inner).forward(recorder.empty(4, 6))
        assert not recorder.taken() or isinstance(inner[1], Resize)


@pytest.mark.parametrize("first", [rs.GELU, rs.SiLU, rs.ReLU, rs.Dropout, rs.Identity])
@pytest.mark.parametrize("outer", [rs.Sequential, rs.Residual])
def test_host_arrays_go_to_the_engine_of_the_layers(recorder, monkeypatch, first, outer):
    """Layers on an engine of their own (another stream, possibly another GPU): nothing of theirs runs on the default one."""
    other = Recorder()
    monkeypatch.setattr("rstorch_amd.engine.default_engine", lambda: other)
    monkeypatch.setattr("rstorch_amd.module.default_engine", lambda: other)
    monkeypatch.setattr(rs.Sequential, "compile_enabled", False)  # (a compiled list keeps to its layers' engine anyway)
    lin = lambda: rs.Linear(6, 6, engine=recorder)
    x = np.zeros((4, 6))
    for inner in ([first(), lin()], [first(), rs.LayerNorm(6, engine=recorder), first()], [lin(), first()],
                  [first(), rs.Sequential([lin()])], [first(), rs.Residual([first(), lin()])]):
        model = outer(inner)
        out = model.forward(x)
        assert out.engine is recorder
        assert rs.as_array2(model.backward(x)).engine is recorder
    assert not other.taken()
    if outer is rs.Residual:  # an array that another engine handed over: the gradient belongs to the layers' engine
        given, seen = Recorder(), []
        monkeypatch.setattr(recorder, "from_numpy", lambda host: seen.append(host.shape) or recorder.empty(*host.shape))
        monkeypatch.setattr(given, "from_numpy", None)
        model = outer([lin()])
        model.forward(given.empty(4, 6))
        model.backward(x)
        assert seen == [x.shape]
    # layers that are bound to no engine keep using the default one
    assert outer([rs.GELU(), rs.Dropout(0.5)]).forward(x).engine is other


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs hipcc to compile the host side")
def test_layers_of_the_cpp_mirror():
    build = subprocess.run(["make", "-C", HOST, "-j8", "-s"], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([os.path.join(HOST, "build", "mirror_layers_driver")], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "mirror layers ok" in run.stdout, (run.stdout + run.stderr)[-3000:]
