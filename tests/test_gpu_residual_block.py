"""The residual block's operators together, as a user runs them: through the Python layers against a plain
numpy network, through the C++ layers, recorded into a graph and replayed, on two engines at once.

Tolerance of the networks: max|got - want| / max|want| <= 1e-10 per tensor, the framework's bound for logits
and gradients (each operator alone is held element by element to a bound of some 1e-15 in its own test)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from block_reference import U, act, blank, guarded
from conftest import rel_err

pytestmark = pytest.mark.gpu
TOL = 1e-10


def check(status):
    from rstorch_amd import _ffi
    _ffi.check(status)


class Plain:
    """x + dropout(act(LN(x) w1^T + b1) w2^T + b2), forward and backward, in numpy."""

    def __init__(self, kind, w1, b1, w2, b2, lw, lb):
        self.kind, self.w1, self.b1, self.w2, self.b2, self.lw, self.lb = kind, w1, b1, w2, b2, lw, lb

    def forward(self, x, mask):
        m = x.mean(1, keepdims=True)
        self.r = 1.0 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + 1e-5)
        self.xh = (x - m) * self.r
        self.y = self.xh * self.lw + self.lb
        self.z = self.y @ self.w1.T + self.b1
        self.a, self.slope = act(self.z, self.kind)
        self.mask = mask
        return x + mask * (self.a @ self.w2.T + self.b2)

    def backward(self, g):
        n = g.shape[0]
        d = g * self.mask
        gw2, gb2 = d.T @ self.a / n, d.mean(0, keepdims=True)
        dz = (d @ self.w2) * self.slope
        gw1, gb1 = dz.T @ self.y / n, dz.mean(0, keepdims=True)
        dy = dz @ self.w1
        u = dy * self.lw
        dx = self.r * (u - u.mean(1, keepdims=True) - self.xh * (u * self.xh).mean(1, keepdims=True))
        return g + dx, [(dy * self.xh).mean(0, keepdims=True), dy.mean(0, keepdims=True), gw1, gb1, gw2, gb2]


def arrays(width, hidden, seed):
    rng = np.random.default_rng(seed)
    return (rng, rng.standard_normal((hidden, width)) / np.sqrt(width), 0.1 * rng.standard_normal((1, hidden)),
            rng.standard_normal((width, hidden)) / np.sqrt(hidden), 0.1 * rng.standard_normal((1, width)),
            1.0 + 0.1 * rng.standard_normal((1, width)), 0.1 * rng.standard_normal((1, width)))


def layers(rs, kind):
    return {"relu": rs.ReLU, "gelu": rs.GELU, "gelu_tanh": lambda: rs.GELU(approximate=True), "silu": rs.SiLU}[kind]()


@pytest.mark.parametrize("batch,width,hidden,kind", [(1, 64, 256, "gelu"), (32, 100, 400, "gelu"), (33, 101, 403, "silu"),
                                                     (257, 384, 1024, "relu"), (1000, 512, 2047, "gelu_tanh")])
def test_block_of_the_python_layers(engine, oracle, batch, width, hidden, kind):
    import rstorch_amd as rs
    rng, w1, b1, w2, b2, lw, lb = arrays(width, hidden, batch)
    norm = rs.LayerNorm(width)
    norm.weight.assign(lw)
    norm.bias.assign(lb)
    block = rs.Residual([norm, rs.Linear.new_with_kernel(width, hidden, rs.FromArrays(w1, b1)), layers(rs, kind),
                         rs.Identity(), rs.Linear.new_with_kernel(hidden, width, rs.FromArrays(w2, b2)),
                         rs.Dropout(0.3, seed=99)])
    plain = Plain(kind, w1.copy(), b1.copy(), w2.copy(), b2.copy(), lw.copy(), lb.copy())
    optim = rs.SGD.new(0.05)
    for step in range(3):
        x, g = rng.standard_normal((batch, width)), rng.standard_normal((batch, width))
        mask = (oracle.fill_uniform((batch, width), 99, step) >= 0.3) / (1.0 - 0.3)
        assert rel_err(block.forward(x).to_numpy(), plain.forward(x, mask)) <= TOL
        gx = block.backward(g).to_numpy()
        want_gx, grads = plain.backward(g)
        assert rel_err(gx, want_gx) <= TOL
        params = list(block.parameters())
        assert len(params) == 6
        for p, want in zip(params, grads):
            assert rel_err(p.grad.to_numpy(), want) <= TOL
        optim.step(block)
        for name, want in zip(("lw", "lb", "w1", "b1", "w2", "b2"), grads):
            getattr(plain, name)[...] -= 0.05 * want
    block.eval()
    x = rng.standard_normal((batch, width))
    assert rel_err(block.forward(x).to_numpy(), plain.forward(x, 1.0)) <= TOL
    with pytest.raises(rs.ShapeError):
        block.backward(np.zeros((batch, width + 1)))
    block.backward(np.ones((batch, width)))
    with pytest.raises(rs.StateError):
        block.backward(np.ones((batch, width)))


def inner_variants(rs, width):
    lin = [rs.Linear(width, width) for _ in range(2)]
    return {
        "linear": [lin[0]], "linear_gelu": [lin[0], rs.GELU()], "linear_relu": [lin[0], rs.Identity(), rs.ReLU()],
        "relu_linear": [rs.ReLU(), lin[0]], "gelu_linear": [rs.GELU(), rs.Identity(), lin[0]],
        "silu_linear_silu": [rs.SiLU(), lin[0], rs.SiLU()], "norm": [rs.LayerNorm(width)], "identity": [rs.Identity()],
        "empty": [], "activation": [rs.GELU()], "two_linears": [lin[0], lin[1]], "softmax_last": [lin[0], rs.Softmax()],
        "nested": [rs.Sequential([lin[0], rs.ReLU(), lin[1]])], "linear_norm_gelu": [lin[0], rs.LayerNorm(width), rs.GELU()],
    }


@pytest.mark.parametrize("name", ["linear", "linear_gelu", "linear_relu", "relu_linear", "gelu_linear", "silu_linear_silu",
                                  "norm", "identity", "empty", "activation", "two_linears", "softmax_last", "nested",
                                  "linear_norm_gelu"])
def test_residual_equals_the_layers_one_by_one(engine, name):
    """Whoever does the addition: x + inner(x) and g + inner'(g) as the layers give them one call at a time."""
    import rstorch_amd as rs
    rng = np.random.default_rng(len(name))
    inner = inner_variants(rs, 24)[name]
    x, g = rng.standard_normal((19, 24)), rng.standard_normal((19, 24))
    block = rs.Residual(inner)
    got, got_g = block.forward(x).to_numpy(), block.backward(g).to_numpy()
    y = rs.as_array2(x)
    for layer in inner:
        y = layer.forward(y)
    want = x + y.to_numpy()
    d = rs.as_array2(g)
    for layer in reversed(inner):
        d = layer.backward(d)
    want_g = g + d.to_numpy()
    assert rel_err(got, want) <= 1e-12 and rel_err(got_g, want_g) <= 1e-12


def test_shapes_that_do_not_fit_are_refused(engine):
    import rstorch_amd as rs

    class Wider(rs.Module):
        def forward(self, input):
            return engine.zeros(input.rows, input.cols + 5)

    x = np.zeros((4, 6))
    with pytest.raises(rs.ShapeError):
        rs.Residual([rs.Linear(6, 7)]).forward(x)
    with pytest.raises(rs.ShapeError):
        rs.Residual([Wider()]).forward(x)
    with pytest.raises(rs.ShapeError):
        rs.Residual([Wider(), rs.Dropout(0.5)]).forward(x)
    with pytest.raises(rs.ShapeError):
        rs.LayerNorm(7).forward(x)
    norm, gelu = rs.LayerNorm(6), rs.GELU()
    norm.forward(x), gelu.forward(x)
    for layer in (norm, gelu):
        with pytest.raises(rs.ShapeError):
            layer.backward(np.zeros((4, 5)))
        layer.backward(np.zeros((4, 6)))  # the refused call has not taken the cache
    with pytest.raises(rs.StateError):
        rs.LayerNorm(3).parameters()
    # one activation object in two places: its second use has another shape than the layer behind the first
    shared = rs.GELU()
    twice = rs.Sequential([shared, rs.Linear(6, 9), shared, rs.Linear(9, 2)])
    twice.forward(x)
    with pytest.raises((rs.ShapeError, rs.StateError)):
        twice.backward(np.zeros((4, 2)))


def test_sequential_trains_through_a_block_with_the_loss(engine, oracle):
    """Gradients of a whole network by central differences of its loss (h = 2^-16): truncation below
    h^2 * 1e2 * loss scale, rounding 1e-13 / h: 1e-6 covers both for values of order 1."""
    import rstorch_amd as rs
    rng = np.random.default_rng(5)
    net = rs.Sequential([rs.Linear(12, 16), rs.Residual([rs.LayerNorm(16), rs.Linear(16, 24), rs.GELU(), rs.Linear(24, 16)]),
                         rs.LayerNorm(16), rs.Linear(16, 5)])
    x, y = rng.standard_normal((9, 12)), np.eye(5)[rng.integers(0, 5, 9)]
    loss = rs.CrossEntropyLoss.new()
    loss.forward(net.forward(x), y)
    net.backward(loss.backward())
    params = [(p.parm, p.grad.to_numpy()) for p in net.parameters()]
    assert len(params) == 2 + 6 + 2 + 2
    h = 2.0 ** -16
    for parm, grad in params:
        host = parm.to_numpy()
        for _ in range(3):
            at = tuple(int(rng.integers(s)) for s in host.shape)
            values = []
            for sign in (1, -1):
                moved = host.copy()
                moved[at] += sign * h
                parm.assign(moved)
                values.append(loss.forward(net.forward(x), y))
            parm.assign(host)
            assert abs((values[0] - values[1]) / (2 * h) - grad[at]) <= 1e-6


def test_mirror_in_cpp():
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rstorch_amd", "cpp", "bin", "test_block")
    assert os.path.exists(exe), "build the C++ mirror first (__graft_entry__.build())"
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "all block tests passed" in out.stdout, out.stdout + out.stderr


# ---- a chain of calls, eager, recorded, on two engines ---------------------------------------------
class Chain:
    """LayerNorm, Linear + GELU, Linear, dropout + residual and back again, on guarded buffers of one engine."""

    def __init__(self, engine, batch, width, hidden, seed):
        from rstorch_amd import _ffi
        self.engine, self.dims, self.ffi = engine, (batch, width, hidden), _ffi
        rng, w1, b1, w2, b2, lw, lb = arrays(width, hidden, seed)
        self.inputs = {"x": rng.standard_normal((batch, width)), "g": rng.standard_normal((batch, width)), "w1": w1, "b1": b1,
                       "w2": w2, "b2": b2, "lw": lw, "lb": lb}
        self.dev = {k: guarded(engine, v) for k, v in self.inputs.items()}
        bw, bh = (batch, width), (batch, hidden)
        self.out = {k: blank(engine, s) for k, s in dict(
            y=bw, mean=(batch, 1), rstd=(batch, 1), a=bh, z=bh, h=bw, out=bw, d=bw, dz=bh, dy=bw, dx=bw, gw1=w1.shape, gb1=b1.shape,
            gw2=w2.shape, gb2=b2.shape, glw=lw.shape, glb=lb.shape).items()}

    def launch(self):
        L, e, f = self.engine.lib, self.engine.handle, self.ffi
        batch, width, hidden = self.dims
        i = {k: v.ptr for k, v in self.dev.items()}
        o = {k: v.ptr for k, v in self.out.items()}
        n = batch * width
        check(L.rst_layer_norm_forward(e, i["x"], i["lw"], i["lb"], o["y"], o["mean"], o["rstd"], batch, width, 1e-5))
        check(L.rst_linear_act_forward(e, o["y"], i["w1"], i["b1"], None, o["z"], o["a"], batch, width, hidden, f.ACT_GELU))
        check(L.rst_linear_act_forward(e, o["a"], i["w2"], i["b2"], None, None, o["h"], batch, hidden, width, f.ACT_NONE))
        check(L.rst_dropout_forward(e, o["h"], i["x"], o["out"], n, 0.2, 11, 12))
        check(L.rst_dropout_backward(e, i["g"], o["d"], n, 0.2, 11, 12))
        check(L.rst_linear_act_backward(e, o["d"], None, f.ACT_NONE, None, o["a"], i["w2"], o["gw2"], o["gb2"], o["dz"], o["z"],
                                        f.ACT_GELU, None, batch, hidden, width))
        check(L.rst_linear_act_backward(e, o["dz"], None, f.ACT_NONE, None, o["y"], i["w1"], o["gw1"], o["gb1"], o["dy"], None,
                                        f.ACT_NONE, None, batch, width, hidden))
        check(L.rst_layer_norm_backward(e, o["dy"], i["x"], i["lw"], o["mean"], o["rstd"], i["g"], o["dx"], o["glw"], o["glb"],
                                        batch, width))

    def results(self):
        return {k: v.get() for k, v in self.out.items()}

    def wipe(self):
        for v in self.out.values():
            check(self.engine.lib.rst_fill(self.engine.handle, v.ptr, v.size, 123.0))


CHAINS = [(1, 64, 256), (37, 101, 403), (300, 1024, 2048)]


@pytest.mark.parametrize("batch,width,hidden", CHAINS)
def test_recorded_graph_replays_the_eager_results(engine, batch, width, hidden):
    """Two recorded graphs of one engine, replayed in turn with eager work, synchronisations and changed inputs between
    the replays; every replay against the eager launches, bit for bit."""
    hip = ctypes.CDLL("libamdhip64.so.7")
    stream = ctypes.c_void_p(engine.lib.rst_engine_stream(engine.handle))
    chains = [Chain(engine, batch, width, hidden, s) for s in (1, 2)]
    execs = []
    for c in chains:
        c.launch()
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 1) == 0  # thread-local
        try:
            c.launch()
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        assert hip.hipGraphDestroy(graph) == 0
        execs.append(exe)
    for turn in range(4):
        for c in chains:  # other inputs than at the recording
            c.inputs["x"] = c.inputs["x"] * 0.9 + turn
            check(engine.lib.rst_upload(engine.handle, c.dev["x"].ptr, c.inputs["x"].ctypes.data_as(c.ffi.c_double_p),
                                        c.inputs["x"].size))
        want = []
        for c in chains:
            c.launch()
            want.append(c.results())
            c.wipe()
        for exe in execs if turn % 2 else execs[::-1]:
            assert hip.hipGraphLaunch(exe, stream) == 0
        engine.zeros(3, 3).to_numpy()
        for c, w in zip(chains, want):
            got = c.results()
            for k in w:
                assert np.array_equal(got[k], w[k]), (turn, k)
    engine.synchronize()
    for exe in execs:
        assert hip.hipGraphExecDestroy(exe) == 0


def test_two_engines_at_once(engine):
    """Each engine has its own stream and scratch: chains that run side by side give what they give alone."""
    import rstorch_amd as rs
    other = rs.Engine(0)
    chains = [Chain(e, *dims, seed) for seed, (e, dims) in enumerate([(engine, CHAINS[2]), (other, CHAINS[2]),
                                                                      (other, CHAINS[1]), (engine, CHAINS[1])])]
    want = []
    for c in chains:
        c.launch()
        c.engine.synchronize()
        want.append(c.results())
        c.wipe()
        c.engine.synchronize()
    for _ in range(3):
        for c in chains:
            c.launch()
    for c, w in zip(chains, want):
        got = c.results()
        for k in w:
            assert np.array_equal(got[k], w[k]), k
    del chains
    other.synchronize()


def test_hand_over_between_engines(engine):
    """An array that one engine writes and another reads, ordered by an event."""
    import rstorch_amd as rs
    other = rs.Engine(0)
    rng = np.random.default_rng(8)
    x = rng.standard_normal((500, 700))
    src, mid, out = engine.from_numpy(x), engine.empty(500, 700), engine.empty(500, 700)
    engine.synchronize()
    for _ in range(5):
        check(engine.lib.rst_dropout_forward(engine.handle, src.ptr, None, mid.ptr, x.size, 0.5, 1, 1))
        other.wait_event(engine.event().record())
        check(other.lib.rst_layer_norm_forward(other.handle, mid.ptr, None, None, out.ptr, None, None, 500, 700, 1e-5))
        engine.wait_event(other.event().record())
    got = out.to_numpy()
    d = mid.to_numpy()
    want = (d - d.mean(1, keepdims=True)) / np.sqrt(d.var(1, keepdims=True) + 1e-5)
    assert np.abs(got - want).max() <= 4096 * U * np.abs(want).max()
    other.synchronize()
