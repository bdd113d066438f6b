"""Workloads of the residual-block operators: layer norm, dropout and the Linear layer with activation and
residual in its epilogue, each forward and backward, f64.

``run`` computes a pass in elementary torch operations, or, with ``own`` set, through the C ABI of
``rstorch_amd`` on the same buffers.  The products, sums and exponentials are in 64 bits, the type of the
framework's arrays."""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
F64 = torch.float64
EPS = 1e-5

# activations of the Linear epilogue, by the names the cases use
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


# ---- cases ---------------------------------------------------------------------------------------
def _norm(name, direction, rows, cols, residual=False, stats=True, affine=True):
    c = {"op": "layer_norm_" + direction, "rows": rows, "cols": cols, "affine": affine}
    if direction == "forward":
        c["stats"] = stats
    else:
        c["residual"] = residual
    return dict(c, name=name) if name else c


def _dropout(name, direction, rows, cols, p, residual=False):
    c = {"op": "dropout_" + direction, "rows": rows, "cols": cols, "p": p}
    if direction == "forward":
        c["residual"] = residual
    return dict(c, name=name) if name else c


def _linear_forward(name, batch, k, n, act, pre, residual, bias=True):
    c = {"op": "linear_forward", "batch": batch, "in": k, "out": n, "act": act, "pre": pre, "residual": residual,
         "bias": bias}
    return dict(c, name=name) if name else c


def _linear_backward(name, batch, k, n, act, input_act, residual):
    c = {"op": "linear_backward", "batch": batch, "in": k, "out": n, "act": act, "input_act": input_act,
         "residual": residual}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one batch of the README network's hidden layer: launch latency
        _norm("norm forward 32x100", "forward", 32, 100),
        # a long batch of the hidden width of the deep network: training keeps the statistics
        _norm("norm forward 16384x4096", "forward", 16384, 4096),
        # every extent odd, no 16-byte aligned rows
        _norm("norm backward 2047x1023", "backward", 2047, 1023),
        # the block's backward pass at the hidden width: the gradient of the residual path joins in
        _norm("norm backward 8192x4096", "backward", 8192, 4096, residual=True),
        _dropout("dropout forward 32x100", "forward", 32, 100, 0.5),
        # the end of a residual block, odd extents
        _dropout("dropout residual 2047x4095", "forward", 2047, 4095, 0.1, residual=True),
        _dropout("dropout backward 16384x4096", "backward", 16384, 4096, 0.1),
        # a single row through the block's last layer: serving, the weights are read once
        _linear_forward("linear forward 1x4096x4096", 1, 4096, 4096, "none", False, True),
        # the block's first layer in training: the pre-activation is kept for the backward pass
        _linear_forward("linear forward 2048x1024x4096", 2048, 1024, 4096, "gelu", True, False),
        # inference through odd extents, activation and residual both
        _linear_forward("linear forward 1023x4095x1023", 1023, 4095, 1023, "silu", False, True),
        # the README network's first layer with its own activation's gradient
        _linear_backward("linear backward 32x784x100", 32, 784, 100, "gelu", "none", False),
        # the block's second layer: the first layer's activation is undone in the input gradient
        _linear_backward("linear backward 2048x4096x1024", 2048, 4096, 1024, "none", "gelu", False),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["norm forward", "norm backward", "dropout forward", "dropout backward", "linear forward",
                     "linear forward", "linear backward", "linear backward"])
    if op.startswith(("norm", "dropout")):
        # up to 2^25 elements, one row to 16384, widths to the logits' 32768 (two values have no spread
        # left once they are normalised: their gradient is what eps leaves of it)
        rows = _spread(rng, 1, 16384)
        cols = _spread(rng, 4 if op.startswith("norm") else 1, min(32768, (1 << 25) // rows))
        if op == "norm forward":
            return _norm("", "forward", rows, cols, stats=rng.random() < 0.7, affine=rng.random() < 0.8)
        if op == "norm backward":
            return _norm("", "backward", rows, cols, residual=rng.random() < 0.5, affine=rng.random() < 0.8)
        p = rng.choice([0.05, 0.1, 0.2, 0.5, 0.9])
        if op == "dropout forward":
            return _dropout("", "forward", rows, cols, p, residual=rng.random() < 0.5)
        return _dropout("", "backward", rows, cols, p)
    batch, k, n = _spread(rng, 1, 4096), _spread(rng, 1, 4096), _spread(rng, 1, 4096)
    flops = 2.0 * batch * k * n * (1 if op == "linear forward" else 2)
    while flops > 3.4e10:  # the largest listed backward pass
        k, n = max(1, k * 3 // 4), max(1, n * 3 // 4)
        flops = 2.0 * batch * k * n * (1 if op == "linear forward" else 2)
    act = rng.choice(list(ACTIVATIONS))
    if op == "linear forward":
        return _linear_forward("", batch, k, n, act, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.8)
    return _linear_backward("", batch, k, n, act, rng.choice(list(ACTIVATIONS)), rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------------
def _share_stream():
    """The engine works on a stream of its own, which torch's default one does not wait for, nor it for that.  A program
    that hands torch's buffers to the engine lets torch work on the engine's stream: inputs are there before a call reads
    them, and what torch does with the outputs comes after it."""
    import rstorch_amd as rs
    engine = rs.default_engine()
    torch.cuda.set_stream(torch.cuda.ExternalStream(engine.lib.rst_engine_stream(engine.handle)))


def prepare(case, seed):
    if own:
        _share_stream()
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, dtype=F64, device=DEVICE, generator=g)

    def empty(*shape):
        return torch.empty(*shape, dtype=F64, device=DEVICE)

    s = {"case": case}
    op = case["op"]
    if op.startswith("layer_norm"):
        r, c = case["rows"], case["cols"]
        # a residual stream: rows of different scale, off centre
        s["x"] = normal(r, c) * torch.exp(0.5 * normal(r, 1)) + normal(r, 1)
        s["weight"] = 1.0 + 0.1 * normal(1, c) if case["affine"] else None
        s["bias"] = 0.1 * normal(1, c) if case["affine"] else None
        if op == "layer_norm_forward":
            s["out"] = empty(r, c)
            s["mean"], s["rstd"] = (empty(r, 1), empty(r, 1)) if case["stats"] else (None, None)
        else:
            s["grad"] = normal(r, c)
            s["residual_grad"] = normal(r, c) if case["residual"] else None
            # what the forward pass kept
            s["mean"] = s["x"].mean(1, keepdim=True)
            s["rstd"] = 1.0 / torch.sqrt((s["x"] - s["mean"]).square().mean(1, keepdim=True) + EPS)
            s["grad_input"] = empty(r, c)
            s["grad_weight"], s["grad_bias"] = (empty(1, c), empty(1, c)) if case["affine"] else (None, None)
    elif op.startswith("dropout"):
        r, c = case["rows"], case["cols"]
        s["x"] = normal(r, c)
        s["residual"] = normal(r, c) if case.get("residual") else None
        s["out"] = empty(r, c)
        s["seed"], s["stream"] = 0x5EED0000 + seed, 7  # 64-bit key of the generator and the call's number
    else:
        b, k, n = case["batch"], case["in"], case["out"]
        s["x"] = normal(b, k)
        s["weight"] = normal(n, k) / math.sqrt(k)  # KaimingNormal
        if op == "linear_forward":
            s["bias"] = 0.1 * normal(1, n) if case["bias"] else None
            s["residual"] = normal(b, n) if case["residual"] else None
            s["pre"] = empty(b, n) if case["pre"] else None
            s["out"] = empty(b, n)
        else:
            s["grad"] = normal(b, n)
            s["pre"] = normal(b, n) if case["act"] != "none" else None
            s["input_pre"] = normal(b, k) if case["input_act"] != "none" else None
            s["residual_grad"] = normal(b, k) if case["residual"] else None
            s["grad_pre"] = empty(b, n) if case["act"] != "none" else None
            s["grad_weight"], s["grad_bias"], s["grad_input"] = empty(n, k), empty(1, n), empty(b, k)
    return s


# ---- plain form ----------------------------------------------------------------------------------
_SQRT_HALF = math.sqrt(0.5)
_TANH_SCALE = 2.0 * math.sqrt(2.0 / math.pi)
_CUBE = 0.044715


def _act(z, kind):
    if kind == "relu":
        return torch.clamp_min(z, 0.0)
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * _SQRT_HALF))
    if kind == "gelu_tanh":  # 0.5 z (1 + tanh(t / 2)) = z / (1 + exp(-t))
        return z / (1.0 + torch.exp(-_TANH_SCALE * (z + _CUBE * z * z * z)))
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_gradient(z, kind):
    if kind == "relu":
        return (z > 0.0).to(F64)
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * _SQRT_HALF)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        s = 1.0 / (1.0 + torch.exp(-_TANH_SCALE * (z + _CUBE * z * z * z)))
        return s + z * s * (1.0 - s) * _TANH_SCALE * (1.0 + 3.0 * _CUBE * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s + z * s * (1.0 - s)


_GOLDEN, _C1, _C2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB
_ALL = (1 << 64) - 1


def _signed(v):
    v &= _ALL
    return v - (1 << 64) if v >> 63 else v


def _key(seed, stream):
    def mix(z):
        z = (z + _GOLDEN) & _ALL
        z = ((z ^ (z >> 30)) * _C1) & _ALL
        z = ((z ^ (z >> 27)) * _C2) & _ALL
        return z ^ (z >> 31)
    return mix(mix(seed & _ALL) ^ ((stream * 0xD1342543DE82EF95) & _ALL))


def _kept(count, p, seed, stream):
    """value(seed, stream, i) >= p for i in [0, count): the top 53 bits of the generator's word, as an integer."""
    z = torch.arange(count, dtype=torch.int64, device=DEVICE) * _signed(_GOLDEN) + _signed(_key(seed, stream) + _GOLDEN)

    def shifted(v, by):  # a logical shift
        return (v >> by) & ((1 << (64 - by)) - 1)

    z = (z ^ shifted(z, 30)) * _signed(_C1)
    z = (z ^ shifted(z, 27)) * _signed(_C2)
    z = z ^ shifted(z, 31)
    return shifted(z, 11) >= math.ceil(p * 2.0 ** 53)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "layer_norm_forward":
        x = s["x"]
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt(d.square().mean(1, keepdim=True) + EPS)
        y = d * rstd
        if case["affine"]:
            y = y * s["weight"] + s["bias"]
        return [y, mean, rstd] if case["stats"] else [y]
    if op == "layer_norm_backward":
        x, g, n = s["x"], s["grad"], float(case["rows"])
        xh = (x - s["mean"]) * s["rstd"]
        gw = g * s["weight"] if case["affine"] else g
        dx = s["rstd"] * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + s["residual_grad"]
        return [dx, (g * xh).sum(0, keepdim=True) / n, g.sum(0, keepdim=True) / n] if case["affine"] else [dx]
    if op.startswith("dropout"):
        x = s["x"]
        kept = _kept(x.numel(), case["p"], s["seed"], s["stream"]).view_as(x)
        y = torch.where(kept, x * (1.0 / (1.0 - case["p"])), 0.0)
        return [y + s["residual"]] if s["residual"] is not None else [y]
    if op == "linear_forward":
        z = s["x"] @ s["weight"].T
        if case["bias"]:
            z = z + s["bias"]
        y = _act(z, case["act"])
        if case["residual"]:
            y = y + s["residual"]
        return [y, z] if case["pre"] else [y]
    n = float(case["batch"])
    dz = s["grad"] * _act_gradient(s["pre"], case["act"]) if case["act"] != "none" else s["grad"]
    dx = dz @ s["weight"]
    if case["input_act"] != "none":
        dx = dx * _act_gradient(s["input_pre"], case["input_act"])
    if case["residual"]:
        dx = dx + s["residual_grad"]
    out = [dz.T @ s["x"] / n, dz.sum(0, keepdim=True) / n, dx]
    return out + [dz] if case["act"] != "none" else out


# ---- the framework's calls -----------------------------------------------------------------------
def _address(t):
    return None if t is None else t.data_ptr()


def _framework(s):
    import rstorch_amd as rs
    case = s["case"]
    op, a, check, engine = case["op"], _address, rs._ffi.check, rs.default_engine()
    lib, e = engine.lib, engine.handle
    if op == "layer_norm_forward":
        check(lib.rst_layer_norm_forward(e, a(s["x"]), a(s["weight"]), a(s["bias"]), a(s["out"]), a(s["mean"]),
                                         a(s["rstd"]), case["rows"], case["cols"], EPS))
        return [s["out"], s["mean"], s["rstd"]] if case["stats"] else [s["out"]]
    if op == "layer_norm_backward":
        check(lib.rst_layer_norm_backward(e, a(s["grad"]), a(s["x"]), a(s["weight"]), a(s["mean"]), a(s["rstd"]),
                                          a(s["residual_grad"]), a(s["grad_input"]), a(s["grad_weight"]),
                                          a(s["grad_bias"]), case["rows"], case["cols"]))
        return [s["grad_input"], s["grad_weight"], s["grad_bias"]] if case["affine"] else [s["grad_input"]]
    if op == "dropout_forward":
        check(lib.rst_dropout_forward(e, a(s["x"]), a(s["residual"]), a(s["out"]), s["x"].numel(), case["p"],
                                      s["seed"], s["stream"]))
        return [s["out"]]
    if op == "dropout_backward":
        check(lib.rst_dropout_backward(e, a(s["x"]), a(s["out"]), s["x"].numel(), case["p"], s["seed"],
                                       s["stream"]))
        return [s["out"]]
    if op == "linear_forward":
        check(lib.rst_linear_act_forward(e, a(s["x"]), a(s["weight"]), a(s["bias"]), a(s["residual"]), a(s["pre"]),
                                         a(s["out"]), case["batch"], case["in"], case["out"],
                                         ACTIVATIONS[case["act"]]))
        return [s["out"], s["pre"]] if case["pre"] else [s["out"]]
    check(lib.rst_linear_act_backward(e, a(s["grad"]), a(s["pre"]), ACTIVATIONS[case["act"]], a(s["grad_pre"]),
                                      a(s["x"]), a(s["weight"]), a(s["grad_weight"]), a(s["grad_bias"]),
                                      a(s["grad_input"]), a(s["input_pre"]), ACTIVATIONS[case["input_act"]],
                                      a(s["residual_grad"]), case["batch"], case["in"], case["out"]))
    out = [s["grad_weight"], s["grad_bias"], s["grad_input"]]
    return out + [s["grad_pre"]] if case["act"] != "none" else out


def run(state):
    return _framework(state) if own else _plain(state)


# ---- work and definition -------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op.startswith("linear"):
        b, k, n = case["batch"], case["in"], case["out"]
        if op == "linear_forward":
            values = b * k + n * k + b * n * (1 + case["pre"] + case["residual"]) + n * case["bias"]
            return {"bytes": 8.0 * values, "flops": 2.0 * b * k * n}
        values = b * n + b * k + 2 * n * k + n + b * k
        values += 2 * b * n * (case["act"] != "none") + b * k * (case["input_act"] != "none") + b * k * case["residual"]
        return {"bytes": 8.0 * values, "flops": 4.0 * b * k * n}
    r, c = case["rows"], case["cols"]
    if op == "layer_norm_forward":
        return {"bytes": 8.0 * (2 * r * c + 2 * c * case["affine"] + 2 * r * case["stats"]), "flops": 8.0 * r * c}
    if op == "layer_norm_backward":
        return {"bytes": 8.0 * ((3 + case["residual"]) * r * c + 3 * c * case["affine"] + 2 * r), "flops": 14.0 * r * c}
    return {"bytes": 8.0 * (2 + bool(case.get("residual"))) * r * c, "flops": 2.0 * r * c}


def _exact_act(z, kind):
    """(act(z), act'(z)) from the definitions: the normal distribution's integral, tanh, the logistic function."""
    if kind == "relu":
        return np.maximum(z, 0.0), np.where(z > 0.0, 1.0, 0.0)
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(torch.from_numpy(-z / math.sqrt(2.0))).numpy()
        return z * phi, phi + z * np.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if kind == "silu":
        sig = 0.5 * (1.0 + np.tanh(0.5 * z))
        return z * sig, sig + z * sig * (1.0 - sig)
    return z, np.ones_like(z)


def _exact_uniform(count, seed, stream):
    """splitmix64 in counter mode: the key mixes seed and stream, word i is the mix of key + i * golden ratio."""
    def mix(v):
        v = v + np.uint64(0x9E3779B97F4A7C15)
        v = (v ^ (v >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        v = (v ^ (v >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return v ^ (v >> np.uint64(31))

    with np.errstate(over="ignore"):
        key = mix(mix(np.array([seed], np.uint64)) ^ (np.array([stream], np.uint64) * np.uint64(0xD1342543DE82EF95)))
        words = mix(key + np.arange(count, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15))
    return (words >> np.uint64(11)).astype(np.float64) * 2.0 ** -53


def exact(case, seed):
    s = prepare(case, seed)
    h = {k: v.cpu().numpy() for k, v in s.items() if torch.is_tensor(v)}
    op = case["op"]
    if op == "layer_norm_forward":
        x = h["x"]
        mean = np.mean(x, axis=1, keepdims=True)
        std = np.sqrt(np.mean((x - mean) ** 2, axis=1, keepdims=True) + EPS)
        y = (x - mean) / std
        if case["affine"]:
            y = y * h["weight"] + h["bias"]
        return [y, mean, 1.0 / std] if case["stats"] else [y]
    if op == "layer_norm_backward":
        # through the normalisation's steps, each with its own gradient
        g, centred, rstd = h["grad"], h["x"] - h["mean"], h["rstd"]
        up = g * h["weight"] if case["affine"] else g
        dvar = np.sum(up * centred, axis=1, keepdims=True) * -0.5 * rstd ** 3
        dc = up * rstd + dvar * 2.0 * centred / case["cols"]
        dx = dc - np.mean(dc, axis=1, keepdims=True)
        if case["residual"]:
            dx = dx + h["residual_grad"]
        if not case["affine"]:
            return [dx]
        return [dx, np.mean(g * centred * rstd, axis=0, keepdims=True), np.mean(g, axis=0, keepdims=True)]
    if op.startswith("dropout"):
        x = h["x"]
        u = _exact_uniform(x.size, s["seed"], s["stream"]).reshape(x.shape)
        y = np.where(u < case["p"], 0.0, x / (1.0 - case["p"]))
        return [y + h["residual"]] if "residual" in h else [y]
    if op == "linear_forward":
        z = np.dot(h["x"], h["weight"].T)
        if case["bias"]:
            z = z + h["bias"]
        y = _exact_act(z, case["act"])[0]
        if case["residual"]:
            y = h["residual"] + y
        return [y, z] if case["pre"] else [y]
    dz = h["grad"]
    if case["act"] != "none":
        dz = dz * _exact_act(h["pre"], case["act"])[1]
    dx = np.dot(dz, h["weight"])
    if case["input_act"] != "none":
        dx = dx * _exact_act(h["input_pre"], case["input_act"])[1]
    if case["residual"]:
        dx = h["residual_grad"] + dx
    out = [np.dot(dz.T, h["x"]) / case["batch"], np.mean(dz, axis=0, keepdims=True), dx]
    return out + [dz] if case["act"] != "none" else out
