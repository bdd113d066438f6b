"""Host-side mirror of the reference's ``module`` package over the HIP backend.

Same names, argument meaning and failure behaviour as
``src/module/{mod,linear,sequential}.rs`` and ``src/module/activation/{relu,identity}.rs``:
``forward`` / ``backward`` / ``parameters`` / ``train`` / ``eval``; caches are consumed by
``backward`` (a second ``backward`` raises, where the reference panics on ``unwrap``);
gradients are overwritten, never accumulated.  Arrays are device-resident ``Array2``.

A ``Sequential`` made only of ``Identity`` / ``Linear`` / ``ReLU`` layers is *compiled*: the first
``forward`` builds a device model (``rst_model``) over the layer list, moves the layers' weights
into its parameter arena (the layers keep views) and from then on

* ``forward`` runs the layers' launches from one call,
* ``backward`` launches nothing: it remembers its gradient, and the pass runs when somebody needs
  its results - ``SGD.step(model)`` runs it with the optimiser update inside the weight-gradient
  launches (the README loop's ``model.backward(loss.backward()); optim.step(model)`` reaches
  exactly the launches of ``rst_model_train_step``), while reading a
  gradient through ``parameters()`` or touching the input gradient that ``backward`` returned runs
  it on its own first, so every value a caller can observe is the value the reference computes at
  that point.  The input gradient itself is only computed if the returned array is kept.

Any other layer list (a ``Softmax`` module, the residual block's ``LayerNorm`` / ``Dropout`` / ``GELU`` /
``SiLU`` / ``Residual``, a user-defined ``Module``) runs layer by layer; a ``Linear`` takes the activation
behind it, a residual and, in the backward pass, the activation in front of it into its own launches.
Changing the layer list (``push`` / ``insert`` / ``remove``) drops the compiled form; it is rebuilt on the next
``forward``.
"""
import ctypes
import weakref

from . import _ffi
from .engine import Array2, as_array2, default_engine
from .init import InitParameters, KaimingNormal, _fresh_seed


class Parameter:
    """src/module/mod.rs:16-19: a parameter and its gradient (device arrays)."""

    def __init__(self, parm, grad):
        self.parm = parm
        self.grad = grad


class Parameters:
    """src/module/mod.rs:21-40."""

    def __init__(self, parms=None):
        self.parms = list(parms or [])

    def add(self, parm, grad):
        self.parms.append(Parameter(parm, grad))
        return self

    def iter(self):
        return iter(self.parms)

    def __iter__(self):
        return iter(self.parms)

    def __len__(self):
        return len(self.parms)


class Module:
    """src/module/mod.rs:42-56."""

    def forward(self, input):
        raise NotImplementedError

    def backward(self, gradient):
        raise NotImplementedError

    def parameters(self):
        return Parameters()

    def train(self):
        pass

    def eval(self):
        pass


class Identity(Module):
    """src/module/activation/identity.rs:15-29."""

    @classmethod
    def new(cls):
        return cls()

    def forward(self, input):
        return input

    def backward(self, gradient):
        return gradient

    def __repr__(self):
        return "Identity"


class ReLU(Module):
    """src/module/activation/relu.rs:17-32."""

    def __init__(self):
        self.prev_input = None  # tensor whose sign gives the mask (pre-activation or output)

    @classmethod
    def new(cls):
        return cls()

    def forward(self, input):
        x = as_array2(input)
        out = x.engine.empty(x.rows, x.cols)
        _ffi.check(x.engine.lib.rst_relu_forward(x.engine.handle, x.ptr, out.ptr, x.size))
        self.prev_input = x
        return out

    def backward(self, gradient):
        if self.prev_input is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "ReLU.backward without a forward")
        g = as_array2(gradient, self.prev_input.engine)
        x, self.prev_input = self.prev_input, None  # take()
        if g.shape != x.shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs input %r" % (g.shape, x.shape))
        out = x.engine.empty(x.rows, x.cols)
        _ffi.check(x.engine.lib.rst_relu_backward(x.engine.handle, g.ptr, x.ptr, out.ptr, x.size))
        return out

    # used by Sequential when the neighbouring Linear kernels do this layer's work
    def _absorb_forward(self, activation):
        self.prev_input = activation

    def _absorb_backward(self):
        if self.prev_input is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "ReLU.backward without a forward")
        self.prev_input = None

    def __repr__(self):
        return "ReLU"


def _same_shape(residual, shape):
    if residual is not None and residual.shape != shape:
        raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "residual %r vs %r" % (residual.shape, shape))


def _add(x, residual):
    """x + residual in a new array."""
    _same_shape(residual, x.shape)
    out = x.engine.empty(x.rows, x.cols)
    _ffi.check(x.engine.lib.rst_activation_forward(x.engine.handle, x.ptr, residual.ptr, out.ptr, x.size,
                                                   _ffi.ACT_NONE))
    return out


class _Activation(Module):
    """An element-wise activation of the residual block: keeps what it was applied to."""

    kind = None

    def __init__(self):
        self.prev_input = None

    @classmethod
    def new(cls):
        return cls()

    def forward(self, input):
        x = as_array2(input)
        out = x.engine.empty(x.rows, x.cols)
        _ffi.check(x.engine.lib.rst_activation_forward(x.engine.handle, x.ptr, None, out.ptr, x.size, self.kind))
        self.prev_input = x
        return out

    def backward(self, gradient):
        if self.prev_input is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "%r.backward without a forward" % self)
        g = as_array2(gradient, self.prev_input.engine)
        if g.shape != self.prev_input.shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs input %r" % (g.shape, self.prev_input.shape))
        x, self.prev_input = self.prev_input, None
        out = x.engine.empty(x.rows, x.cols)
        _ffi.check(x.engine.lib.rst_activation_backward(x.engine.handle, g.ptr, x.ptr, None, out.ptr, x.size,
                                                        self.kind))
        return out

    # used by Sequential when the neighbouring Linear kernels do this layer's work
    def _absorb_forward(self, pre):
        self.prev_input = pre

    def _absorb_backward(self):
        self.prev_input = None

    def __repr__(self):
        return type(self).__name__


class GELU(_Activation):
    """x P(x), P the normal distribution's integral; ``approximate``: its tanh form."""

    def __init__(self, approximate=False):
        super().__init__()
        self.kind = _ffi.ACT_GELU_TANH if approximate else _ffi.ACT_GELU

    def __repr__(self):
        return "GELU(approximate=True)" if self.kind == _ffi.ACT_GELU_TANH else "GELU"


class SiLU(_Activation):
    """x / (1 + exp(-x))."""

    kind = _ffi.ACT_SILU


# the layers that a neighbouring Linear can take into its launches
_FUSED = (ReLU, GELU, SiLU)


class Dropout(Module):
    """In training (the state a module starts in; ``train`` / ``eval`` switch) zeroes each element with
    probability ``p`` and scales the others by 1 / (1 - p); in evaluation hands its input through.  No
    mask is stored: call number n of the module draws value(seed, n, index) of the library's generator,
    and ``backward`` draws it again."""

    def __init__(self, p=0.5, seed=None):
        if not 0.0 <= p < 1.0:
            raise ValueError("p = %r is not in [0, 1)" % (p,))
        self.p, self.seed = float(p), _fresh_seed() if seed is None else int(seed) & 0xFFFFFFFFFFFFFFFF
        self.training = True
        self._calls = 0
        self._kept = None  # (shape, engine, stream) of the last forward; stream None: handed through

    @classmethod
    def new(cls, p):
        return cls(p)

    def train(self):
        self.training = True

    def eval(self):
        self.training = False

    def _forward(self, input, residual):
        x = as_array2(input)
        _same_shape(residual, x.shape)
        if not self.training or self.p == 0.0:
            self._kept = (x.shape, x.engine, None)
            return x if residual is None else _add(x, residual)
        stream, self._calls = self._calls, self._calls + 1
        out = x.engine.empty(x.rows, x.cols)
        _ffi.check(x.engine.lib.rst_dropout_forward(x.engine.handle, x.ptr, residual.ptr if residual else None,
                                                    out.ptr, x.size, self.p, self.seed, stream))
        self._kept = (x.shape, x.engine, stream)
        return out

    def forward(self, input):
        return self._forward(input, None)

    def backward(self, gradient):
        if self._kept is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "Dropout.backward without a forward")
        shape, engine, stream = self._kept
        g = as_array2(gradient, engine)
        if g.shape != shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs input %r" % (g.shape, shape))
        self._kept = None
        if stream is None:
            return g
        out = g.engine.empty(g.rows, g.cols)
        _ffi.check(g.engine.lib.rst_dropout_backward(g.engine.handle, g.ptr, out.ptr, g.size, self.p, self.seed,
                                                     stream))
        return out

    def __repr__(self):
        return "Dropout(%g)" % self.p


class LayerNorm(Module):
    """Each row to mean 0 and variance 1 (over its ``size`` columns, ``eps`` added to the variance), then
    times ``weight`` plus ``bias`` (1, size), which start as ones and zeros.  Their gradients are divided
    by the number of rows, as Linear's are."""

    def __init__(self, size, eps=1e-5, engine=None):
        eng = engine or default_engine()
        self.engine, self.size, self.eps = eng, int(size), float(eps)
        self.weight, self.bias = eng.full(1, self.size, 1.0), eng.zeros(1, self.size)
        self.grad_weight = self.grad_bias = None
        self._kept = None  # (x, mean, rstd) of the last forward

    @classmethod
    def new(cls, size):
        return cls(size)

    def forward(self, input):
        x = as_array2(input, self.engine)
        if x.cols != self.size:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "input has %d features, layer expects %d" % (x.cols, self.size))
        out, mean, rstd = (self.engine.empty(x.rows, n) for n in (x.cols, 1, 1))
        _ffi.check(self.engine.lib.rst_layer_norm_forward(
            self.engine.handle, x.ptr, self.weight.ptr, self.bias.ptr, out.ptr, mean.ptr, rstd.ptr, x.rows, x.cols,
            self.eps))
        self._kept = (x, mean, rstd)
        return out

    def _backward(self, gradient, residual):
        if self._kept is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "LayerNorm.backward without a forward")
        g = as_array2(gradient, self.engine)
        x, mean, rstd = self._kept
        if g.shape != x.shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs input %r" % (g.shape, x.shape))
        _same_shape(residual, x.shape)
        self._kept = None
        grad_weight = self.grad_weight or self.engine.empty(1, self.size)
        grad_bias = self.grad_bias or self.engine.empty(1, self.size)
        gx = self.engine.empty(x.rows, x.cols)
        _ffi.check(self.engine.lib.rst_layer_norm_backward(
            self.engine.handle, g.ptr, x.ptr, self.weight.ptr, mean.ptr, rstd.ptr, residual.ptr if residual else None,
            gx.ptr, grad_weight.ptr, grad_bias.ptr, x.rows, x.cols))
        self.grad_weight, self.grad_bias = grad_weight, grad_bias
        return gx

    def backward(self, gradient):
        return self._backward(gradient, None)

    def parameters(self):
        if self.grad_weight is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "LayerNorm.parameters before any backward (no gradient yet)")
        return Parameters().add(self.weight, self.grad_weight).add(self.bias, self.grad_bias)

    def __repr__(self):
        return "LayerNorm(%d)" % self.size


class Softmax(Module):
    """src/module/activation/softmax.rs:5-78: softmax along an axis; the backward pass builds the
    reference's single batch-summed Jacobian."""

    def __init__(self, axis=1):
        self.axis = int(axis)
        self.output = None

    @classmethod
    def new(cls):
        return cls(1)

    @classmethod
    def with_axis(cls, axis):
        return cls(axis)

    def forward(self, input):
        x = as_array2(input)
        out = x.engine.empty(x.rows, x.cols)
        _ffi.check(x.engine.lib.rst_softmax_forward(x.engine.handle, x.ptr, out.ptr, x.rows, x.cols,
                                                    self.axis))
        self.output = out
        return out.clone()  # the reference returns a clone and keeps the output (softmax.rs:58-59)

    def backward(self, gradient):
        if self.output is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "Softmax.backward without a forward")
        out, self.output = self.output, None  # take()
        g = as_array2(gradient, out.engine)
        if g.shape != out.shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs output %r" % (g.shape, out.shape))
        gin = out.engine.empty(out.rows, out.cols)
        _ffi.check(out.engine.lib.rst_softmax_backward(out.engine.handle, g.ptr, out.ptr, gin.ptr,
                                                       out.rows, out.cols))
        return gin

    def __repr__(self):
        return "Softmax(axis=%d)" % self.axis


class Linear(Module):
    """src/module/linear.rs:8-79.  weight (out, in), bias (1, out)."""

    def __init__(self, input_size, output_size, init=None, engine=None):
        init = init if init is not None else KaimingNormal()
        eng = engine or default_engine()
        self.engine = eng
        self.input_size, self.output_size = int(input_size), int(output_size)
        self.weight = as_array2(init.weight(self.input_size, self.output_size, eng), eng)
        self.bias = as_array2(init.bias(self.input_size, self.output_size, eng), eng)
        if self.weight.shape != (self.output_size, self.input_size):
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "init.weight returned %r" % (self.weight.shape,))
        if self.bias.shape != (1, self.output_size):
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "init.bias returned %r" % (self.bias.shape,))
        self.prev_input = None
        self.grad_weight = None
        self.grad_bias = None
        self._home = None       # the compiled Sequential (_Plan) whose arena holds the parameters
        self._has_grad = False  # a backward pass has been asked for since the layer was made

    @classmethod
    def new(cls, input_size, output_size):
        return cls(input_size, output_size)

    @classmethod
    def new_with_kernel(cls, input_size, output_size, init):
        return cls(input_size, output_size, init)

    def _forward(self, input, fuse_relu):
        x = as_array2(input, self.engine)
        if x.cols != self.input_size:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "input has %d features, layer expects %d"
                                  % (x.cols, self.input_size))
        out = self.engine.empty(x.rows, self.output_size)
        _ffi.check(self.engine.lib.rst_linear_forward(
            self.engine.handle, x.ptr, self.weight.ptr, self.bias.ptr, out.ptr, x.rows,
            self.input_size, self.output_size, 1 if fuse_relu else 0))
        self.prev_input = x
        return out

    def forward(self, input):
        return self._forward(input, False)

    def _backward(self, gradient, mask_by_input, need_input_grad=True):
        if self.prev_input is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "Linear.backward without a forward")
        g = as_array2(gradient, self.engine)
        x, self.prev_input = self.prev_input, None  # take()
        if g.shape != (x.rows, self.output_size):
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs expected %r"
                                  % (g.shape, (x.rows, self.output_size)))
        if self.grad_weight is None:
            self.grad_weight = self.engine.empty(self.output_size, self.input_size)
            self.grad_bias = self.engine.empty(1, self.output_size)
        self._has_grad = True
        gx = self.engine.empty(x.rows, self.input_size) if need_input_grad else None
        _ffi.check(self.engine.lib.rst_linear_backward(
            self.engine.handle, g.ptr, x.ptr, self.weight.ptr, self.grad_weight.ptr,
            self.grad_bias.ptr, gx.ptr if gx is not None else None,
            x.ptr if (mask_by_input and gx is not None) else None, x.rows, self.input_size,
            self.output_size))
        return gx

    def backward(self, gradient):
        return self._backward(gradient, False)

    # The same with an activation behind the layer, a residual, an activation in front of it.
    def _forward_act(self, input, activation, residual):
        """(act(z) + residual, z) in one pass; z only with an activation."""
        x = as_array2(input, self.engine)
        if x.cols != self.input_size:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "input has %d features, layer expects %d"
                                  % (x.cols, self.input_size))
        _same_shape(residual, (x.rows, self.output_size))
        out = self.engine.empty(x.rows, self.output_size)
        pre = self.engine.empty(x.rows, self.output_size) if activation != _ffi.ACT_NONE else None
        _ffi.check(self.engine.lib.rst_linear_act_forward(
            self.engine.handle, x.ptr, self.weight.ptr, self.bias.ptr, residual.ptr if residual else None,
            pre.ptr if pre else None, out.ptr, x.rows, self.input_size, self.output_size, activation))
        self.prev_input = x
        return out, pre

    def _backward_act(self, gradient, input_pre, input_activation, residual):
        if self.prev_input is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "Linear.backward without a forward")
        g = as_array2(gradient, self.engine)
        x = self.prev_input
        if g.shape != (x.rows, self.output_size):
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs expected %r"
                                  % (g.shape, (x.rows, self.output_size)))
        _same_shape(residual, x.shape)
        if input_pre is not None and input_pre.shape != x.shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "the activation in front saw %r, this layer %r"
                                  % (input_pre.shape, x.shape))
        self.prev_input = None
        if self.grad_weight is None:
            self.grad_weight = self.engine.empty(self.output_size, self.input_size)
            self.grad_bias = self.engine.empty(1, self.output_size)
        self._has_grad = True
        gx = self.engine.empty(x.rows, self.input_size)
        _ffi.check(self.engine.lib.rst_linear_act_backward(
            self.engine.handle, g.ptr, None, _ffi.ACT_NONE, None, x.ptr, self.weight.ptr, self.grad_weight.ptr,
            self.grad_bias.ptr, gx.ptr, input_pre.ptr if input_pre else None, input_activation,
            residual.ptr if residual else None, x.rows, self.input_size, self.output_size))
        return gx

    def parameters(self):
        if not self._has_grad:
            raise _ffi.StateError(_ffi.RST_ERR_STATE,
                                  "Linear.parameters before any backward (no gradient yet)")
        return Parameters().add(self.weight, self.grad_weight).add(self.bias, self.grad_bias)

    def __repr__(self):
        return "Linear(%d, %d)" % (self.input_size, self.output_size)


class _Plan:
    """The compiled form of a Sequential of Identity / Linear / ReLU layers: an ``rst_model`` whose
    arena holds the layers' parameters and gradients, plus the backward pass that has been asked
    for but not launched yet."""

    def __init__(self, layers):
        from .model import DeviceModel
        self.key = tuple(id(l) for l in layers)
        self.linears = [l for l in layers if type(l) is Linear]
        spec = []
        for l in layers:
            if type(l) is Linear:
                spec.append(("linear", l.input_size, l.output_size))
            else:
                spec.append(("relu",) if type(l) is ReLU else ("identity",))
        self.engine = self.linears[0].engine
        for l in self.linears:  # whatever another compiled Sequential still owes these layers
            if l._home is not None:
                l._home.flush()
        self.device = DeviceModel(spec, self.engine)
        eng, params = self.engine, self.device.parameters()
        for i, l in enumerate(self.linears):
            (w, gw), (b, gb) = params[2 * i], params[2 * i + 1]
            _ffi.check(eng.lib.rst_copy(eng.handle, w._ptr, l.weight.ptr, w.size))
            _ffi.check(eng.lib.rst_copy(eng.handle, b._ptr, l.bias.ptr, b.size))
            if l._has_grad and l.grad_weight is not None:  # gradients computed before the move stay readable
                _ffi.check(eng.lib.rst_copy(eng.handle, gw._ptr, l.grad_weight.ptr, gw.size))
                _ffi.check(eng.lib.rst_copy(eng.handle, gb._ptr, l.grad_bias.ptr, gb.size))
            l.weight, l.bias = w, b
            # a look at (or a write into) a parameter between the loss and the backward pass: input
            # gradients launched ahead were computed with the weights of before
            w._before_access = b._before_access = self._parameters_touched
            # reading a gradient first runs the backward pass that is still owed
            gw._before_access = gb._before_access = self.flush
            l.grad_weight, l.grad_bias = gw, gb
            l._home = self
        self.in_width, self.out_width = self.device.in_width, self.device.out_width
        self.x = self.out = None      # the forward pass whose caches are live (kept alive until backward)
        self.pending = None           # (gradient, weak reference to the deferred input gradient)
        # a loss on the logits that a backward pass followed: the next step is taken for one of a training loop
        self._training = self._loss_seen = self._backward_followed = False
        self._inputs_from = None      # weak reference to the loss gradient that input gradients were launched from

    def valid_for(self, layers):
        return self.key == tuple(id(l) for l in layers) and all(l._home is self for l in self.linears)

    def forward(self, input):
        self.flush()  # a backward pass nobody looked at would otherwise read the new activations
        x = as_array2(input, self.engine)
        if x.cols != self.in_width:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "input has %d features, layer expects %d"
                                  % (x.cols, self.in_width))
        out = self.engine.empty(x.rows, self.out_width)
        _ffi.check(self.engine.lib.rst_model_forward_to(self.device.handle, x.ptr, x.rows, out.ptr))
        self.x, self.out = x, out
        self._training = self._loss_seen and self._backward_followed
        self._loss_seen = self._backward_followed = False
        self._inputs_from = None
        out._loss_through = weakref.WeakMethod(self._loss_through)
        return out

    def _loss_through(self, pred, truth, grad):
        """CrossEntropyLoss.forward on the logits of the latest forward pass: the loss, or None when
        this is not the array forward() returned.  In a training loop the input gradients of the
        layers above the first are launched behind the loss before the host waits for it
        (rst_model_loss_accuracy_to), and the backward pass skips them if the gradient array reaches
        backward() without anybody having looked at it."""
        if self.x is None or self.pending is not None or pred is not self.out or pred.shape != truth.shape:
            return None
        loss = ctypes.c_double()
        _ffi.check(self.engine.lib.rst_model_loss_accuracy_to(
            self.device.handle, pred.ptr, truth.ptr, grad.ptr, 1 if self._training else 0, ctypes.byref(loss), None))
        self._loss_seen = True
        if self._training:
            self._inputs_from = weakref.ref(grad)
            grad._before_access = self._inputs_touched
        return loss.value

    def _parameters_touched(self):
        if self._inputs_from is not None:
            self._inputs_touched()

    def _inputs_touched(self):
        """Somebody looked at (and may have rewritten) the gradient the input gradients were launched from."""
        _ffi.check(self.engine.lib.rst_model_discard_inputs(self.device.handle))
        self._inputs_from = None

    def backward(self, gradient):
        if self.x is None or self.pending is not None:  # no forward yet, or its caches are taken
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "Sequential.backward without a forward")
        g = as_array2(gradient, self.engine)
        if g.shape != (self.x.rows, self.out_width):
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs expected %r"
                                  % (g.shape, (self.x.rows, self.out_width)))
        gin = Array2(self.engine, self.x.rows, self.in_width, resolver=self._resolve_input_grad)
        self.pending = (g, weakref.ref(gin))
        self._backward_followed = True
        for l in self.linears:
            l._has_grad = True
        return gin

    def _resolve_input_grad(self, gin):
        """Somebody looks at the array that backward() returned."""
        if self.pending is not None and self.pending[1]() is gin:
            self._run(False, 0.0)
        if gin._ptr is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "this input gradient was never computed")

    def _run(self, apply_sgd, lr):
        g, ref = self.pending
        self.pending = None
        gin = ref()  # still wanted by somebody?
        if gin is not None:
            gin._resolver = None
            gin._materialise()
        if self._inputs_from is not None:
            if self._inputs_from() is g:   # untouched since: our own access keeps the launched gradients
                g._before_access = None
            else:
                self._inputs_touched()
            self._inputs_from = None
        _ffi.check(self.engine.lib.rst_model_backward_to(
            self.device.handle, g.ptr, gin._ptr if gin is not None else None, 1 if apply_sgd else 0, float(lr)))
        self.x = self.out = None  # the caches are consumed

    def flush(self):
        """Runs the backward pass that is still owed, without an optimiser step."""
        if self.pending is not None:
            self._run(False, 0.0)

    def step_sgd(self, lr):
        """backward + SGD::step in one pass, if a backward is still owed; else False."""
        if self.pending is None:
            return False
        self._run(True, lr)
        return True


class Sequential(Module):
    """src/module/sequential.rs:11-110.  The layer list may change at any time; the
    Linear/ReLU fusion is decided afresh on every call."""

    # False (on the class or on one instance): always run layer by layer, one call per layer
    compile_enabled = True

    def __init__(self, layers=None):
        self.layers = list(layers or [])
        self._plan = None

    def _compiled(self):
        """The compiled form, built on demand; None when the layer list has a layer it cannot hold."""
        if not self.compile_enabled:
            self._drop_plan()
            return None
        if self._plan is not None and self._plan.valid_for(self.layers):
            return self._plan
        self._drop_plan()
        linears = [l for l in self.layers if type(l) is Linear]
        if not linears or any(type(l) not in (Linear, ReLU, Identity) for l in self.layers):
            return None
        if any(l.engine is not linears[0].engine for l in linears):
            return None
        if any(a.output_size != b.input_size for a, b in zip(linears, linears[1:])):
            return None  # the layer-by-layer pass raises the shape error where the reference panics
        self._plan = _Plan(self.layers)
        return self._plan

    def _drop_plan(self):
        if self._plan is not None:
            self._plan.flush()
            self._plan = None

    @classmethod
    def new(cls, layers):
        return cls(layers)

    def push(self, layer):
        self._drop_plan()
        self.layers.append(layer)

    push_box = push

    def insert(self, index, layer):
        self._drop_plan()
        self.layers.insert(index, layer)

    insert_box = insert

    def len(self):
        return len(self.layers)

    __len__ = len

    def is_empty(self):
        return not self.layers

    def remove(self, index):
        if index >= len(self.layers):
            return None
        self._drop_plan()
        return self.layers.pop(index)

    def _engine(self):
        """The engine of the first layer that has one; None: no layer is bound to any."""
        for layer in self.layers:
            if isinstance(layer, (Linear, LayerNorm)):
                return layer.engine
            inner = layer.inner if isinstance(layer, Residual) else layer
            engine = inner._engine() if isinstance(inner, Sequential) else None
            if engine is not None:
                return engine
        return None

    def _output_size(self, width):
        """Columns of what the layers return for an input of ``width`` columns; None where a layer of the caller's own
        decides that."""
        for layer in self.layers:
            if type(layer) is Linear:
                width = layer.output_size
            elif type(layer) is Sequential:
                width = layer._output_size(width)
            elif type(layer) not in _SAME_WIDTH:
                width = None
        return width

    # (exact types, here and where a Linear takes its neighbour's work: a subclass may override forward or
    # backward, and is called like any other layer)
    def _next_real(self, i):
        for j in range(i + 1, len(self.layers)):
            if type(self.layers[j]) is not Identity:
                return j
        return -1

    def _prev_real(self, i):
        for j in range(i - 1, -1, -1):
            if type(self.layers[j]) is not Identity:
                return j
        return -1

    def forward(self, input):
        plan = self._compiled()
        if plan is not None:
            return plan.forward(input)
        return self._layers_forward(input, None)

    def _layers_forward(self, input, residual):
        """Layer by layer; residual (or None) is added to the result, by the last layer where it can."""
        x = input
        last = self._prev_real(len(self.layers))  # (-1: nothing but Identity)
        if last >= 0 and type(self.layers[self._next_real(-1)]) in _ANY_ENGINE:
            x = as_array2(input, self._engine())  # (the layer alone would put a host array on the default engine)
        skip = set()
        for i, layer in enumerate(self.layers):
            if i in skip:
                continue
            if type(layer) is Linear:
                j = self._next_real(i)
                behind = self.layers[j] if j >= 0 else None
                if type(behind) is ReLU and (residual is None or j != last):
                    x = layer._forward(x, True)
                    behind._absorb_forward(x)
                    skip.add(j)
                    continue
                if type(behind) in _FUSED:
                    kind = _ffi.ACT_RELU if type(behind) is ReLU else behind.kind
                    x, pre = layer._forward_act(x, kind, residual if j == last else None)
                    behind._absorb_forward(pre)
                    skip.add(j)
                    residual = None if j == last else residual
                    continue
                if residual is not None and i == last:
                    x, _ = layer._forward_act(x, _ffi.ACT_NONE, residual)
                    residual = None
                    continue
            if residual is not None and i == last and type(layer) is Dropout:
                x = layer._forward(x, residual)
                residual = None
                continue
            x = layer.forward(x)
        return x if residual is None else _add(as_array2(x), residual)

    def backward(self, gradient):
        if self._plan is not None and self._plan.valid_for(self.layers):
            return self._plan.backward(gradient)
        return self._layers_backward(gradient, None)

    def _layers_backward(self, gradient, residual):
        """Layer by layer; residual (or None) is added to the input gradient, by the first layer where it can."""
        g = gradient
        first = self._next_real(-1)
        skip = set()
        for i in range(len(self.layers) - 1, -1, -1):
            if i in skip:
                continue
            layer = self.layers[i]
            if type(layer) is Linear:
                j = self._prev_real(i)
                before = self.layers[j] if j >= 0 else None
                if type(before) is ReLU and before.prev_input is not None and (residual is None or j != first):
                    g = layer._backward(g, True)
                    before._absorb_backward()
                    skip.add(j)
                    continue
                if type(before) in _FUSED and before.prev_input is not None:
                    kind = _ffi.ACT_RELU if type(before) is ReLU else before.kind
                    g = layer._backward_act(g, before.prev_input, kind, residual if j == first else None)
                    before._absorb_backward()
                    skip.add(j)
                    residual = None if j == first else residual
                    continue
                if residual is not None and i == first:
                    g = layer._backward_act(g, None, _ffi.ACT_NONE, residual)
                    residual = None
                    continue
            if residual is not None and i == first and type(layer) is LayerNorm:
                g = layer._backward(g, residual)
                residual = None
                continue
            g = layer.backward(g)
        return g if residual is None else _add(as_array2(g), residual)

    def train(self):
        for layer in self.layers:
            layer.train()

    def eval(self):
        for layer in self.layers:
            layer.eval()

    def parameters(self):
        out = Parameters()
        for layer in self.layers:
            for p in layer.parameters():
                out.parms.append(p)
        return out

    def __repr__(self):
        return "Sequential(%s)" % ", ".join(repr(l) for l in self.layers)


class Residual(Module):
    """x + inner(x); ``inner``: a layer or a list of layers whose output has the shape of its input.  The
    addition (and, in the backward pass, that of the gradient that passes the layers by) is done by the
    inner layers' own launches where the last one is a Linear, an activation behind a Linear, or Dropout, and
    the first one a Linear or LayerNorm."""

    def __init__(self, inner):
        if type(inner) is Sequential:  # (a subclass is a layer like any other: its own passes are called)
            self.inner = inner
        else:
            self.inner = Sequential(list(inner) if isinstance(inner, (list, tuple)) else [inner])
        self._kept = None  # (shape of the last forward's input, engine for the gradient)

    @classmethod
    def new(cls, inner):
        return cls(inner)

    def forward(self, input):
        engine = self.inner._engine()
        x = as_array2(input, engine)
        self.inner._drop_plan()  # (a compiled form would add in a pass of its own)
        wide = self.inner._output_size(x.cols)
        if wide is not None and wide != x.cols:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "a residual of %d features around layers that return %d"
                                  % (x.cols, wide))
        out = self.inner._layers_forward(x, x)
        self._kept = (x.shape, engine or x.engine)
        return out

    def backward(self, gradient):
        if self._kept is None:
            raise _ffi.StateError(_ffi.RST_ERR_STATE, "Residual.backward without a forward")
        shape, engine = self._kept
        g = as_array2(gradient, engine)
        if g.shape != shape:
            raise _ffi.ShapeError(_ffi.RST_ERR_SHAPE, "gradient %r vs input %r" % (g.shape, shape))
        self._kept = None
        return self.inner._layers_backward(g, g)

    def parameters(self):
        return self.inner.parameters()

    def train(self):
        self.inner.train()

    def eval(self):
        self.inner.eval()

    def __repr__(self):
        return "Residual(%s)" % ", ".join(repr(l) for l in self.inner.layers)


# layers that take an array of any engine
_ANY_ENGINE = (ReLU, Softmax, GELU, SiLU, Dropout)
# layers that return as many columns as they are given
_SAME_WIDTH = (Identity, ReLU, Softmax, GELU, SiLU, Dropout, LayerNorm, Residual)


def sequential(*layers):
    """The ``sequential!`` macro (src/module/sequential.rs:62-74): both spellings of the
    reference are accepted - layer instances, or ``(LayerClass, arg, ...)`` tuples."""
    built = []
    for l in layers:
        if isinstance(l, tuple):
            built.append(l[0].new(*l[1:]))
        elif isinstance(l, type):
            built.append(l.new())
        else:
            built.append(l)
    return Sequential.new(built)
