"""Operators on sequences over the C ABI in include/genn_mi355x.h: a short causal convolution of every channel, a selective state space
scan and a gated delta rule, for whole sequences (with gradients) and for one token of every running sequence; and what stands around them: layer norm
with its gradients, and dropout.

As a model's arrays are handed to its runner once and stepped many times, an operator's arrays are bound once (checked then) and
``run()`` / ``backward()`` are single calls of the library.  Arrays are ``Array`` objects of this package or tensors on the device.
``stream`` is the address of a HIP stream; 0, the default, is the null stream.  A call while another device than the operator's is current is refused.
"""
import ctypes as C
import threading
from numbers import Integral

from . import _abi
from .genn_model import Array
from .operands import Operand, current_device, same_device


def _count(n, name):
    """As the descriptors' 32 bits take it."""
    if not 0 <= n < 1 << 31:
        raise ValueError(f"{name} is a count below 2^31, not {n}")
    return int(n)


class _SequenceOperator:
    def __init__(self, sequences, length, dtype, device):
        if dtype not in _abi.FLOAT_TYPES:
            raise NotImplementedError(f"element type {dtype}")
        self.sequences, self.length, self.dtype, self.device = _count(sequences, "sequences"), _count(length, "length"), dtype, device
        self._lib = _abi.load()
        _abi.check(self._lib.gennmi_init(device))
        self._bound = self._gradients = None        # operands (kept alive) of the descriptors
        self._packed = self._bound_packed = None    # rows of packed arrays: of a call of bind(), and of the one that held
        self._workspaces = {}           # (which pass, stream): one each, as calls on different streams may overlap
        self._lock = threading.Lock()   # of them: two threads may make the first call on a stream at once

    def _operand(self, array, name, shape=None):
        return None if array is None else Operand(array, name, shape)

    def _rows(self, array, name, width, given, dtype=None):
        """A ``Rows`` of the operator's element type (or of ``dtype``), or an empty one."""
        if array is None:
            return _abi.Rows()
        shape = None
        if isinstance(array, Array):
            count = self._packed if self._packed is not None else self.sequences * self.length
            shape = (count, width) if array.count == count * width or self._packed is None else (array.count // width, width)
        o = Operand(array, name, shape).wants(dtype or self.dtype)
        given.append(o)
        return o.rows(self.sequences, self.length, width, self._packed)

    def _flat(self, array, name, shape, dtype, given):
        if array is None:
            return None
        o = Operand(array, name, shape).wants(dtype).contiguous(shape)
        given.append(o)
        return o.address

    def _sequences(self, offsets, slots, first, given):
        """The descriptor of the sequences; ``first``: the array whose rows a packed operator counts."""
        s = _abi.Sequences(count=self.sequences, length=self.length, device=self.device + 1)
        self._packed = None
        if offsets is not None:
            s.offsets = self._flat(offsets, "offsets", (self.sequences + 1,), ("int32", "uint32"), given)
            rows = Operand(first, "the first array")
            self._packed = rows.shape[0] if len(rows.shape) > 1 else rows.shape[0] // self._width
            s.rows = self._packed
        if slots is not None:
            s.slots = self._flat(slots, "slots", (self.sequences,), "int32", given)
        return s

    def _states(self, state, name, slots, shape, dtype, given):
        """The state of every sequence, or with slots of every place; their number."""
        if state is None:
            return None, None
        places = self.sequences
        if slots is not None:
            size = 1
            for n in shape:
                size *= n
            places = state.count // max(1, size) if isinstance(state, Array) else int(state.shape[0])
        return self._flat(state, name, (places,) + shape, dtype, given), places

    def _workspace(self, key, given, needed, stream):
        """``given`` by the caller, or the operator's own for that stream."""
        if given is not None:
            o = Operand(given, "workspace").wants(("uint8", "float32"))
            o.contiguous(o.shape)
            same_device([o], self.device)
            size = o.shape[0] if len(o.shape) == 1 else 0
            return o.address, size * (4 if o.dtype == "float32" else 1)
        if not needed:
            return None, 0
        if stream:
            capturing = _int()
            _abi.check(self._lib.gennmi_stream_is_capturing(stream, _byref(capturing)))
            if capturing.value:
                raise ValueError("the stream is being captured: give the call a workspace of its own, which the graph then keeps using")
        with self._lock:
            own = self._workspaces.get((key, stream))
            if own is None or own.count < needed:
                current_device(self._lib, self.device)
                if own is not None:
                    own.free()
                own = self._workspaces[key, stream] = Array(needed, "uint8", device_only=True)
            return own.ptr, own.count

    def free(self):
        """Gives the operator's own workspaces back."""
        for w in self._workspaces.values():
            w.free()
        self._workspaces = {}

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def _need(self, what, name):
        if what is None:
            raise RuntimeError(f"{name} must be called first")


class CausalConvolution(_SequenceOperator):
    """out[t] = f(bias + sum_k weight[:, k] x[t - (taps - 1) + k]), channel by channel, with f the identity or (``silu``) s sigmoid(s).

    ``x`` and ``out``: [sequences, length, channels] (or both first axes as one), or with ``offsets`` packed rows [rows, channels], of which sequence s
    has offsets[s] .. offsets[s + 1] - 1 (``length``: the most).  States: the last taps - 1 inputs, [sequences, taps - 1, channels];
    with ``slots`` [places, taps - 1, channels], sequence s at place slots[s] (outside of them: padding, nothing of it is read or written).  ``length=1``
    with the same array as initial and final state is a token of every running sequence."""

    def __init__(self, sequences, length, channels, taps, dtype="float32", silu=False, device=0):
        super().__init__(sequences, length, dtype, device)
        self.channels, self.taps, self.silu = _count(channels, "channels"), _count(taps, "taps"), bool(silu)
        self._width = self.channels

    def bind(self, x, weight, bias=None, out=None, initial_state=None, final_state=None, offsets=None, slots=None):
        given = []
        c = _abi.CausalConv(type=_abi.FLOAT_TYPES[self.dtype], channels=self.channels, taps=self.taps, silu=self.silu)
        c.sequences = self._sequences(offsets, slots, x, given)
        c.x, c.out = self._rows(x, "x", self.channels, given), self._rows(out, "out", self.channels, given)
        c.weight = self._flat(weight, "weight", (self.channels, self.taps), "float32", given)
        c.bias = self._flat(bias, "bias", (self.channels,), "float32", given)
        shape = (self.taps - 1, self.channels)
        c.initialState, first = self._states(initial_state, "initial_state", slots, shape, self.dtype, given)
        c.finalState, last = self._states(final_state, "final_state", slots, shape, self.dtype, given)
        if slots is not None:
            if first is not None and last is not None and first != last:
                raise ValueError("initial_state and final_state have different numbers of places")
            c.sequences.numSlots = first or last or 0
        same_device(given, self.device)
        self._bound, self._bound_packed, self._descriptor, self._reference, self._gradients = given, self._packed, c, C.byref(c), None

    def run(self, stream=0):
        if self._bound is None:
            raise RuntimeError("bind() must be called first")
        rc = self._lib.gennmi_causal_conv(self._reference, stream)
        if rc:
            _abi.check(rc)

    def bind_gradients(self, out, x=None, weight=None, bias=None, initial_state=None, final_state=None):
        """``out`` and ``final_state``: gradients that come in; the others are written."""
        self._need(self._bound, "bind()")
        self._packed = self._bound_packed
        given = []
        g = _abi.CausalConvGradient()
        g.out, g.x = self._rows(out, "the gradient of out", self.channels, given), self._rows(x, "the gradient of x", self.channels, given)
        shape = (self.sequences, self.taps - 1, self.channels)
        g.finalState = self._flat(final_state, "the gradient of final_state", shape, self.dtype, given)
        g.initialState = self._flat(initial_state, "the gradient of initial_state", shape, self.dtype, given)
        g.weight = self._flat(weight, "the gradient of weight", (self.channels, self.taps), "float32", given)
        g.bias = self._flat(bias, "the gradient of bias", (self.channels,), "float32", given)
        same_device(given, self.device)
        size = C.c_size_t()
        _abi.check(self._lib.gennmi_causal_conv_backward_workspace(self._reference, C.byref(size)))
        self.backward_workspace_bytes = size.value if weight is not None or bias is not None else 0
        self._gradients, self._gradient_descriptor, self._gradient_reference = given, g, C.byref(g)

    def backward(self, stream=0, workspace=None):
        """``workspace``: ``backward_workspace_bytes`` on the device, for a call that is captured into a graph (which keeps using it)."""
        self._need(self._gradients, "bind_gradients()")
        address, size = self._workspace("backward", workspace, self.backward_workspace_bytes, stream)
        rc = self._lib.gennmi_causal_conv_backward(self._reference, self._gradient_reference, address, size, stream)
        if rc:
            _abi.check(rc)


class SelectiveScan(_SequenceOperator):
    """h[t] = exp(dt A) h[t-1] + dt u B[t],  out[t] = (sum_n C[t] h[t] + D u) z sigmoid(z),  dt = delta + delta_bias or (``softplus``) log(1 + exp of it).

    ``u, delta, z, out``: rows of channels; ``B, C``: rows of groups x states (channels / groups neighbouring channels share a group's); ``A``: [channels, states].
    Rows, ``offsets`` and ``slots`` as for ``CausalConvolution``; states [sequences or places, channels, states] are float32.  ``length=1`` is a token of
    every running sequence."""

    def __init__(self, sequences, length, channels, states, groups=1, dtype="float32", softplus=False, device=0):
        super().__init__(sequences, length, dtype, device)
        self.channels, self.states, self.groups, self.softplus = _count(channels, "channels"), _count(states, "states"), _count(groups, "groups"), bool(softplus)
        self._width = self.channels

    def bind(self, u, delta, A, B, C, out=None, D=None, delta_bias=None, z=None, initial_state=None, final_state=None, offsets=None, slots=None):
        given, width = [], self.groups * self.states
        c = _abi.Scan(type=_abi.FLOAT_TYPES[self.dtype], channels=self.channels, states=self.states, groups=self.groups, softplus=self.softplus)
        c.sequences = self._sequences(offsets, slots, u, given)
        c.u, c.delta = self._rows(u, "u", self.channels, given), self._rows(delta, "delta", self.channels, given)
        c.z, c.out = self._rows(z, "z", self.channels, given), self._rows(out, "out", self.channels, given)
        c.B, c.C = self._rows(B, "B", width, given), self._rows(C, "C", width, given)
        c.A = self._flat(A, "A", (self.channels, self.states), "float32", given)
        c.D = self._flat(D, "D", (self.channels,), "float32", given)
        c.deltaBias = self._flat(delta_bias, "delta_bias", (self.channels,), "float32", given)
        shape = (self.channels, self.states)
        c.initialState, first = self._states(initial_state, "initial_state", slots, shape, "float32", given)
        c.finalState, last = self._states(final_state, "final_state", slots, shape, "float32", given)
        if slots is not None:
            if first is not None and last is not None and first != last:
                raise ValueError("initial_state and final_state have different numbers of places")
            c.sequences.numSlots = first or last or 0
        same_device(given, self.device)
        size = _size_t()
        if out is not None:
            _abi.check(self._lib.gennmi_selective_scan_workspace(_byref(c), _byref(size)))
        self.workspace_bytes = size.value
        self._bound, self._bound_packed, self._descriptor, self._reference, self._gradients = given, self._packed, c, _byref(c), None

    def run(self, stream=0, workspace=None):
        """``workspace``: ``workspace_bytes`` on the device, for a call that is captured into a graph (which keeps using it)."""
        if self._bound is None:
            raise RuntimeError("bind() must be called first")
        address, size = self._workspace("forward", workspace, self.workspace_bytes, stream) if self.workspace_bytes else (None, 0)
        rc = self._lib.gennmi_selective_scan(self._reference, address, size, stream)
        if rc:
            _abi.check(rc)

    def bind_gradients(self, out, u=None, delta=None, A=None, B=None, C=None, D=None, delta_bias=None, z=None, initial_state=None, final_state=None):
        """``out`` and ``final_state``: gradients that come in; the others are written."""
        self._need(self._bound, "bind()")
        self._packed = self._bound_packed
        given, width = [], self.groups * self.states
        g = _abi.ScanGradient()
        for field, array, n in (("out", out, self.channels), ("u", u, self.channels), ("delta", delta, self.channels), ("z", z, self.channels),
                                ("B", B, width), ("C", C, width)):
            setattr(g, field, self._rows(array, f"the gradient of {field}", n, given))
        shape = (self.sequences, self.channels, self.states)
        g.finalState = self._flat(final_state, "the gradient of final_state", shape, "float32", given)
        g.initialState = self._flat(initial_state, "the gradient of initial_state", shape, "float32", given)
        g.A = self._flat(A, "the gradient of A", (self.channels, self.states), "float32", given)
        g.D = self._flat(D, "the gradient of D", (self.channels,), "float32", given)
        g.deltaBias = self._flat(delta_bias, "the gradient of delta_bias", (self.channels,), "float32", given)
        same_device(given, self.device)
        size = _size_t()
        _abi.check(self._lib.gennmi_selective_scan_backward_workspace(self._reference, _byref(size)))
        self.backward_workspace_bytes = size.value
        self._gradients, self._gradient_descriptor, self._gradient_reference = given, g, _byref(g)

    def backward(self, stream=0, workspace=None):
        """``workspace``: ``backward_workspace_bytes`` on the device, as for ``run``."""
        self._need(self._gradients, "bind_gradients()")
        address, size = self._workspace("backward", workspace, self.backward_workspace_bytes, stream)
        rc = self._lib.gennmi_selective_scan_backward(self._reference, self._gradient_reference, address, size, stream)
        if rc:
            _abi.check(rc)


class GatedDeltaRule(_SequenceOperator):
    """S[t] = a S[t-1] + k (x) beta (v - a S[t-1]' k) with a = exp(g),  out[t] = scale S[t]' q; with ``normalise`` q and k divided by sqrt(sum of squares + epsilon).

    ``q, k``: rows of key_heads x keys (heads / key_heads neighbouring heads share a key head); ``v, out``: rows of heads x values; ``g, beta``: rows of heads,
    float32.  Rows, ``offsets`` and ``slots`` as for ``CausalConvolution``; states [sequences or places, heads, keys, values] are float32.  ``scale``: keys ** -0.5 unless it
    is given.  ``length=1`` is a token of every running sequence."""

    def __init__(self, sequences, length, heads, keys, values, key_heads=None, dtype="float32", normalise=False, scale=None, epsilon=1e-6, device=0):
        super().__init__(sequences, length, dtype, device)
        self.heads, self.keys, self.values = _count(heads, "heads"), _count(keys, "keys"), _count(values, "values")
        self.key_heads = self.heads if key_heads is None else _count(key_heads, "key_heads")
        self.normalise, self.epsilon = bool(normalise), float(epsilon)
        self.scale = max(1, self.keys) ** -0.5 if scale is None else float(scale)
        self._width = self.key_heads * self.keys

    def _widths(self):
        return (("q", self._width, None), ("k", self._width, None), ("v", self.heads * self.values, None), ("g", self.heads, "float32"), ("beta", self.heads, "float32"))

    def bind(self, q, k, v, g, beta, out=None, initial_state=None, final_state=None, offsets=None, slots=None):
        given = []
        c = _abi.DeltaRule(type=_abi.FLOAT_TYPES[self.dtype], heads=self.heads, keyHeads=self.key_heads, keys=self.keys, values=self.values, normalise=self.normalise,
                           scale=self.scale, epsilon=self.epsilon)
        c.sequences = self._sequences(offsets, slots, q, given)
        for (field, width, dtype), array in zip(self._widths(), (q, k, v, g, beta)):
            setattr(c, field, self._rows(array, field, width, given, dtype))
        c.out = self._rows(out, "out", self.heads * self.values, given)
        shape = (self.heads, self.keys, self.values)
        c.initialState, first = self._states(initial_state, "initial_state", slots, shape, "float32", given)
        c.finalState, last = self._states(final_state, "final_state", slots, shape, "float32", given)
        if slots is not None:
            if first is not None and last is not None and first != last:
                raise ValueError("initial_state and final_state have different numbers of places")
            c.sequences.numSlots = first or last or 0
        same_device(given, self.device)
        size = _size_t()
        if out is not None:
            _abi.check(self._lib.gennmi_delta_rule_workspace(_byref(c), _byref(size)))
        self.workspace_bytes = size.value
        self._bound, self._bound_packed, self._descriptor, self._reference, self._gradients = given, self._packed, c, _byref(c), None

    def run(self, stream=0, workspace=None):
        """``workspace``: ``workspace_bytes`` on the device, for a call that is captured into a graph (which keeps using it)."""
        if self._bound is None:
            raise RuntimeError("bind() must be called first")
        address, size = self._workspace("forward", workspace, self.workspace_bytes, stream) if self.workspace_bytes else (None, 0)
        rc = self._lib.gennmi_delta_rule(self._reference, address, size, stream)
        if rc:
            _abi.check(rc)

    def bind_gradients(self, out, q=None, k=None, v=None, g=None, beta=None, initial_state=None, final_state=None):
        """``out`` and ``final_state``: gradients that come in; the others are written."""
        self._need(self._bound, "bind()")
        self._packed = self._bound_packed
        given = []
        d = _abi.DeltaRuleGradient()
        d.out = self._rows(out, "the gradient of out", self.heads * self.values, given)
        for (field, width, dtype), array in zip(self._widths(), (q, k, v, g, beta)):
            setattr(d, field, self._rows(array, f"the gradient of {field}", width, given, dtype))
        shape = (self.sequences, self.heads, self.keys, self.values)
        d.finalState = self._flat(final_state, "the gradient of final_state", shape, "float32", given)
        d.initialState = self._flat(initial_state, "the gradient of initial_state", shape, "float32", given)
        same_device(given, self.device)
        size = _size_t()
        _abi.check(self._lib.gennmi_delta_rule_backward_workspace(self._reference, _byref(size)))
        self.backward_workspace_bytes = size.value
        self._gradients, self._gradient_descriptor, self._gradient_reference = given, d, _byref(d)

    def backward(self, stream=0, workspace=None):
        """``workspace``: ``backward_workspace_bytes`` on the device, as for ``run``."""
        self._need(self._gradients, "bind_gradients()")
        address, size = self._workspace("backward", workspace, self.backward_workspace_bytes, stream)
        rc = self._lib.gennmi_delta_rule_backward(self._reference, self._gradient_reference, address, size, stream)
        if rc:
            _abi.check(rc)


class LayerNorm(_SequenceOperator):
    """out = (x' weight + bias) gate sigmoid(gate) with x' = (x - mean) / sqrt(variance + epsilon) of every row, or with ``rms`` x / sqrt(mean of squares + epsilon).

    ``x, gate, out``: [sequences, length, channels] (or both first axes as one); the heads of a row are such a length.  ``weight, bias``: [channels], float32; without them 1 and 0.
    ``out`` may be ``x`` or ``gate`` itself."""

    def __init__(self, sequences, length, channels, epsilon=1e-5, rms=False, dtype="float32", device=0):
        super().__init__(sequences, length, dtype, device)
        self.channels, self.epsilon, self.rms = _count(channels, "channels"), float(epsilon), bool(rms)

    def bind(self, x, weight=None, bias=None, gate=None, out=None):
        given = []
        c = _abi.LayerNorm(type=_abi.FLOAT_TYPES[self.dtype], channels=self.channels, rms=self.rms, epsilon=self.epsilon)
        c.sequences = self._sequences(None, None, x, given)
        for field, array in (("x", x), ("gate", gate), ("out", out)):
            setattr(c, field, self._rows(array, field, self.channels, given))
        c.weight = self._flat(weight, "weight", (self.channels,), "float32", given)
        c.bias = self._flat(bias, "bias", (self.channels,), "float32", given)
        same_device(given, self.device)
        self._bound, self._descriptor, self._reference, self._gradients = given, c, C.byref(c), None

    def run(self, stream=0):
        if self._bound is None:
            raise RuntimeError("bind() must be called first")
        rc = self._lib.gennmi_layer_norm(self._reference, stream)
        if rc:
            _abi.check(rc)

    def bind_gradients(self, out, x=None, weight=None, bias=None, gate=None):
        """``out``: the gradient that comes in; the others are written."""
        self._need(self._bound, "bind()")
        given = []
        g = _abi.LayerNormGradient()
        for field, array in (("out", out), ("x", x), ("gate", gate)):
            setattr(g, field, self._rows(array, f"the gradient of {field}", self.channels, given))
        g.weight = self._flat(weight, "the gradient of weight", (self.channels,), "float32", given)
        g.bias = self._flat(bias, "the gradient of bias", (self.channels,), "float32", given)
        same_device(given, self.device)
        size = C.c_size_t()
        _abi.check(self._lib.gennmi_layer_norm_backward_workspace(self._reference, C.byref(size)))
        self.backward_workspace_bytes = size.value if weight is not None or bias is not None else 0
        self._gradients, self._gradient_descriptor, self._gradient_reference = given, g, C.byref(g)

    def backward(self, stream=0, workspace=None):
        """``workspace``: ``backward_workspace_bytes`` on the device, for a call that is captured into a graph (which keeps using it)."""
        self._need(self._gradients, "bind_gradients()")
        address, size = self._workspace("backward", workspace, self.backward_workspace_bytes, stream)
        rc = self._lib.gennmi_layer_norm_backward(self._reference, self._gradient_reference, address, size, stream)
        if rc:
            _abi.check(rc)


class Dropout(_SequenceOperator):
    """out = residual + (kept ? x / (1 - probability) : 0), the probability in 65536ths.  No mask is stored: ``backward`` draws it again.

    ``x, residual, out``: [sequences, length, channels] (or both first axes as one).  What is kept depends on ``seed``, on the ``call`` (the number of a step and layer, say)
    and on the place of an element among rows and channels, not on strides.  ``out`` may be ``x`` or ``residual`` itself."""

    def __init__(self, sequences, length, channels, probability, seed=0, dtype="float32", device=0):
        super().__init__(sequences, length, dtype, device)
        self.channels, self.probability, self.seed = _count(channels, "channels"), float(probability), int(seed)
        self._numbers, self._captured = {}, []          # numbers on the device that are kept alive: the last one of each direction and stream, those of captured calls
        if not 0.0 <= self.probability <= 1.0:
            raise ValueError(f"probability is between 0 and 1, not {probability}")
        if not 0 <= self.seed < 1 << 64:
            raise ValueError("seed has 64 bits")

    def _descriptor_of(self, given, x, out, residual, names):
        d = _abi.Dropout(type=_abi.FLOAT_TYPES[self.dtype], channels=self.channels, probability=self.probability, seed=self.seed)
        d.sequences = self._sequences(None, None, x, given)
        for field, array, name in zip(("x", "out", "residual"), (x, out, residual), names):
            setattr(d, field, self._rows(array, name, self.channels, given))
        same_device(given, self.device)
        return d

    def bind(self, x, out, residual=None):
        given = []
        self._forward = self._descriptor_of(given, x, out, residual, ("x", "out", "residual"))
        self._bound = given

    def bind_gradients(self, out, x):
        """``out``: the gradient that comes in; ``x``: the one that is written (may be the same array).  The residual's gradient is ``out`` itself."""
        given = []
        self._backward = self._descriptor_of(given, out, x, None, ("the gradient of out", "the gradient of x", ""))
        self._gradients = given

    def _call(self, which, call, stream):
        d = _abi.Dropout.from_buffer_copy(getattr(self, which))         # (of this call alone: other threads may call with other numbers)
        if isinstance(call, Integral):          # (numpy's numbers are that too)
            if not 0 <= call < 1 << 64:
                raise ValueError("call has 64 bits")
            d.call = int(call)
        else:
            o = Operand(call, "call").wants(("uint64", "int64"))
            if any(n != 1 for n in o.shape):
                raise ValueError("call is one value")
            same_device([o], self.device)
            d.callDevice = o.address
            capturing = _int()
            if stream:
                _abi.check(self._lib.gennmi_stream_is_capturing(stream, _byref(capturing)))
            if not capturing.value:
                self._numbers[which, stream] = o
            elif all(k.address != o.address for k in self._captured):
                self._captured.append(o)
        rc = self._lib.gennmi_dropout(_byref(d), stream)
        if rc:
            _abi.check(rc)

    def run(self, call, stream=0):
        """``call``: a number, or an int64 or uint64 array of one element on the device that is read when the call runs.  It has to live until then; the object itself keeps
        those of captured calls, which go on reading them, and the last one of every stream."""
        self._need(self._bound, "bind()")
        self._call("_forward", call, stream)

    def backward(self, call, stream=0):
        """``call``: that of ``run``."""
        self._need(self._gradients, "bind_gradients()")
        self._call("_backward", call, stream)


# (`C` names an array of the scan)
_byref, _size_t, _int = C.byref, C.c_size_t, C.c_int
