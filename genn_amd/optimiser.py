"""AdamW over many tensors in one launch, over the C ABI in include/genn_mi355x.h."""
import ctypes as C
from numbers import Real

from . import _abi
from .genn_model import Array
from .operands import Operand, current_device, same_device

BLOCK = 256         # weights that share a scale of the states in 8 bits


class AdamW:
    """Decoupled weight decay (Loshchilov & Hutter 2019).  As a model's populations are added, built and then stepped:

        optimiser = AdamW(learning_rate=1e-3)
        optimiser.add(synapses.vars["g"], gradients)        # an Array of a model, or a tensor on the device
        optimiser.build()
        optimiser.step()                                    # one launch for all of them

    States are float32, or with ``state_bits=8`` codes in e4m3 with a float32 scale for each block of 256 weights.  The optimiser makes them
    (zero) unless they are given.  A step while another device than the optimiser's is current is refused.  Weights that a model's runner holds copies of reach it before its next step."""

    def __init__(self, learning_rate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, state_bits=32, device=0):
        self._lib = _abi.load()
        self._optimiser = C.c_void_p()
        _abi.check(self._lib.gennmi_init(device))
        settings = _abi.AdamWSettings(beta1=beta1, beta2=beta2, epsilon=epsilon, stateBits=state_bits)
        _abi.check(self._lib.gennmi_optimiser_create(C.byref(self._optimiser), C.byref(settings)))
        self.learning_rate, self.state_bits, self.device = learning_rate, state_bits, device
        self.states = []            # of each tensor: its arrays m, v (and m_scale, v_scale), as given or made
        self._own, self._given, self._built = [], [], False
        self._step = _abi.AdamWStep()
        self._reference = C.byref(self._step)

    def _array(self, array, name, count, dtypes, made):
        """An operand of `count` elements, of a shape that does not matter; made here where none is given."""
        if array is None:
            array = Array(count, made)
            self._own.append(array)
        o = Operand(array, name).wants(dtypes)
        size = 1
        for n in o.shape:
            size *= n
        if size != count:
            raise ValueError(f"{name} has {size} elements, not {count}")
        o.contiguous(o.shape)
        same_device([o], self.device)
        self._given.append(o)
        return o

    def add(self, weights, gradients, m=None, v=None, m_scale=None, v_scale=None, copy=None, weight_decay=0.0):
        """One tensor.  ``copy``: float16 or bfloat16, receives the new weights rounded (the ones a forward pass reads)."""
        if not self._optimiser:
            raise RuntimeError("the optimiser has been freed")
        current_device(self._lib, self.device)
        count = 1
        for n in Operand(weights, "weights").shape:
            count *= n
        floats = tuple(_abi.FLOAT_TYPES)
        w, g = self._array(weights, "weights", count, floats, None), self._array(gradients, "gradients", count, floats, None)
        p = _abi.Parameter(weight=w.address, gradient=g.address, count=count, weightType=_abi.FLOAT_TYPES[w.dtype], gradientType=_abi.FLOAT_TYPES[g.dtype],
                           weightDecay=weight_decay)
        if copy is not None:
            c = self._array(copy, "copy", count, ("float16", "bfloat16"), None)
            p.copy, p.copyType = c.address, _abi.FLOAT_TYPES[c.dtype]
        dtypes, made = (("float32",), "float32") if self.state_bits == 32 else (("float8_e4m3fn", "uint8"), "uint8")
        state = {"m": self._array(m, "m", count, dtypes, made), "v": self._array(v, "v", count, dtypes, made)}
        p.m, p.v = state["m"].address, state["v"].address
        if self.state_bits == 8:
            blocks = -(-count // BLOCK)
            state["m_scale"], state["v_scale"] = (self._array(s, n, blocks, ("float32",), "float32") for s, n in ((m_scale, "m_scale"), (v_scale, "v_scale")))
            p.mScale, p.vScale = state["m_scale"].address, state["v_scale"].address
        elif m_scale is not None or v_scale is not None:
            raise ValueError("states in 32 bits have no scales")
        index = C.c_uint32()
        _abi.check(self._lib.gennmi_optimiser_push(self._optimiser, C.byref(p), C.byref(index)))
        self.states.append({k: o.array for k, o in state.items()})
        return index.value

    def build(self):
        current_device(self._lib, self.device)
        _abi.check(self._lib.gennmi_optimiser_finalise(self._optimiser))
        self._built = True

    def step(self, learning_rate=None, gradient_scale=None, skip=None, stream=0):
        """``learning_rate``: a number, or a float32 array of one element on the device that the step reads when it runs.  ``gradient_scale`` (float32) and
        ``skip`` (int32 or uint32: not 0 leaves everything as it is): such arrays, or None.  A captured step goes on reading the arrays that it was given."""
        s = self._step
        rate = self.learning_rate if learning_rate is None else learning_rate
        on_device = not isinstance(rate, (int, float)) and not isinstance(rate, Real)       # (numpy's numbers are the second)
        s.rate, s.rateDevice = (0.0, self._scalar(rate, "learning_rate", "float32")) if on_device else (rate, None)
        self._values = (rate, gradient_scale, skip)         # (kept alive until the next step)
        s.gradientScale = None if gradient_scale is None else self._scalar(gradient_scale, "gradient_scale", "float32")
        s.skip = None if skip is None else self._scalar(skip, "skip", ("int32", "uint32"))
        rc = self._lib.gennmi_optimiser_step(self._optimiser, self._reference, stream)
        if rc:
            _abi.check(rc)

    def _scalar(self, array, name, dtypes):
        o = Operand(array, name).wants(dtypes)
        size = 1
        for n in o.shape:
            size *= n
        if size != 1:
            raise ValueError(f"{name} is one value")
        same_device([o], self.device)
        return o.address

    @property
    def steps(self):
        """Steps taken so far; assigned to after a checkpoint's states have been loaded."""
        n = C.c_uint64()
        _abi.check(self._lib.gennmi_optimiser_get_step(self._optimiser, C.byref(n)))
        return n.value

    @steps.setter
    def steps(self, n):
        _abi.check(self._lib.gennmi_optimiser_set_step(self._optimiser, n))

    def free(self):
        """Gives the table and the states that the optimiser made back."""
        if self._optimiser:
            self._lib.gennmi_optimiser_destroy(self._optimiser)
            self._optimiser = C.c_void_p()
        for a in self._own:
            a.free()
        self._own, self._given = [], []

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
