"""Device arrays as the operators take them: an ``Array`` of this package, or a tensor that says where it lies, what it holds and how
(``data_ptr()``, ``dtype``, ``shape``, ``stride()``: torch's do).  Nothing is copied or cast."""
import ctypes as C

from . import _abi
from .genn_model import Array


class Operand:
    """``address``, name of the element type, ``shape`` and ``strides`` (in elements) of an array on the device."""

    def __init__(self, array, name, shape=None):
        if isinstance(array, Array):
            if not array.ptr:
                raise ValueError(f"{name}: the array has been freed")
            self.address, self.dtype = array.ptr, array.dtype.name
            self.shape = (array.count,)
            if shape is not None:       # (an Array is flat: it has the shape that is asked for, if its size is that)
                count = 1
                for n in shape:
                    count *= n
                if array.count != count:
                    raise ValueError(f"{name} has {array.count} elements, not {count}")
                self.shape = tuple(shape)
            self.strides = [1] * len(self.shape)
            for k in range(len(self.shape) - 2, -1, -1):
                self.strides[k] = self.strides[k + 1] * self.shape[k + 1]
            self.device = None
        elif hasattr(array, "data_ptr") and hasattr(array, "stride"):
            if not getattr(array, "is_cuda", False):
                raise ValueError(f"{name} is not on the device")
            self.address, self.dtype = array.data_ptr(), str(array.dtype).replace("torch.", "")
            self.shape, self.strides = tuple(array.shape), list(array.stride())
            self.device = array.device.index
        else:
            raise TypeError(f"{name}: neither an Array nor a tensor on the device")
        self.name = name
        self.array = array          # (kept alive by whoever keeps the operand)

    def wants(self, dtypes):
        if self.dtype not in ((dtypes,) if isinstance(dtypes, str) else dtypes):
            raise TypeError(f"{self.name} holds {self.dtype}, not {dtypes}")
        return self

    def contiguous(self, shape):
        """All of an array of that shape, its elements one behind another."""
        if self.shape != tuple(shape):
            raise ValueError(f"{self.name} has shape {self.shape}, not {tuple(shape)}")
        step = 1
        for n, stride in zip(reversed(self.shape), reversed(self.strides)):
            if n > 1 and stride != step:
                raise ValueError(f"{self.name} is not contiguous")
            step *= n
        return self

    def rows(self, sequences, length, width, packed_rows=None):
        """``Rows`` of [sequences, length, width], of [sequences * length, width], or of packed [at least packed_rows, width]."""
        shape, strides = self.shape, self.strides
        if packed_rows is not None:
            if len(shape) != 2 or shape[1] != width or shape[0] < packed_rows:
                raise ValueError(f"{self.name} has shape {shape}, not ({packed_rows} or more, {width})")
            row, sequence = strides[0], 0
        elif len(shape) == 3 and shape == (sequences, length, width):
            row, sequence = strides[1], strides[0]
        elif len(shape) == 2 and shape == (sequences * length, width):
            row, sequence = strides[0], strides[0] * length
        else:
            raise ValueError(f"{self.name} has shape {shape}, not ({sequences}, {length}, {width})")
        if width > 1 and strides[-1] != 1:
            raise ValueError(f"{self.name}: the elements of a row are not neighbours")
        if min(strides) < 0:
            raise ValueError(f"{self.name}: negative stride")
        return _abi.Rows(self.address, row, sequence)


def current_device(lib, device):
    """What is allocated lies on the device that is current: it has to be the operator's."""
    now = C.c_int()
    _abi.check(lib.gennmi_current_device(C.byref(now)))
    if now.value != device:
        raise ValueError(f"the current device is {now.value}, the operator's is {device}")


def same_device(operands, device):
    """The operators launch on the device that the library was initialised for."""
    for o in operands:
        if o is not None and o.device is not None and o.device != device:
            raise ValueError(f"{o.name} is on device {o.device}, the library on device {device}")
