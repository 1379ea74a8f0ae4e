"""What a call of dropout hands to the library is that call's own: other threads may call the same object meanwhile; and a number on the device lives as long as a call of the object may read it."""
import ctypes as C
import gc
import weakref

import pytest

from genn_amd import _abi
from genn_amd.sequence import Dropout


class Library:
    """Stands for the library: notes the numbers of the calls when it reads them, in the midst of which another thread may have called."""

    def __init__(self):
        self.read, self.meanwhile, self.capturing = [], None, False

    def gennmi_init(self, device):
        return 0

    def gennmi_stream_is_capturing(self, stream, result):
        C.cast(result, C.POINTER(C.c_int)).contents.value = self.capturing
        return 0

    def gennmi_dropout(self, descriptor, stream):
        if self.meanwhile:
            call, self.meanwhile = self.meanwhile, None
            call()
        d = C.cast(descriptor, C.POINTER(_abi.Dropout)).contents
        self.read.append((d.call, d.callDevice, d.channels, stream))
        return 0


class Tensor:
    """As much of a tensor on the device as an operand asks for."""
    is_cuda, dtype, device = True, "torch.int64", type("Device", (), dict(index=0))

    def __init__(self, address, shape=(1,)):
        self.address, self.shape = address, shape

    def data_ptr(self):
        return self.address

    def stride(self):
        return [1] * len(self.shape)


@pytest.fixture
def drop(monkeypatch):
    library = Library()
    monkeypatch.setattr(_abi, "load", lambda: library)
    made = Dropout(1, 1, 8, 0.5)
    made._forward, made._backward = _abi.Dropout(channels=8), _abi.Dropout(channels=8)
    made._bound = made._gradients = [1]
    return made


def test_a_call_in_the_midst_of_another_does_not_change_its_number(drop):
    drop._lib.meanwhile = lambda: drop.run(2, 7)
    drop.run(1, 5)
    assert drop._lib.read == [(2, None, 8, 7), (1, None, 8, 5)]
    drop._lib.meanwhile = lambda: drop.backward(4)
    drop.backward(3)
    assert drop._lib.read[2:] == [(4, None, 8, 0), (3, None, 8, 0)]
    drop._lib.meanwhile = lambda: drop.run(6)
    drop.run(Tensor(4096))
    drop.run(7)
    assert drop._lib.read[4:] == [(6, None, 8, 0), (0, 4096, 8, 0), (7, None, 8, 0)]


def test_numbers_on_the_device_are_kept_while_a_call_may_read_them(drop):
    numbers = [Tensor(4096 * k) for k in range(1, 6)]
    alive = [weakref.ref(n) for n in numbers]
    drop._lib.capturing = True
    drop.run(numbers[0], 3)
    drop.backward(numbers[0], 3)
    drop._lib.capturing = False
    drop.run(numbers[1], 3)
    drop.run(numbers[2], 4)
    drop.backward(numbers[3], 4)
    drop.run(8, 4)
    drop.run(numbers[4])
    del numbers
    gc.collect()
    assert all(a() is not None for a in alive)          # a graph's, and the last one of each stream and direction
    drop.run(Tensor(1 << 20), 3)
    gc.collect()
    assert alive[1]() is None and alive[0]() is not None and alive[2]() is not None
