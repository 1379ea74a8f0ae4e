"""What a call of dropout hands to the library is that call's own: other threads may call the same object meanwhile."""
import ctypes as C

from genn_amd import _abi
from genn_amd.sequence import Dropout


class Library:
    """Stands for the library: notes the numbers of the calls when it reads them, in the midst of which another thread may have called."""

    def __init__(self):
        self.read, self.meanwhile = [], None

    def gennmi_dropout(self, descriptor, stream):
        if self.meanwhile:
            call, self.meanwhile = self.meanwhile, None
            call()
        d = C.cast(descriptor, C.POINTER(_abi.Dropout)).contents
        self.read.append((d.call, d.callDevice, d.channels, stream))
        return 0


def plan():
    drop = Dropout.__new__(Dropout)
    drop._lib, drop._workspaces, drop.device = Library(), {}, 0
    drop._forward, drop._backward = _abi.Dropout(channels=8), _abi.Dropout(channels=8)
    drop._bound = drop._gradients = [1]
    return drop


def test_a_call_in_the_midst_of_another_does_not_change_its_number():
    drop = plan()
    drop._lib.meanwhile = lambda: drop.run(2, 7)
    drop.run(1, 5)
    assert drop._lib.read == [(2, None, 8, 7), (1, None, 8, 5)]
    drop._lib.meanwhile = lambda: drop.backward(4)
    drop.backward(3)
    assert drop._lib.read[2:] == [(4, None, 8, 0), (3, None, 8, 0)]
