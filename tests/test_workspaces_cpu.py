"""An operator's own workspaces, where two threads make the first call on a stream at once: both get the one that is kept."""
import threading

from genn_amd import _abi, sequence


class Library:
    def gennmi_init(self, device):
        return 0

    def gennmi_current_device(self, result):
        return 0


def test_two_first_calls_at_once_share_a_workspace(monkeypatch):
    inside = threading.Barrier(2)

    class Array:
        made = 0

        def __init__(self, count, dtype, device_only):
            Array.made += 1
            self.count, self.ptr = count, 4096 * Array.made
            try:
                inside.wait(0.3)            # (until the other thread is in here as well, if it can be)
            except threading.BrokenBarrierError:
                pass

        def free(self):
            pass

    monkeypatch.setattr(_abi, "load", Library)
    monkeypatch.setattr(sequence, "Array", Array)
    op = sequence.LayerNorm(1, 2, 8)
    got = []
    threads = [threading.Thread(target=lambda: got.append(op._workspace("backward", None, 64, 0))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert Array.made == 1 and got == [(4096, 64)] * 2
