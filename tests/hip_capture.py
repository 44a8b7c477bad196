"""Graphs of what a backend queues on a stream of the caller's, through the HIP runtime that the library has loaded."""
import contextlib
import ctypes
from ctypes import byref, c_void_p

import sparse_hip as sh


def _runtime():
    with open("/proc/self/maps") as f:
        paths = {line.split()[-1] for line in f if "libamdhip64" in line}
    assert len(paths) == 1, paths
    return ctypes.CDLL(paths.pop())


def _ok(status):
    assert status == 0, f"HIP error {status}"


class Captured:
    """A stream that `be` is set to, and on it: with cap.capture(): calls; then cap.replay()."""

    def __init__(self, be: sh.Backend):
        self.be, self.hip, self.stream, self.made = be, _runtime(), c_void_p(), None
        _ok(self.hip.hipStreamCreateWithFlags(byref(self.stream), 1))  # non-blocking
        be.set_stream(self.stream.value)

    @contextlib.contextmanager
    def capture(self):
        graph, made = c_void_p(), c_void_p()
        _ok(self.hip.hipStreamBeginCapture(self.stream, 1))  # of this thread
        try:
            yield
        finally:
            status = self.hip.hipStreamEndCapture(self.stream, byref(graph))
        _ok(status)  # (a call that cannot be captured ends the capture)
        _ok(self.hip.hipGraphInstantiate(byref(made), graph, None, None, ctypes.c_size_t(0)))
        _ok(self.hip.hipGraphDestroy(graph))
        self.made = made

    def replay(self):
        _ok(self.hip.hipGraphLaunch(self.made, self.stream))

    def close(self):
        self.be.synchronize()
        self.be.set_stream(None)
        self.be.synchronize()
        if self.made is not None:
            _ok(self.hip.hipGraphExecDestroy(self.made))
        _ok(self.hip.hipStreamDestroy(self.stream))
