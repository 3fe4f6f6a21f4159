"""Streams and graphs of the HIP runtime that the library runs on, for tests."""
import ctypes
import re


def runtime():
    """The runtime that is loaded already: another copy of it would have a device of its own."""
    with open("/proc/self/maps") as f:
        paths = set(re.findall(r"(/\S*libamdhip64\.so\S*)", f.read()))
    assert len(paths) == 1, paths
    return ctypes.CDLL(paths.pop())


def ok(rc):
    assert rc == 0, f"HIP error {rc}"


class Stream:
    def __init__(self):
        self.hip = runtime()
        p = ctypes.c_void_p()
        ok(self.hip.hipStreamCreateWithFlags(ctypes.byref(p), 1))  # non-blocking
        self.ptr = p.value

    def sync(self):
        ok(self.hip.hipStreamSynchronize(ctypes.c_void_p(self.ptr)))

    def begin(self):
        ok(self.hip.hipStreamBeginCapture(ctypes.c_void_p(self.ptr), 0))

    def end(self):
        g, e = ctypes.c_void_p(), ctypes.c_void_p()
        ok(self.hip.hipStreamEndCapture(ctypes.c_void_p(self.ptr), ctypes.byref(g)))
        ok(self.hip.hipGraphInstantiate(ctypes.byref(e), g, None, None, ctypes.c_size_t(0)))
        return e

    def replay(self, e):
        ok(self.hip.hipGraphLaunch(e, ctypes.c_void_p(self.ptr)))
        self.sync()
