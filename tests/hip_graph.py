"""A context on a stream of its own, and graphs captured from its calls (the HIP runtime that
the library itself has loaded)."""
import ctypes as C

import numpy as np


class Hip:
    def __init__(self):
        with open("/proc/self/maps") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        self.lib = C.CDLL(path)

    def __getattr__(self, name):
        def call(*args):
            rc = getattr(self.lib, name)(*args)
            assert rc == 0, (name, rc)
        return call


class Captured:
    """A context (ctx) on its own stream; capture(call) is a replayable graph of call()."""

    def __init__(self, ops):
        self.ops, self.ctx = ops, ops.Context()
        self.hip, self.stream, self.graphs = Hip(), C.c_void_p(), []
        self.hip.hipStreamCreate(C.byref(self.stream))
        self.ctx.set_stream(self.stream.value)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.hip.hipStreamSynchronize(self.stream)
        for graph, exe in self.graphs:
            self.hip.hipGraphExecDestroy(exe)
            self.hip.hipGraphDestroy(graph)
        self.ctx.close()
        self.hip.hipStreamDestroy(self.stream)

    def buffer(self, x):
        return self.ops.DeviceBuffer.from_array(x, self.ctx)

    def put(self, buf, x):
        """New contents of a buffer, once the stream is done with it."""
        self.wait()
        x = np.ascontiguousarray(x)
        assert x.nbytes <= buf.nbytes
        self.hip.hipMemcpy(C.c_void_p(buf.ptr), x.ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes), 1)

    def wait(self):
        self.hip.hipStreamSynchronize(self.stream)

    def capture(self, call):
        graph, exe = C.c_void_p(), C.c_void_p()
        self.hip.hipStreamBeginCapture(self.stream, 0)
        try:
            call()
        finally:
            self.hip.hipStreamEndCapture(self.stream, C.byref(graph))
        self.hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0))
        self.graphs.append((graph, exe))
        return lambda: self.hip.hipGraphLaunch(exe, self.stream)
