"""A HIP graph of library calls, captured on the library's stream through the HIP runtime it has loaded."""
import ctypes

import freeml_amd as fh


def _runtime():
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64" in line)
    return ctypes.CDLL(path)


class Captured:
    def __init__(self, calls):
        self.hip, self.stream = _runtime(), ctypes.c_void_p(fh.lib().fmlh_get_stream())
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        fh.synchronize()
        self._check(self.hip.hipStreamBeginCapture(self.stream, 1))  # thread-local
        try:
            calls()
        finally:
            rc = self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph))
        self._check(rc)
        self._check(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)))
        self._check(self.hip.hipGraphDestroy(graph))

    def _check(self, rc):
        assert rc == 0, f"HIP error {rc}"

    def replay(self):
        self._check(self.hip.hipGraphLaunch(self.exec, self.stream))

    def close(self):
        fh.synchronize()
        self._check(self.hip.hipGraphExecDestroy(self.exec))
