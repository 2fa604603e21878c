"""A stream and captured graphs for the GPU tests, on a thread of their own (whose scratch starts empty)."""
import ctypes as C
import threading

from atlas_amd._lib import check, load


def hip_runtime():
    """The HIP runtime that the library uses (the copy loaded in this process)."""
    load()
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64.so" in line)
    hip = C.CDLL(path)
    for name in ("hipStreamCreate", "hipStreamDestroy", "hipStreamBeginCapture", "hipStreamEndCapture",
                 "hipGraphInstantiate", "hipGraphLaunch", "hipStreamSynchronize", "hipGraphExecDestroy",
                 "hipGraphDestroy"):
        getattr(hip, name).restype = C.c_int
    return hip


class Stream:
    """A stream that the thread's calls go to while it is entered."""

    def __init__(self, hip):
        self.hip, self.st, self.made = hip, C.c_void_p(), []

    def __enter__(self):
        assert self.hip.hipStreamCreate(C.byref(self.st)) == 0
        self.use()
        return self

    def use(self):
        check(load().atlas_set_thread_stream(self.st))

    def capture(self, fn):
        """fn()'s calls as a graph, and what fn returned."""
        graph, exe = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.st, 0) == 0
        try:
            got = fn()
        finally:
            rc = self.hip.hipStreamEndCapture(self.st, C.byref(graph))
        assert rc == 0
        assert self.hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        self.made.append((graph, exe))
        return exe, got

    def launch(self, exe):
        assert self.hip.hipGraphLaunch(exe, self.st) == 0

    def sync(self):
        assert self.hip.hipStreamSynchronize(self.st) == 0

    def __exit__(self, *exc):
        self.hip.hipStreamSynchronize(self.st)
        load().atlas_clear_thread_stream()
        for graph, exe in self.made:
            self.hip.hipGraphExecDestroy(exe)
            self.hip.hipGraphDestroy(graph)
        self.hip.hipStreamDestroy(self.st)


def on_thread(fn):
    """fn(hip) on a fresh thread; what it raises is raised here."""
    hip, bad = hip_runtime(), []

    def work():
        try:
            fn(hip)
        except BaseException as e:
            bad.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if bad:
        raise bad[0]
