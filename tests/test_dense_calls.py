"""The dense operators' calls without a GPU, over the stand-in for the HIP runtime: streams, arrays and what is refused."""

from pathlib import Path

from .fake_runtime import run_fake
from .test_dense import PRELUDE


def test_per_thread_streams(tmp_path: Path) -> None:
    """hipStreamPerThread (2) names another stream in each thread: a call on it waits for the workspace's last one, whichever
    thread that came from."""
    run_fake(tmp_path, PRELUDE + """
l = linear(4096, 1024)
x, y = arr(300, 1024), arr(300, 4096)
l(x, y, stream=2)
before = hip.waits
l(x, y, stream=2)
assert hip.waits == before + 1
l(x, y, stream=5); l(x, y, stream=5)
assert hip.waits == before + 2
""")


CAI = """
class Cai:  # (nothing but the interface)
    def __init__(self, a, rows=None, cols=None, typestr=None):
        n, c = a.shape
        self.keep = a
        self.__cuda_array_interface__ = {"shape": (n if rows is None else rows, cols or c), "strides": None, "version": 3,
                                         "typestr": typestr or {2: "<u2", 4: "<f4"}[a.dtype.itemsize],
                                         "data": (a.data_ptr(), False)}
"""


def test_arrays_of_the_interface_alone(tmp_path: Path) -> None:
    """Objects that have ``__cuda_array_interface__`` and nothing else, given and refused."""
    run_fake(tmp_path, PRELUDE + CAI + """
l, f = linear(96, 64), block(64, 96)
x, y, z, w = arr(5, 64), arr(5, 96), arr(5, 64), arr(5, 64)
before = hip.launches
out = Cai(y)
assert l(Cai(x), out) is out and hip.launches == before + 1
f(Cai(x), Cai(z))
f.backward(Cai(x), Cai(w), dx=Cai(z), dgate=Cai(arr(96, 64)))
assert hip.launches > before + 3
at = hip.launches
refused("for 96 rows of 64 values", lambda: l(Cai(x), Cai(z)))
refused("x (5, 64) of dtype 1, out (4, 96) of dtype 1", lambda: l(Cai(x), Cai(y, rows=4)))
refused("out is (4, 64)", lambda: f(Cai(x), Cai(z, rows=4)))
refused("float32 or bfloat16", lambda: l(Cai(x, typestr="<f8"), Cai(y)))
refused("dy is (4, 64)", lambda: f.backward(Cai(x), Cai(w, rows=4), dx=Cai(z)))
refused("x: NoneType is no array", lambda: f(None, z))
refused("x: list is no array", lambda: f.backward([1.0], w, dx=z))
assert hip.launches == at
""")
