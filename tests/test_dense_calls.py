"""The dense operators' calls without a GPU, over the stand-in for the HIP runtime: streams, arrays and what is refused."""

from pathlib import Path

import numpy as np

from artlite_amd import _hip
from artlite_amd.device import overlap
from artlite_amd.gguf_model import TYPE_ID
from artlite_amd.linear import FORMATS

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


class Span:
    """A view's fields, of bf16 values."""

    code = 1

    def __init__(self, at: int, rows: int, cols: int, row: int):
        self.at, self.rows, self.cols, self.row = at, rows, cols, row

    def bytes(self) -> set[int]:
        return {self.at + 2 * (i * self.row + j) + k for i in range(self.rows) for j in range(self.cols) for k in range(2)}


def test_overlap() -> None:
    """Against the bytes themselves: views of one buffer's columns share none, whatever they span. Where rows are different
    strides apart the answer may be yes without any."""
    rng = np.random.default_rng(1)
    apart = 0
    for _ in range(6000):
        s = int(rng.integers(1, 9))
        a, b = (Span(2 * int(rng.integers(0, 30)), int(rng.integers(0, 5)), int(rng.integers(1, 6)), s) for _ in range(2))
        exact = s >= max(a.cols, b.cols) or min(a.rows, b.rows) == 0 or max(a.rows, b.rows) == 1
        if rng.random() < 0.2:
            b.row = int(rng.integers(0, 9))
            exact = exact and (min(a.rows, b.rows) < 1 or a.row == b.row)
        met = bool(a.bytes() & b.bytes())
        assert overlap(a, b) == overlap(b, a)
        assert overlap(a, b) == met if exact else overlap(a, b) or not met, (vars(a), vars(b))
        ends = max(a.bytes(), default=0), max(b.bytes(), default=0)
        apart += exact and not met and a.at <= ends[1] and b.at <= ends[0]
    assert apart > 100  # (interleaved)


def test_columns_of_one_buffer(tmp_path: Path) -> None:
    run_fake(tmp_path, PRELUDE + """
l, f = linear(96, 64), block(64, 96)
whole = arr(300, 256)
class Columns:
    def __init__(self, first, cols): self.first, self.shape, self.dtype = first, (300, cols), whole.dtype
    def data_ptr(self): return whole.data_ptr() + 2 * self.first
    def stride(self): return 256, 1
x, y, z = Columns(0, 64), Columns(64, 96), Columns(192, 64)
assert l(x, y) is y and f(x, z) is z
f.backward(x, z, dx=Columns(128, 64))
refused("out overlaps x", lambda: l(x, Columns(63, 96)))
refused("out overlaps x", lambda: f(x, Columns(1, 64)))
refused("dx overlaps dy", lambda: f.backward(x, z, dx=Columns(190, 64)))
""")


def test_outputs_that_require_grad(tmp_path: Path) -> None:
    """A tensor that requires grad is not written while torch records a graph; it may be read, and written under no_grad."""
    run_fake(tmp_path, PRELUDE + """
import types
torch = types.ModuleType("torch")
torch.is_grad_enabled = lambda: RECORDS
sys.modules["torch"] = torch
class Tensor:
    requires_grad = True
    def __init__(self, n, c):
        self.a, self.shape, self.dtype = arr(n, c), (n, c), np.dtype(np.uint16)
        self.data_ptr, self.stride = self.a.data_ptr, self.a.stride
l, f = linear(96, 64), block(64, 96)
t64, t96, s64, w = Tensor(5, 64), Tensor(5, 96), Tensor(5, 64), Tensor(96, 64)
RECORDS = True
before = hip.launches
refused("linear: out: requires grad", lambda: l(t64, t96))
refused("ffn: out: requires grad", lambda: f(t64, s64))
refused("ffn backward: dx: requires grad", lambda: f.backward(t64, s64, dx=Tensor(5, 64)))
refused("ffn backward: dgate: requires grad", lambda: f.backward(t64, s64, dgate=w))
assert hip.launches == before
l(t64, arr(5, 96)); f.backward(t64, s64, dx=arr(5, 64))
RECORDS = False
l(t64, t96); f(t64, s64); f.backward(t64, s64, dgate=w)
""")


def test_streams_of_the_interface(tmp_path: Path) -> None:
    """A call waits for the stream that an array's ``__cuda_array_interface__`` names, where that is another than its own."""
    run_fake(tmp_path, PRELUDE + CAI + """
def on(stream, a):
    c = Cai(a)
    c.__cuda_array_interface__["stream"] = stream
    return c
l, f = linear(96, 64), block(64, 96)
x, y, z, w = arr(5, 64), arr(5, 96), arr(5, 64), arr(5, 64)
f(x, z)  # (its workspace)
def waits(call):
    before = hip.waits
    call()
    return hip.waits - before
assert waits(lambda: l(on(None, x), on(None, y))) == 0
assert waits(lambda: l(on(7, x), on(7, y))) == 1 == waits(lambda: l(x, on(7, y)))
assert waits(lambda: l(on(7, x), on(8, y))) == 2
assert waits(lambda: l(on(7, x), on(7, y), stream=7)) == 0
assert waits(lambda: l(on(1, x), y)) == 0 == waits(lambda: l(on(1, x), y, stream=None))
assert waits(lambda: l(on(1, x), y, stream=7)) == 1 == waits(lambda: l(on(2, x), y))
assert waits(lambda: f(on(7, x), z)) == 1 == waits(lambda: f.backward(x, on(7, w), dx=z))
refused("stream is 0", lambda: l(on(0, x), y))
at = hip.launches
hip.capturing = 1
refused("being captured", lambda: l(on(7, x), y))
assert hip.launches == at
l(on(None, x), y)
hip.capturing = 0
""")


def test_read_only_outputs(tmp_path: Path) -> None:
    """Memory whose interface says that it is read-only is read, not written."""
    run_fake(tmp_path, PRELUDE + CAI + """
def fixed(a):
    c = Cai(a)
    c.__cuda_array_interface__["data"] = (a.data_ptr(), True)
    return c
l, f = linear(96, 64), block(64, 96)
x, y, z, w = arr(5, 64), arr(5, 96), arr(5, 64), arr(5, 64)
l(fixed(x), y); f.backward(fixed(x), fixed(w), dx=z)
at = hip.launches
refused("linear: out: read-only", lambda: l(x, fixed(y)))
refused("ffn: out: read-only", lambda: f(x, fixed(z)))
refused("dup: read-only", lambda: f.backward(x, w, dup=fixed(arr(96, 64))))
assert hip.launches == at
""")


def test_formats() -> None:
    """What ``artlite_matrix_supported`` says is what the classes take."""
    assert {q for q, i in TYPE_ID.items() if _hip.lib().artlite_matrix_supported(i)} == set(FORMATS)
    assert not _hip.lib().artlite_matrix_supported(-1) and not _hip.lib().artlite_matrix_supported(1 << 20)


def test_shared_workspace_is_one(tmp_path: Path) -> None:
    """Growing frees what was outgrown (once no call uses it), and what is held is at most a quarter
    more than a call has needed."""
    run_fake(tmp_path, PRELUDE + """
import weakref
from artlite_amd import device as D
l = linear(4096, 1024)
x, y = arr(9000, 1024), arr(9000, 4096)
class Rows:
    def __init__(self, a, n): self.shape, self.dtype, self.data_ptr, self.stride = (n, a.shape[1]), a.dtype, a.data_ptr, a.stride
def run(n): l(Rows(x, n), Rows(y, n))
sizes = [300, 2000, 2100, 4000, 600, 610, 9000, 1000]
assert sorted(sizes, key=l.workspace_bytes) == sizes
old = None
for n in sizes:
    run(n)
    w = D._shared[0]
    assert l.workspace_bytes(n) <= w.nbytes <= 1.25 * l.workspace_bytes(n)
    assert old is None or old() is None or old() is w
    old = weakref.ref(w)
    del w
kept = shared_workspace(0, 1, 0)
run(5); shared_workspace(0, 2 * kept.nbytes, 0)
assert D._shared[0] is not kept and kept.handle and D._shared[0].nbytes == 2 * kept.nbytes
""")


def test_host_arrays_refused(tmp_path: Path) -> None:
    """A backward call on host arrays takes host arrays throughout, and no memory for two of its outputs."""
    run_fake(tmp_path, PRELUDE + """
f = block(64, 96)
x, dy, dx, g, u = (np.zeros(s, np.uint16) for s in ((5, 64), (5, 64), (5, 64), (96, 64), (96, 64)))
f.backward(x, dy, dx=dx, dgate=g, dup=u)
f.backward(x, dy, dx=x)  # (x is copied before)
both = np.zeros((96, 128), np.uint16)
f.backward(x, dy, dgate=both[:, :64], dup=both[:, 64:])
at = hip.launches
refused("dy is no host array", lambda: f.backward(x, None, dx=dx))
refused("dy is no host array", lambda: f.backward(x, arr(5, 64), dx=dx))
refused("dx is no host array", lambda: f.backward(x, dy, dx=arr(5, 64)))
refused("dgate is no host array", lambda: f.backward(x, dy, dgate=g.reshape(-1)))
refused("dup overlaps dgate", lambda: f.backward(x, dy, dgate=g, dup=g))
refused("dup overlaps dgate", lambda: f.backward(x, dy, dgate=both[:, 10:74], dup=both[:, 64:]))
assert hip.launches == at
""")
