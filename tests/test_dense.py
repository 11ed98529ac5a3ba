"""The dense operators without a GPU: the oracle's gradients against differences, arguments refused before any device is
touched, and the host code over a stand-in for the HIP runtime (which launches a call makes, its workspace, its refusals)."""

from pathlib import Path

import numpy as np
import pytest

from artlite_amd import _hip
from artlite_amd.device import View, overlap
from oracle import dense

from .fake_runtime import run_fake

PRELUDE = """
from artlite_amd.device import DeviceArray, Workspace, shared_workspace
from artlite_amd.ffn import GatedFFN
from artlite_amd.linear import QLinear
def refused(text, call):
    try: call()
    except _hip.Error as e: assert text in str(e), e
    else: raise AssertionError(text)
def linear(N, K, q="Q4_0", bias=False):
    l = QLinear(q, N, K)
    l.upload(np.zeros(N * (K // BLOCK[q][0]) * BLOCK[q][1], np.uint8), bias=np.zeros(N, np.float32) if bias else None)
    return l
def block(H, F, q="Q4_0", d="Q4_1"):
    f = GatedFFN(hidden=H, ffn=F, gate_type=q, down_type=d)
    for name, t, r, c in (("ffn_gate", q, F, H), ("ffn_up", q, F, H), ("ffn_down", d, H, F)):
        f.upload(name, np.zeros(r * (c // BLOCK[t][0]) * BLOCK[t][1], np.uint8))
    return f
def arr(n, c, dtype=np.uint16): return DeviceArray((n, c), dtype)
"""


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_oracle_gradients(act: str) -> None:
    """Central differences with a step of 1e-5 in 64 bits: off by the step's square and 1e-16 over the step."""
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((3, 5)), rng.standard_normal((3, 5))
    w = [rng.standard_normal(s) for s in ((7, 5), (7, 5), (5, 7))]
    got = dense.ffn_grad(act, x, dy, *w)
    for name, i in (("dx", None), ("dgate", 0), ("dup", 1), ("ddown", 2)):
        at = x if i is None else w[i]
        want = np.empty_like(at)
        for j in np.ndindex(at.shape):
            v = at[j]
            at[j] = v + 1e-5
            hi = (dense.ffn(act, x, *w) * dy).sum()
            at[j] = v - 1e-5
            want[j] = (hi - (dense.ffn(act, x, *w) * dy).sum()) / 2e-5
            at[j] = v
        assert np.abs(got[name] - want).max() < 1e-7 * max(1.0, np.abs(want).max())


def test_views() -> None:
    """What an argument's description says, and which memory two of them share."""
    class Cai:
        def __init__(self, ptr: int, shape: tuple, typestr: str, strides: tuple | None = None):
            self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "strides": strides}

    v = View(Cai(4096, (3, 8), "<u2", (32, 2)), "x")
    assert (v.at, v.code, v.rows, v.cols, v.row) == (4096, 1, 3, 8, 16)
    assert View(Cai(4096, (3, 8), "<f4"), "x").row == 8
    for bad, text in ((Cai(0, (3, 8), "<f8"), "float32 or bfloat16"), (Cai(0, (8,), "<f4"), "not .rows, values."),
                      (Cai(0, (3, 8), "<u2", (2, 6)), "values are 3.0 apart"),
                      (Cai(0, (3, 8), "<u2", (17, 2)), "rows 8.5 values apart"), (np.zeros((2, 2)), "is no array")):
        with pytest.raises(_hip.Error, match=text):
            View(bad, "x")
    a, b = View(Cai(0, (3, 8), "<u2", (32, 2)), "a"), View(Cai(80, (3, 8), "<u2", (32, 2)), "b")
    assert not overlap(a, b) and overlap(a, View(Cai(79, (1, 8), "<u2"), "c")) and overlap(a, a)
    assert not overlap(a, View(Cai(0, (0, 8), "<u2"), "none"))


def test_shapes_refused(tmp_path: Path) -> None:
    run_fake(tmp_path, PRELUDE + """
for q, N, K, text in (("Q8_0", 64, 64, "weight type 8 (Q8_0) is not one of"), ("Q4_0", 64, 48, "in blocks of 32"),
                      ("Q4_K", 64, 128, "in blocks of 256"), ("Q4_0", 0, 32, "0 rows"), ("Q4_0", 32, 0, "of 0 values"),
                      ("Q4_0", 1 << 25, 32, "rows of 32"), ("none", 64, 64, "weight type -1 (unknown)")):
    refused(text, lambda: QLinear(q, N, K))
l = QLinear("Q4_0", 64, 64)
refused("not uploaded", lambda: l(arr(1, 64), arr(1, 64)))
refused("100 bytes, not 2304", lambda: l.upload(np.zeros(100, np.uint8)))
refused("63 values for 64 rows", lambda: l.upload(np.zeros(2304, np.uint8), bias=np.zeros(63, np.float32)))
refused("activation 'relu'", lambda: GatedFFN(hidden=64, ffn=64, gate_type="Q4_0", down_type="Q4_0", act="relu"))
lib, f = _hip.lib(), block(64, 96)
refused("'ffn_norm', not one of ffn_gate, ffn_up, ffn_down", lambda: f.upload("ffn_norm", np.zeros(4, np.uint8)))
import ctypes
def matrix(N, K, q="Q4_0", bias=False): return linear(N, K, q, bias)._m
g, u, d = matrix(96, 64), matrix(96, 64), matrix(64, 96)
KEEP = []
def need(*m, act=0, n=4, dtype=1):
    KEEP.append(m)
    z = ctypes.c_size_t(0)
    _hip.check(lib.artlite_ffn_workspace(ctypes.byref(_hip.Ffn(*(x.handle.value for x in m), act)), dtype, n, 0, ctypes.byref(z)))
    return z.value
assert need(g, u, d) > 0 and need(g, u, d, n=0) == 0
refused("gate 96 x 64 (Q4_0), up 96 x 64 (Q4_1)", lambda: need(g, matrix(96, 64, "Q4_1"), d))
refused("down 96 x 64", lambda: need(g, u, matrix(96, 64)))
refused("a matrix with a bias", lambda: need(g, u, matrix(64, 96, bias=True)))
refused("activation 2", lambda: need(g, u, d, act=2))
refused("dtype 2", lambda: need(g, u, d, dtype=2))
refused("-1 rows", lambda: need(g, u, d, n=-1))
refused("rows", lambda: need(g, u, d, n=1 << 30))
""")


def test_device_arguments_refused(tmp_path: Path) -> None:
    """Addresses, strides and workspaces that the kernels could not take, at the C entry."""
    run_fake(tmp_path, PRELUDE + """
import ctypes
lib = _hip.lib()
l, f = linear(4096, 1024), block(1024, 96)
x, y = arr(400, 1024), arr(400, 4096)
def call(x=x.data_ptr(), n=4, xs=1024, y=y.data_ptr(), ys=4096, dtype=1, work=None):
    _hip.check(lib.artlite_linear(l._m.handle, x, dtype, n, xs, y, ys, work, None))
before = hip.launches
call()
assert hip.launches == before + 1
call(n=0, x=None, y=None)
assert hip.launches == before + 1
refused("x: null", lambda: call(x=None))
refused("y: rows of 4096 values 63 apart", lambda: call(ys=63))
refused("x: rows of 1024 values -1 apart", lambda: call(xs=-1))
refused("not aligned to its values", lambda: call(x=x.data_ptr() + 1))
refused("not aligned to its values", lambda: call(dtype=0, x=x.data_ptr() + 2))
refused("dtype 7", lambda: call(dtype=7))
refused("-1 rows", lambda: call(n=-1))
refused("needs a workspace of", lambda: call(n=300))
small, enough = Workspace(64), Workspace(l.workspace_bytes(300))
refused("a workspace of 64 bytes, not", lambda: call(n=300, work=small.handle))
hip.host_pointers = 1
refused("x: not device memory", call)
hip.host_pointers = 0
assert hip.launches == before + 1
call(n=300, work=enough.handle)
z = arr(400, 1024)
def back(dx=z, dy=x, **w): f.backward(x, dy, dx=dx, **w)
refused("dx overlaps dy", lambda: back(dy=z))
refused("no dy", lambda: back(dy=None))
refused("ddown is (96, 1024)", lambda: back(ddown=arr(96, 1024)))
""".replace("hip.fake_host = 0\n", ""))


def test_workspaces(tmp_path: Path) -> None:
    """Calls that are given no workspace share one a device; it grows, refuses captures and is free again after a call that
    failed; calls on another stream than the last one's wait for it."""
    run_fake(tmp_path, PRELUDE + """
l, f = linear(4096, 1024), block(1024, 96)
mallocs = lambda: hip.mallocs
def run(n, stream=0, **k): l(X[:n], Y[:n], stream=stream, **k)
class Rows:
    def __init__(self, a, n): self.a, self.shape, self.dtype = a, (n, a.shape[1]), a.dtype
    def data_ptr(self): return self.a.data_ptr()
    def stride(self): return self.a.stride()
class Whole:
    def __init__(self, n, c): self.a = arr(n, c)
    def __getitem__(self, s): return Rows(self.a, s.stop)
X, Y = Whole(5000, 1024), Whole(5000, 4096)
assert l.workspace_bytes(16) == 0 == l.workspace_bytes(16, "f32") and l.workspace_bytes(300) > 0
run(300)
Z = Whole(200, 1024)
at = hip.mallocs
run(300); f(X[:200], Z[:200]); run(290)
assert hip.mallocs <= at + 1
big = hip.mallocs
run(5000); run(5000); run(300)
assert hip.mallocs == big + 1
waits = hip.waits
run(300); run(300)
assert hip.waits == waits
run(300, stream=5); run(300, stream=5); run(300)
assert hip.waits == waits + 2
big_rows = arr(50000, 1024), arr(50000, 4096)
hip.capturing = 1
refused("a captured call takes a workspace of its own", lambda: run(300))
at = hip.mallocs
refused("a captured call takes a workspace of its own", lambda: l(*big_rows))
assert hip.mallocs == at
run(16)
own = Workspace(l.workspace_bytes(300))
run(300, work=own)
hip.capturing = 0
for i in range(3):
    hip.fail_launch = hip.launches + i
    refused("invalid", lambda: run(300))
    hip.fail_launch = -1
    run(300)
own.close()
# what a call needs does not depend on what a matrix holds
for q in ("Q4_0", "Q4_1"):
    w = QLinear(q, 256, 32768)
    need = [w.workspace_bytes(n) for n in (300, 512, 2000)]
    for fill in (0, 0x3c, 0x7c):
        w.upload(np.full(256 * 1024 * BLOCK[q][1], fill, np.uint8))
        assert need == [w.workspace_bytes(n) for n in (300, 512, 2000)]
refused("closed", lambda: run(300, work=own))
""")


def test_launch_shapes(tmp_path: Path) -> None:
    """Every launch of calls from one row to thousands, of odd and large shapes, is one that the device takes."""
    run_fake(tmp_path, PRELUDE + """
for q in ("Q4_0", "Q4_1", "Q4_K", "IQ4_NL", "IQ4_XS"):
    for N, K in ((1, 256), (17, 768), (131072, 2048), (4096, 12288), (2048, 16384)):
        l = linear(N, K, q)
        for dtype in (np.uint16, np.float32):
            for n in (1, 4, 5, 8, 16, 17, 32, 33, 64, 128, 129, 256, 257, 1000, 5000):
                l(arr(n, K, dtype), arr(n, N, dtype))
        l.close()
for H, F in ((32, 32), (2048, 8192), (4096, 11008)):
    f = block(H, F)
    for dtype in (np.uint16, np.float32):
        for n in (1, 16, 17, 64, 128, 129, 1000, 4096):
            x, dy, y = (arr(n, H, dtype) for _ in range(3))
            f(x, y)
            f.backward(x, dy, dx=y)
            f.backward(x, dy, dx=y, dgate=arr(F, H, dtype), dup=arr(F, H, dtype), ddown=arr(H, F, dtype))
""")
