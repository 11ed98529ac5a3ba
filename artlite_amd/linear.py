"""One matrix of a GGUF file as a product: ``y = x W^T + b`` for an attention projection, the output head or any other 2-D
tensor in a 4-bit format (Q4_0, Q4_1, Q4_K, IQ4_NL, IQ4_XS), from single tokens to prompts (``artlite_linear``). Beside
``moe.layer.MoELayer``, which takes a block's experts."""

import ctypes

import numpy as np

from . import _hip
from .device import DeviceArray, View, Workspace, after, overlap, shared_workspace
from .gguf_model import TYPE_ID, GGUFFile

FORMATS = ("Q4_0", "Q4_1", "Q4_K", "IQ4_NL", "IQ4_XS")


class Matrix:
    """A matrix's blocks in HBM (``artlite_matrix``)."""

    def __init__(self, qtype: str, rows: int, cols: int):
        self.qtype, self.rows, self.cols = qtype, rows, cols
        self._lib = _hip.lib()  # (close() may run when the module is gone)
        h = ctypes.c_void_p()
        _hip.check(self._lib.artlite_matrix_create(TYPE_ID.get(qtype, -1), rows, cols, ctypes.byref(h)))
        self._h = h
        d = ctypes.c_int(0)
        _hip.check(self._lib.artlite_matrix_device(h, ctypes.byref(d)))
        self.device = d.value

    @property
    def handle(self) -> ctypes.c_void_p:
        if self._h is None:
            raise _hip.Error("matrix: closed")
        return self._h

    def upload(self, raw: np.ndarray) -> None:
        a = np.ascontiguousarray(raw)
        _hip.check(_hip.lib().artlite_matrix_upload(self.handle, a.ctypes.data, a.nbytes))

    def upload_bias(self, bias: np.ndarray | None) -> None:
        b = np.empty(0, np.float32) if bias is None else np.ascontiguousarray(bias, np.float32).reshape(-1)
        _hip.check(_hip.lib().artlite_matrix_upload_bias(self.handle, b.ctypes.data if b.size else None, b.size))

    def close(self) -> None:
        if getattr(self, "_h", None) is not None:
            self._lib.artlite_matrix_destroy(self._h)
            self._h = None

    def __del__(self) -> None:
        self.close()


class QLinear:
    """``y = x W^T + b``: W (rows, cols) raw blocks, b fp32 or none; x and y (n, cols) and (n, rows), both bf16 or both
    fp32, any n. Products of x with the blocks' values are summed in fp32 and rounded once to y's type."""

    def __init__(self, qtype: str, rows: int, cols: int):
        self.rows, self.cols = rows, cols
        self._m = Matrix(qtype, rows, cols)

    @classmethod
    def from_gguf(cls, gguf: GGUFFile, name: str, bias: str = "") -> "QLinear":
        """Tensor ``name`` of a file (``blk.0.attn_q.weight``, ``output.weight``), with the F32 tensor ``bias`` if named."""
        t = gguf.tensor(name)
        if t.qtype not in FORMATS:
            raise ValueError(f"{gguf.path}: {name} is {t.qtype}, not one of {', '.join(FORMATS)}")
        b = None
        if bias:
            tb = gguf.tensor(bias)
            if tb.qtype != "F32" or tb.rows * tb.cols != t.rows:
                raise ValueError(f"{gguf.path}: {bias} is {tb.qtype} ({tb.rows * tb.cols} values) for {t.rows} rows")
            b = np.asarray(tb.raw)
        lin = cls(t.qtype, t.rows, t.cols)
        lin.upload(t.raw, bias=b)
        return lin

    def upload(self, raw: np.ndarray, bias: np.ndarray | None = None) -> None:
        """The rows' blocks as the file holds them, and the bias (none: without)."""
        self._m.upload(raw)
        self._m.upload_bias(bias)

    def close(self) -> None:
        self._m.close()

    def workspace_bytes(self, n: int, dtype: str = "bf16") -> int:
        """What a call of n rows needs (0 for up to 16)."""
        return self._need({"f32": 0, "bf16": 1}[dtype], n)

    def _need(self, code: int, n: int) -> int:
        z = ctypes.c_size_t(0)
        _hip.check(_hip.lib().artlite_linear_workspace(self._m.handle, code, n, ctypes.byref(z)))
        return z.value

    def __call__(self, x: object, out: object = None, *, stream: int = 0, work: Workspace | None = None) -> object:
        """x (n, cols) -> out (n, rows). Device arrays (``device``): enqueued on ``stream`` (a hipStream_t's address; 0: the
        null stream), ``out`` given by the caller, ``work`` its workspace (none: one that the device's
        calls share, which a captured call may not use; up to 16 rows need none). A numpy x (fp32, or uint16 bf16 bits): the
        result as a numpy array."""
        if isinstance(x, np.ndarray):
            if out is not None:
                raise _hip.Error("linear: out goes with device arrays")
            d = DeviceArray.of(x, self._m.device)
            return self(d, DeviceArray((d.shape[0], self.rows), x.dtype, d.device), stream=stream, work=work).numpy()
        a, y = View(x, "linear: x"), View(out, "linear: out", True)
        n = a.rows
        if a.cols != self.cols or y.rows != n or y.cols != self.rows or y.code != a.code:
            raise _hip.Error(f"linear: x ({a.rows}, {a.cols}) of dtype {a.code}, out ({y.rows}, {y.cols}) of dtype {y.code} for "
                             f"{self.rows} rows of {self.cols} values")
        if overlap(a, y):
            raise _hip.Error("linear: out overlaps x")
        handle = self._m.handle
        w = None
        if work is not None:
            w = work.handle
        elif n > 16:
            need = self._need(a.code, n)
            if need:
                work = shared_workspace(self._m.device, need, stream)
                w = work.handle
        if a.stream is not None or y.stream is not None:
            after(self._m.device, stream, (a, y))
        _hip.check(_hip.lib().artlite_linear(handle, a.at, a.code, n, a.row, y.at, y.row, w, stream))
        return out
