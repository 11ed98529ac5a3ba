"""Arrays in GPU memory for the dense operators (``linear``, ``ffn``), and their workspaces. No torch: an operator takes

- a ``DeviceArray`` (this module's own, for programs without an allocator),
- any object that describes device memory: with ``data_ptr()``, ``shape``, ``stride()`` and ``dtype`` (a torch tensor), or
  with ``__cuda_array_interface__``
  (a program that uses torch imports it before this package's library loads, so that both share torch's HIP runtime: memory
  of another runtime is refused),
- or a host numpy array: copied to the GPU, computed there, and its result copied back before the call returns.

Calls record no graph for torch's autograd: as with torch's own ``out=``, a tensor that requires grad is not written while it
records one.

Arrays are (rows, values) of fp32 or bf16 (numpy has no bf16: uint16 bit patterns), each row's values consecutive."""

import ctypes
import sys
import threading
from collections.abc import Iterable

import numpy as np

from . import _hip

F32, BF16 = 0, 1  # artlite_dtype
_CODES: dict[object, int] = {}  # a dtype object seen before -> its code
_NAMES = {"float32": F32, "torch.float32": F32, "<f4": F32, "bfloat16": BF16, "torch.bfloat16": BF16, "uint16": BF16,
          "torch.uint16": BF16, "<u2": BF16}


def _code(dtype: object) -> int:
    try:
        return _CODES[dtype]
    except KeyError:
        code = _NAMES.get(str(dtype))
        if code is None:
            raise _hip.Error(f"device arrays are float32 or bfloat16 (uint16 bits), not {dtype}") from None
        _CODES[dtype] = code
        return code


class DeviceArray:
    """(rows, values) in GPU memory, on a device (-1: the current one). dtype: ``float32``, or ``uint16`` for bf16 bits."""

    requires_grad = False

    def __init__(self, shape: tuple[int, int], dtype: object = np.float32, device: int = -1):
        self.dtype = np.dtype(dtype)
        _code(self.dtype)
        self.shape = (int(shape[0]), int(shape[1]))
        self._lib = _hip.lib()  # (close() may run when the module is gone)
        p, dev = ctypes.c_void_p(), ctypes.c_int(device)
        _hip.check(self._lib.artlite_device_alloc(ctypes.byref(dev), self.nbytes, ctypes.byref(p)))
        self._p, self.device = p, dev.value

    @classmethod
    def of(cls, a: np.ndarray, device: int = -1) -> "DeviceArray":
        """A host array's copy."""
        if a.ndim != 2:
            raise _hip.Error(f"DeviceArray: {a.shape}, not (rows, values)")
        d = cls(a.shape, a.dtype, device)
        d.copy_from(a)
        return d

    @property
    def nbytes(self) -> int:
        return self.shape[0] * self.shape[1] * self.dtype.itemsize

    def data_ptr(self) -> int:
        if self._p is None:
            raise _hip.Error("DeviceArray: closed")
        return self._p.value or 0

    def stride(self) -> tuple[int, int]:
        return self.shape[1], 1

    def copy_from(self, a: np.ndarray) -> None:
        a = np.ascontiguousarray(a)
        if a.shape != self.shape or a.dtype != self.dtype:
            raise _hip.Error(f"DeviceArray: {a.dtype} {a.shape} into {self.dtype} {self.shape}")
        _hip.check(_hip.lib().artlite_device_copy(self.device, self.data_ptr(), a.ctypes.data, a.nbytes, 0))

    def numpy(self) -> np.ndarray:
        """A host copy, behind everything queued on the device."""
        a = np.empty(self.shape, self.dtype)
        _hip.check(_hip.lib().artlite_device_copy(self.device, a.ctypes.data, self.data_ptr(), a.nbytes, 1))
        return a

    def close(self) -> None:
        if getattr(self, "_p", None) is not None:
            self._lib.artlite_device_free(self._p)
            self._p = None

    def __del__(self) -> None:
        self.close()


class Workspace:
    """Scratch memory of the operators' calls, of a fixed size, on a device (-1: the current one). Calls outside a stream
    capture order themselves on it; graphs that run beside each other, or beside calls, take one each. eager_only: calls
    under capture are refused."""

    def __init__(self, nbytes: int, device: int = -1, *, eager_only: bool = False):
        self._lib = _hip.lib()  # (close() may run when the module is gone)
        h = ctypes.c_void_p()
        _hip.check(self._lib.artlite_workspace_create(device, nbytes, int(eager_only), ctypes.byref(h)))
        self._h, self.nbytes = h, nbytes

    @property
    def handle(self) -> ctypes.c_void_p:
        if self._h is None:
            raise _hip.Error("Workspace: closed")
        return self._h

    def close(self) -> None:
        if getattr(self, "_h", None) is not None:
            self._lib.artlite_workspace_destroy(self._h)
            self._h = None

    def __del__(self) -> None:
        self.close()


_shared: dict[int, Workspace] = {}
_shared_lock = threading.Lock()


def shared_workspace(device: int, nbytes: int, stream: object) -> Workspace:
    """The workspace of a device's calls that are given none, grown as they need more (not while ``stream`` is captured: such
    a call is refused), by a quarter at least. The caller keeps it until its call has returned; one that is outgrown is freed
    with the last that does, behind its calls."""
    with _shared_lock:
        w = _shared.get(device)
        if w is None or w.nbytes < nbytes:
            capturing = ctypes.c_int(0)
            _hip.check(_hip.lib().artlite_stream_capturing(stream, ctypes.byref(capturing)))
            if capturing.value:
                raise _hip.Error("a captured call takes a workspace of its own")
            nbytes = max(nbytes, w.nbytes * 5 // 4 if w else 0)
            _shared.pop(device, None)
            w = None  # (freed before the new one is allocated)
            w = _shared[device] = Workspace(nbytes, device, eager_only=True)
        return w


def _records() -> bool:
    torch = sys.modules.get("torch")
    return torch is not None and torch.is_grad_enabled()


class View:
    """An argument as a call takes it: address, dtype code, rows, values a row, row stride in values; the stream that its
    interface names (none: nothing to wait for)."""

    __slots__ = ("at", "code", "rows", "cols", "row", "stream")

    def __init__(self, a: object, what: str, written: bool = False):
        self.stream = None
        if hasattr(a, "data_ptr"):
            if written and getattr(a, "requires_grad", False) and _records():
                raise _hip.Error(f"{what}: requires grad, and a call records no graph (torch.no_grad(), or a tensor without)")
            shape, strides, self.code = a.shape, a.stride(), _code(a.dtype)
            if len(shape) != 2:
                raise _hip.Error(f"{what}: {tuple(shape)}, not (rows, values)")
            self.at = a.data_ptr()
        elif hasattr(a, "__cuda_array_interface__"):
            d = a.__cuda_array_interface__
            shape, self.at, self.code = d["shape"], d["data"][0], _code(d["typestr"])
            if len(shape) != 2:
                raise _hip.Error(f"{what}: {tuple(shape)}, not (rows, values)")
            if written and d["data"][1]:
                raise _hip.Error(f"{what}: read-only")
            self.stream = d.get("stream")
            if self.stream == 0:
                raise _hip.Error(f"{what}: an interface whose stream is 0 (1: the null stream, 2: the per-thread one)")
            size = 4 if self.code == F32 else 2
            strides = [s / size for s in d["strides"]] if d.get("strides") else (shape[1], 1)
        else:
            raise _hip.Error(f"{what}: {type(a).__name__} is no array of device memory")
        self.rows, self.cols = shape
        self.row = int(strides[0])
        if self.row != strides[0]:
            raise _hip.Error(f"{what}: rows {strides[0]} values apart")
        if strides[1] != 1 and self.cols > 1:
            raise _hip.Error(f"{what}: a row's values are {strides[1]} apart")


def after(device: int, stream: int | None, views: Iterable[View]) -> None:
    """A call on ``stream`` comes after what the streams named by its arrays' interfaces (1: the null stream) have by now."""
    for s in {0 if v.stream == 1 else v.stream for v in views if v.stream is not None} - {stream or 0}:
        _hip.check(_hip.lib().artlite_stream_wait(device, stream, s))


def overlap(a: View, b: View) -> bool:
    """Whether two views have memory in common. (Views whose rows are different strides apart, or overlap themselves: whether the
    memory that they span meets.)"""
    size, other = 4 if a.code == F32 else 2, 4 if b.code == F32 else 2
    if not (a.rows and b.rows and a.at < b.at + ((b.rows - 1) * b.row + b.cols) * other
            and b.at < a.at + ((a.rows - 1) * a.row + a.cols) * size):
        return False
    na, nb = (1 if v.row == 0 else v.rows for v in (a, b))
    wa, wb = a.cols * size, b.cols * other
    s = a.row * size if nb == 1 else b.row * other
    if (na > 1 and nb > 1 and a.row * size != s) or s < max(wa, wb):
        return True
    # b's row j begins r bytes into a's row j + k
    k, r = divmod(b.at - a.at, s)

    def pair(k: int) -> bool:
        return max(0, -k) < min(nb, na - k)

    return (r < wa and pair(k)) or (r + wb > s and pair(k + 1))
