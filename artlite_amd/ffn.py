"""The gated feed-forward block of a model's dense layers over GGUF blocks in 4-bit formats, forward and backward
(``artlite_ffn_*``): ``y = (act(x gate^T) * (x up^T)) down^T``. Beside ``moe.layer.MoELayer``, for the blocks that have no
experts (an MoE model's leading dense blocks)."""

import ctypes
import itertools

import numpy as np

from . import _hip
from .device import DeviceArray, View, Workspace, after, overlap, shared_workspace
from .gguf_model import GGUFFile
from .linear import FORMATS, Matrix

ACTS = {"silu": 0, "gelu_tanh": 1}


class GatedFFN:
    """A block's three matrices in HBM: ``ffn_gate``, ``ffn_up`` (ffn rows of hidden values, one format) and ``ffn_down``
    (hidden rows of ffn values). Inputs and outputs are (n, hidden), all bf16 or all fp32, any n."""

    def __init__(self, *, hidden: int, ffn: int, gate_type: str, down_type: str, act: str = "silu"):
        if act not in ACTS:
            raise _hip.Error(f"ffn: activation {act!r}, not one of {', '.join(ACTS)}")
        self.hidden, self.ffn, self.act = hidden, ffn, act
        self._m = {"ffn_gate": Matrix(gate_type, ffn, hidden), "ffn_up": Matrix(gate_type, ffn, hidden),
                   "ffn_down": Matrix(down_type, hidden, ffn)}
        self._d = _hip.Ffn(*(m.handle.value for m in self._m.values()), ACTS[act])

    @classmethod
    def from_gguf(cls, gguf: GGUFFile, block: int, *, act: str = "silu") -> "GatedFFN":
        """Block ``block``'s dense FFN: its ``blk.{block}.ffn_gate`` / ``ffn_up`` / ``ffn_down``."""
        t = {}
        for name in ("ffn_gate", "ffn_up", "ffn_down"):
            full = f"blk.{block}.{name}.weight"
            if full not in gguf:
                raise ValueError(f"{gguf.path}: block {block} has no dense FFN ({full} missing)")
            t[name] = gguf.tensor(full)
            if t[name].qtype not in FORMATS:
                raise ValueError(f"{gguf.path}: {full} is {t[name].qtype}, not one of {', '.join(FORMATS)}")
        g, u, d = t.values()
        if (g.rows, g.cols, g.qtype) != (u.rows, u.cols, u.qtype) or (d.rows, d.cols) != (g.cols, g.rows):
            raise ValueError(f"{gguf.path}: block {block} has {g.rows} x {g.cols} {g.qtype}, {u.rows} x {u.cols} {u.qtype}, "
                             f"{d.rows} x {d.cols}")
        f = cls(hidden=g.cols, ffn=g.rows, gate_type=g.qtype, down_type=d.qtype, act=act)
        for name, q in t.items():
            f.upload(name, q.raw)
        return f

    def upload(self, name: str, raw: np.ndarray) -> None:
        """A matrix's rows as the file holds them."""
        if name not in self._m:
            raise _hip.Error(f"ffn: {name!r}, not one of {', '.join(self._m)}")
        self._m[name].upload(raw)

    def close(self) -> None:
        for m in self._m.values():
            m.close()

    def workspace_bytes(self, n: int, dtype: str = "bf16", *, backward: bool = False, weights: bool = False) -> int:
        """What a call of n rows needs: forward, backward, or backward with the weights' gradients. (Not always less for fewer
        rows.)"""
        return self._need({"f32": 0, "bf16": 1}[dtype], n, 2 if weights else int(backward))

    def _need(self, code: int, n: int, backward: int) -> int:
        z = ctypes.c_size_t(0)
        _hip.check(_hip.lib().artlite_ffn_workspace(ctypes.byref(self._open()), code, n, backward, ctypes.byref(z)))
        return z.value

    def _open(self) -> _hip.Ffn:
        for m in self._m.values():
            m.handle  # (raises when closed)
        return self._d

    def _work(self, work: Workspace | None, v: dict[str, View], backward: int, stream: object) -> Workspace | None:
        """The call's workspace (to be kept until it has returned), and the call ordered behind its arrays' streams."""
        code, n = v["x"].code, v["x"].rows
        for w in v.values():
            if w.stream is not None:
                after(self._m["ffn_gate"].device, stream, v.values())
                break
        if work is not None or not n:
            return work
        return shared_workspace(self._m["ffn_gate"].device, self._need(code, n, backward), stream)

    def _views(self, what: str, x: object, shapes: dict[str, tuple[object, int | None, int]]) -> dict[str, View]:
        """The views of x and of the arrays (array, rows, or none: x's, cols) that are given: all of one dtype, none of the
        written ones (all but x and dy) over another."""
        w = View(x, f"{what}: x")
        v, n, code = {"x": w}, w.rows, w.code
        if w.cols != self.hidden:
            raise _hip.Error(f"{what}: x is ({n}, {w.cols}), not of {self.hidden} columns")
        for k, (a, rows, cols) in shapes.items():
            if a is None:
                continue
            w = v[k] = View(a, f"{what}: {k}", k != "dy")
            rows = n if rows is None else rows
            if w.rows != rows or w.cols != cols or w.code != code:
                raise _hip.Error(f"{what}: {k} is ({w.rows}, {w.cols}) of dtype {w.code}, x of {code}; expected ({rows}, {cols})")
        names = list(v)
        for i, a in enumerate(names):
            for b in names[i + 1:]:
                if not (a in ("x", "dy") and b in ("x", "dy")) and overlap(v[a], v[b]):
                    raise _hip.Error(f"{what}: {b} overlaps {a}")
        return v

    def __call__(self, x: object, out: object = None, *, stream: int = 0, work: Workspace | None = None) -> object:
        """x (n, hidden) -> out (n, hidden). Device arrays (``device``): enqueued on ``stream`` (a hipStream_t's address; 0:
        the null stream), ``out`` given by the caller, ``work`` its workspace (none: one that the device's calls
        share, which a captured call may not use). A numpy x (fp32, or
        uint16 bf16 bits): the result as a numpy array."""
        if isinstance(x, np.ndarray):
            if out is not None:
                raise _hip.Error("ffn: out goes with device arrays")
            d = DeviceArray.of(x, self._m["ffn_gate"].device)
            return self(d, DeviceArray(d.shape, x.dtype, d.device), stream=stream, work=work).numpy()
        v = self._views("ffn", x, {"out": (out, None, self.hidden)})
        if "out" not in v:
            raise _hip.Error("ffn: device arrays need out")
        a, y = v["x"], v["out"]
        n = a.rows
        d = ctypes.byref(self._open())
        work = self._work(work, v, 0, stream)
        _hip.check(_hip.lib().artlite_ffn_forward(d, a.at, a.code, n, a.row, y.at, y.row,
                                                  work.handle if work is not None else None, stream))
        return out

    def backward(self, x: object, dy: object, *, dx: object = None, dgate: object = None, dup: object = None,
                 ddown: object = None, stream: int = 0, work: Workspace | None = None) -> None:
        """From x and the output's gradient dy (n, hidden): the gradients that are asked for, into dx (n, hidden), dgate, dup
        (ffn, hidden) and ddown (hidden, ffn; rows without gaps): those of the blocks' values, zeros where n is 0. Device
        arrays, or numpy arrays throughout (written in place)."""
        H, F = self.hidden, self.ffn
        outs = {"dx": (dx, None, H), "dgate": (dgate, F, H), "dup": (dup, F, H), "ddown": (ddown, H, F)}
        if isinstance(x, np.ndarray):
            host = {k: a for k, (a, _, _) in outs.items() if a is not None}
            for k, a in {"dy": dy, **host}.items():
                if not isinstance(a, np.ndarray) or a.ndim != 2:
                    raise _hip.Error(f"ffn backward: {k} is no host array of (rows, values), as x is")
            for i, j in itertools.combinations(host, 2):
                if np.shares_memory(host[i], host[j]):
                    raise _hip.Error(f"ffn backward: {j} overlaps {i}")
            on = self._m["ffn_gate"].device
            dev = {k: DeviceArray(a.shape, a.dtype, on) for k, a in host.items()}
            self.backward(DeviceArray.of(x, on), DeviceArray.of(dy, on), **dev, stream=stream, work=work)
            for k, a in host.items():
                a[...] = dev[k].numpy()
            return
        v = self._views("ffn backward", x, {"dy": (dy, None, H), **outs})
        for k in ("dgate", "dup", "ddown"):
            if k in v and v[k].row != v[k].cols:
                raise _hip.Error(f"ffn backward: {k}'s rows are {v[k].row} values apart")
        if "dy" not in v:
            raise _hip.Error("ffn backward: no dy")
        a, d, o = v["x"], v["dy"], v.get("dx")
        n = a.rows
        weights = any(k in v for k in ("dgate", "dup", "ddown"))
        at = [v[k].at if k in v else None for k in ("dgate", "dup", "ddown")]
        f = ctypes.byref(self._open())
        work = self._work(work, v, 2 if weights else 1, stream)
        _hip.check(_hip.lib().artlite_ffn_backward(
            f, a.at, a.row, d.at, d.row, a.code, n, o.at if o else None, o.row if o else 0, *at,
            work.handle if work is not None else None, stream))
