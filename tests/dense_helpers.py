"""Arrays for the dense operators' tests: rows inside a larger device array, their values and tolerances."""

import numpy as np

from artlite_amd.device import DeviceArray
from oracle.tensors import bf16_bits, from_bf16_bits

DTYPE = {"bf16": np.uint16, "f32": np.float32}


def small(rows: int, cols: int, M: int, planes: int, gated: bool = False) -> bool:
    """Whether a product's blocks of 16 rows are workgroups of their own (and stay with the few rows' path)."""
    units = -(-rows // 16) * -(-cols // 256) * (2 if gated else 1)
    return M <= 16 or units * -(-M // 16) <= 16384 // (2 if planes > 1 else 1)


def past_small(rows: int, cols: int, planes: int, gated: bool = False) -> int:
    """The first number of rows that is not."""
    units = -(-rows // 16) * -(-cols // 256) * (2 if gated else 1)
    return 16 * max(1, 16384 // (2 if planes > 1 else 1) // units) + 1


def values(a: np.ndarray) -> np.ndarray:
    """A host array's values in 64 bits."""
    return (from_bf16_bits(a) if a.dtype == np.uint16 else a).astype(np.float64)


def encode(a: np.ndarray, dtype: str) -> np.ndarray:
    return bf16_bits(a.astype(np.float32)) if dtype == "bf16" else a.astype(np.float32)


class Rows:
    """(rows, cols) of a device array of its own, the first value ``at`` values into it and the rows ``stride`` apart; what
    surrounds them holds a pattern that ``guarded`` looks for afterwards."""

    def __init__(self, rows: int, cols: int, dtype: str, *, at: int = 0, stride: int = 0, data: np.ndarray | None = None):
        self.shape, self.at, self.row = (rows, cols), at, stride or cols
        self.dtype = np.dtype(DTYPE[dtype])
        n = at + max(rows - 1, 0) * self.row + cols + 37
        self.flat = (np.arange(n) % 251 + 3000).astype(self.dtype)
        if data is not None:
            self._rows(self.flat)[...] = data
        self.dev = DeviceArray((1, n), self.dtype)
        self.dev.copy_from(self.flat[None])

    def _rows(self, flat: np.ndarray) -> np.ndarray:
        return np.lib.stride_tricks.as_strided(flat[self.at:], self.shape, (self.row * flat.itemsize, flat.itemsize))

    def data_ptr(self) -> int:
        return self.dev.data_ptr() + self.at * self.dtype.itemsize

    def stride(self) -> tuple[int, int]:
        return self.row, 1

    def numpy(self) -> np.ndarray:
        """The rows; what surrounds them is as it was."""
        got = self.dev.numpy()[0]
        inside = np.zeros(got.shape, bool)
        self._rows(inside)[...] = True
        assert np.array_equal(got[~inside], self.flat[~inside]), "written past the rows"
        return self._rows(got).copy()


def check(got: np.ndarray, want: np.ndarray, tol: float, terms: np.ndarray | None = None) -> None:
    """Within tol relative L2, and no value further off than 8 tol of the output's size (or its own).

    terms: the 2-norm of each output's terms, sqrt(sum_k (w x)^2). Each term (or partial sum) carries its own rounding of at
    most a share t of it, so an output is off by about t times that norm, however small the terms' sum itself comes out: the
    size of a set of outputs is that of their terms where these have cancelled. (Of many outputs with random signs the two are
    alike, since E[(sum_k w x)^2] = sum_k (w x)^2; of one or two they need not be: one output of 416 values, -0.0006 of terms
    with a norm of 0.0196 by their own size, is 32 times smaller than them.)"""
    g = values(got)
    assert g.shape == want.shape and np.isfinite(g).all()
    if not want.size:
        return
    d, norm = g - want, np.linalg.norm(want)
    if terms is not None:
        norm = max(norm, np.linalg.norm(terms))
    assert np.linalg.norm(d) <= tol * norm, (np.linalg.norm(d) / norm, tol)
    size = np.maximum(np.abs(want), norm / np.sqrt(want.size))
    assert (np.abs(d) <= 8 * tol * size).all(), float((np.abs(d) / size).max())
