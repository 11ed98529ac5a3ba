"""``QLinear`` over matrices with scales that are no numbers. Tolerances are test_linear_gpu's."""

import numpy as np
import pytest

from artlite_amd.device import DeviceArray
from artlite_amd.linear import QLinear
from oracle import dense

from .dense_helpers import check, encode, values
from .test_linear_gpu import TOL, few, x_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize(("q", "at"), [("Q4_0", 0), ("Q4_1", 0), ("Q4_1", 2), ("Q4_K", 0), ("IQ4_NL", 0), ("IQ4_XS", 0)])
def test_infinite_scales(q: str, at: int, dtype: str) -> None:
    """A block whose scale (Q4_1: or offset) is infinite reaches its own matrix row's outputs alone."""
    N, K = 1600, 512
    raw, w = dense.matrix(q, N, K, 3)
    raw = raw.reshape(N, -1).copy()
    raw[7, at:at + 2] = np.array([np.inf], np.float16).view(np.uint8)
    lin = QLinear(q, N, K)
    lin.upload(raw)
    for M in (3, 90, 300, 1300):
        x = x_rows(M, K, dtype, M)
        got, want = lin(x), values(x) @ w.T
        assert not np.isfinite(values(got)[:, 7]).any()
        check(np.delete(got, 7, 1), np.delete(want, 7, 1), TOL[dtype, few(N, K, M, dtype)])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_columns_of_one_buffer(dtype: str) -> None:
    """x and the output as columns of one device array: what is beside them stays."""
    K, N = 256, 100
    raw, w = dense.matrix("Q4_K", N, K, 3)
    lin = QLinear("Q4_K", N, K)
    lin.upload(raw)
    for M in (1, 20, 300, 20000):
        whole = encode(np.random.default_rng(M).standard_normal((M, 420)), dtype)
        dev = DeviceArray.of(whole)

        class Columns:
            def __init__(self, first: int, cols: int):
                self.first, self.shape, self.dtype = first, (M, cols), dev.dtype

            def data_ptr(self) -> int:
                return dev.data_ptr() + self.first * dev.dtype.itemsize

            def stride(self) -> tuple[int, int]:
                return 420, 1

        lin(Columns(3, K), Columns(3 + K, N))
        got = dev.numpy()
        check(got[:, 3 + K:3 + K + N], values(whole[:, 3:3 + K]) @ w.T, TOL[dtype, few(N, K, M, dtype)])
        assert np.array_equal(np.delete(got, np.s_[3 + K:3 + K + N], 1), np.delete(whole, np.s_[3 + K:3 + K + N], 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q", dense.FORMATS)
def test_smallest_rows(q: str, dtype: str) -> None:
    """Rows of x about the smallest normal values beside ordinary ones, each row as exact as its own values are. On top of the
    tolerance: a bf16 output's smallest half step (2^-134; fp32's 2^-150 is nothing beside the next), and of fp32 rows half the
    smallest step of the planes that few of them go as (2^-134 a value; each of the output's K terms has one, times a weight)."""
    N, K = 400, 512
    raw, w = dense.matrix(q, N, K, 3)
    lin = QLinear(q, N, K)
    lin.upload(raw)
    for M in (3, 16, 90, 300, 1300):
        size = np.resize([1e-37, 1.0, 3e-36, 1e-33], M)[:, None]
        x = encode(size * np.random.default_rng(M).standard_normal((M, K)), dtype)
        got, want = lin(x), values(x) @ w.T
        step = 2.0 ** -134 * (1.0 if dtype == "bf16" else np.sqrt((w ** 2).sum(1)).max())
        for r in range(min(M, 24)):
            top = step * np.sqrt(N) / np.linalg.norm(want[r])
            check(got[r:r + 1], want[r:r + 1], 1.5 * TOL[dtype, few(N, K, M, dtype)] + top,
                  np.sqrt(values(x[r:r + 1]) ** 2 @ (w ** 2).T))
