"""``QLinear`` over matrices with scales that are no numbers. Tolerances are test_linear_gpu's."""

import numpy as np
import pytest

from artlite_amd.linear import QLinear
from oracle import dense

from .dense_helpers import check, values
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
