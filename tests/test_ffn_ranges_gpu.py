"""``GatedFFN`` on rows of very different sizes: zeros, the smallest values, infinities and outliers, in x and in dy apart.

Tolerances are test_ffn_gpu's: each rounding enters relative to the values that it is a rounding of, whatever their size."""

import numpy as np
import pytest

from oracle import dense

from .dense_helpers import check, encode, values
from .test_ffn_gpu import BACKWARD, FORWARD, GRADS, grads, make, rows

pytestmark = pytest.mark.gpu

H, F = 96, 160
# rows on every path: the few rows' launches, tiles that make gate and up from their blocks (bf16), the large tiles (fp32)
ROWS = (1, 5, 70, 193, 1500)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_rows_of_zeros_in_x(act: str, dtype: str) -> None:
    """A row of zeros in x beside one of dy that is not (a padded token): its dx is 0, it adds nothing to the others."""
    f, w = make(H, F, "Q4_0", "Q4_1", act)
    for n in ROWS:
        x, dy = rows(n, H, dtype, n, 3.0), rows(n, H, dtype, n + 1)
        x[::3] = 0
        want = dense.ffn_grad(act, values(x), values(dy), *w)
        got = grads(f, x, dy)
        assert not values(got["dx"][::3]).any(), n
        for k in GRADS:
            check(got[k], want[k], BACKWARD[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_small_rows_backward(dtype: str) -> None:
    """Rows of x down to the smallest normal values, with gradients that bring dx back to where it has all its bits. (Few rows
    of fp32 x go as three planes of bf16, whose smallest step is 2^-133: half of that relative to the row on top.)"""
    f, w = make(H, F, "Q4_0", "Q4_1")
    for n in ROWS:
        size = np.resize([1e-37, 1.0, 1e-30, 1e-20, 3e-36], n)[:, None]
        x = encode(size * np.random.default_rng(n).standard_normal((n, H)), dtype)
        dy = encode(np.random.default_rng(n + 1).standard_normal((n, H)) * np.minimum(1e8, 1 / np.sqrt(size)), dtype)
        want = dense.ffn_grad("silu", values(x), values(dy), *w)
        got = grads(f, x, dy, ("dx",))
        for r in range(min(n, 40)):
            planes = 2.0 ** -134 / size[r, 0] if dtype == "f32" else 0.0
            check(got["dx"][r:r + 1], want["dx"][r:r + 1], 1.5 * BACKWARD[dtype] + planes)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_small_rows_forward(dtype: str) -> None:
    """Rows whose h has no value but 0 in fp32, and rows that are small."""
    f, w = make(H, F, "Q4_0", "Q4_1")
    for n in (*ROWS, 18000):
        size = np.resize([1e-37, 1.0, 1e-15, 3e-36, 0.0, 1e-33], n)[:, None]
        x = encode(size * np.random.default_rng(n).standard_normal((n, H)), dtype)
        got, want = values(f(x)), dense.ffn("silu", values(x), *w)
        assert np.isfinite(got).all(), n
        nothing = size[:, 0] < 1e-30
        assert not got[nothing].any(), n
        for r in range(min(n, 40)):
            if not nothing[r]:
                check(got[r:r + 1], want[r:r + 1], 1.5 * FORWARD[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinite_gradients(dtype: str) -> None:
    """An infinite value of dy reaches its row's dx, the gate's and up's gradients (sums over that row too) and its own row
    of ddown alone."""
    f, w = make(H, F, "Q4_0", "Q4_1")
    for n in ROWS[1:]:
        x, dy = rows(n, H, dtype, n, 3.0), rows(n, H, dtype, n + 1)
        clean = grads(f, x, dy, ("dx",))["dx"]
        want = dense.ffn_grad("silu", values(x), values(dy), *w)["ddown"]
        dy[1, 3] = encode(np.array([np.inf]), dtype)[0]
        got = grads(f, x, dy)
        assert not np.isfinite(values(got["dx"])[1]).any() and not np.isfinite(values(got["ddown"])[3]).any()
        assert not np.isfinite(values(got["dgate"])).any() and not np.isfinite(values(got["dup"])).any()
        assert np.array_equal(np.delete(got["dx"], 1, 0), np.delete(clean, 1, 0))
        check(np.delete(got["ddown"], 3, 0), np.delete(want, 3, 0), BACKWARD[dtype])
