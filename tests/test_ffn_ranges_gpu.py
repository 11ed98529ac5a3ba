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


def terms(x: np.ndarray, dy: np.ndarray, w: list[np.ndarray], tol: float) -> dict[str, np.ndarray]:
    """The 2-norm of each gradient's terms (``dense_helpers.check``), silu's. The terms are made of sums themselves: g, u and dh
    are off by a share t of the 2-norms G, U, D of their own terms, however small they come out, which moves dg = dh u act'(g)
    by t (D |u act'| + |dh| U |act'| + |dh u act''| G) to first order (|act''| <= 1/2), du = dh act(g) by t (D |act| +
    |dh act'| G) and h = act(g) u by t (|act'| G |u| + |act| U). These stand in the place of the terms' own sizes, which they
    are never below (D >= |dh| and so on, but for few terms that add up: the larger of the two).

    And dg, du and h go as fp16 (fp32 calls: two of them), whose smallest step is 2^-24 with a row's bound at 2^15: each is off
    by up to 2^-40 of its row's bound, a power of two no less than |x| |dy| max |down| sqrt(H) 2 (the larger of the rows of gate
    and up in the 2-norm) and |x|^2 (gate's) (up's), each factor a power of two itself. Divided by tol that counts as terms."""
    g, u, dh = x @ w[0].T, x @ w[1].T, dy @ w[2]
    a, da = dense.act("silu", g)
    G, U, D = (np.sqrt(v ** 2 @ m ** 2) for v, m in ((x, w[0].T), (x, w[1].T), (dy, w[2])))
    a, da, u, dh = np.abs(a), np.abs(da), np.abs(u), np.abs(dh)
    dg = np.maximum(dh * u * da, D * u * da + dh * U * da + 0.5 * dh * u * G)
    du = np.maximum(dh * a, D * a + dh * da * G)
    h = np.maximum(a * u, da * G * u + a * U)

    def above(v: np.ndarray) -> np.ndarray:
        return 2.0 ** np.where(v > 0, np.frexp(v)[1], -200.0)

    nx, ny = (above(1.01 * np.linalg.norm(v, axis=1, keepdims=True)) for v in (x, dy))
    ng, nu = (above(1.001 * np.linalg.norm(m, axis=1).max()) for m in w[:2])
    grad = 2.0 ** -40 / tol * nx * ny * above(np.abs(w[2]).max()) * 2.0 ** np.ceil(0.5 * np.log2(H)) * 2 * max(ng, nu)
    dg, du, h = dg + grad, du + grad, h + 2.0 ** -40 / tol * nx ** 2 * ng * nu
    return {"dgate": np.sqrt((dg ** 2).T @ x ** 2), "dup": np.sqrt((du ** 2).T @ x ** 2),
            "ddown": np.sqrt((dy ** 2).T @ h ** 2)}


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
        got = grads(f, x, dy)
        for r in range(min(n, 40)):
            planes = 2.0 ** -134 / size[r, 0] if dtype == "f32" else 0.0
            check(got["dx"][r:r + 1], want["dx"][r:r + 1], 1.5 * BACKWARD[dtype] + planes)
        if n > 1:
            for k in GRADS:
                check(got[k], want[k], BACKWARD[dtype])


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


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_rows_without_gradients(dtype: str) -> None:
    """Rows of x far larger than the others with no gradient or next to none (a masked first token): the weights' gradients
    are the others'."""
    f, w = make(H, F, "Q4_0", "Q4_1")
    for n in ROWS[1:]:
        for large in (16.0, 4096.0, 2.0 ** 40):
            for little in (0.0, 2.0 ** -100):
                x, dy = (np.random.default_rng(s).standard_normal((n, H)) for s in (n, n + 1))
                x[0] *= large
                dy[0] *= little
                x, dy = encode(x, dtype), encode(dy, dtype)
                want, size = dense.ffn_grad("silu", values(x), values(dy), *w), terms(values(x), values(dy), w, BACKWARD[dtype])
                for k, g in grads(f, x, dy, ("dgate", "dup", "ddown")).items():
                    check(g, want[k], BACKWARD[dtype], size[k])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradients_of_many_sizes(dtype: str) -> None:
    """Rows of x over six and of dy over twelve decades, and one value of dy of 2^60: each row of a weight's gradient is as
    exact as its own terms are large."""
    f, w = make(H, F, "Q4_0", "Q4_1")
    for n in ROWS[1:]:
        rng = np.random.default_rng(n)
        x = encode(10.0 ** rng.uniform(-6, 0.5, (n, 1)) * rng.standard_normal((n, H)), dtype)
        dy = 10.0 ** rng.uniform(-6, 6, (n, 1)) * rng.standard_normal((n, H))
        for spike in (0.0, 2.0 ** 60):
            if spike:
                dy[2] = 0.0
                dy[2, 5] = spike
            d = encode(dy, dtype)
            want, size = dense.ffn_grad("silu", values(x), values(d), *w), terms(values(x), values(d), w, BACKWARD[dtype])
            for k, g in grads(f, x, d, ("dgate", "dup", "ddown")).items():
                for r in range(g.shape[0]):
                    check(g[r:r + 1], want[k][r:r + 1], 1.5 * BACKWARD[dtype], size[k][r:r + 1])
