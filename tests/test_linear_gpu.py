"""``QLinear`` against 64-bit math in every format and on every path: few rows (bf16 1 to 256, fp32 1 to 128, more of a
small matrix: one, two and four blocks of 16), tall matrices, the large tiles past them (both sizes), widths of a single
block, of partial units and of partial 64 values, odd numbers of outputs, rows at any stride and address; bias, zeros,
infinities and NaN.

Tolerances (relative L2). A bf16 output is rounded once: half a step is 2^-8. Of few rows no weight is rounded and sums are
fp32: 2^-8 + 2^-14. Past that each weight is rounded to fp16 (half a step 2^-11; the errors of a sum's terms are independent,
so the sum's is 2^-11 of its size), or its scale's product, its offset and itself are (uniform codes 0 .. 15 with an offset of
7.5: 8.8, 7.5 and 4.6 times the scale in the mean square, each off by 2^-11 / sqrt(3) of itself: together 2.7 2^-11 / sqrt(3) =
1.6 2^-11 of the values): 2^-8 + 2^-10. fp32: a sum of n terms in fp32 is off by about sqrt(n) 2^-24 (n the groups
of 32 values and their MFMA steps, at most 2 * 90 * 3 here: 1.4e-6), the three bf16 planes by 2^-24, two fp16 planes by 2^-22
a factor: 4e-6."""

import numpy as np
import pytest

from artlite_amd import _hip
from artlite_amd.device import DeviceArray, Workspace
from artlite_amd.linear import QLinear
from oracle import dense

from .dense_helpers import Rows, check, encode, past_small, small, values

pytestmark = pytest.mark.gpu

FEW = {"bf16": 256, "f32": 128}
TOL = {("bf16", True): 2.0 ** -8 + 2.0 ** -14, ("bf16", False): 2.0 ** -8 + 2.0 ** -10, ("f32", True): 4e-6,
       ("f32", False): 4e-6}


def few(N: int, K: int, M: int, dtype: str) -> bool:
    return M <= FEW[dtype] or small(N, K, M, 1 if dtype == "bf16" else 3)


def widths(q: str) -> list[int]:
    return [256, 768] if q in ("Q4_K", "IQ4_XS") else [32, 96, 256, 416, 2880]


def make(q: str, N: int, K: int, seed: int, bias: bool = False) -> tuple[QLinear, np.ndarray, np.ndarray | None]:
    raw, w = dense.matrix(q, N, K, seed)
    b = np.random.default_rng(seed + 1).standard_normal(N).astype(np.float32) if bias else None
    lin = QLinear(q, N, K)
    lin.upload(raw, bias=b)
    return lin, w, b


def x_rows(M: int, K: int, dtype: str, seed: int) -> np.ndarray:
    return encode(np.random.default_rng(seed).standard_normal((M, K)), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q", dense.FORMATS)
def test_rows_and_widths(q: str, dtype: str) -> None:
    """Every number of rows on either side of the paths' borders, with every width of a few matrices."""
    for K in widths(q):
        for N in (1, 17, 100):
            lin, w, _ = make(q, N, K, 7 * N + K)
            past = [max(FEW[dtype] + 1, past_small(N, K, 1 if dtype == "bf16" else 3))] if N == 100 else []
            for M in (1, 4, 5, 8, 9, 16, 17, 33, 65, 128, 129, 256, 257, *past):
                x = x_rows(M, K, dtype, M + K)
                check(lin(x), values(x) @ w.T, TOL[dtype, few(N, K, M, dtype)], np.sqrt(values(x) ** 2 @ (w ** 2).T))
            lin.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize(("q", "N", "K"), [("Q4_0", 1531, 2880), ("Q4_K", 512, 2048), ("Q4_1", 272, 4128),
                                           ("IQ4_NL", 4100, 576), ("IQ4_XS", 96, 8192), ("Q4_1", 2080, 3104)])
def test_larger(q: str, N: int, K: int, dtype: str) -> None:
    """Units shared by every number of waves; tiles of the large products in several rows and columns."""
    lin, w, b = make(q, N, K, 5, bias=True)
    for M in (1, 5, 20, 40, 100, 300, 1400):
        x = x_rows(M, K, dtype, M)
        check(lin(x), values(x) @ w.T + b, TOL[dtype, few(N, K, M, dtype)])


def test_large_tiles() -> None:
    """More tiles of 256 x 256 than CUs, the last of each row and column partial."""
    lin, w, b = make("Q4_0", 4100, 288, 9, bias=True)
    x = x_rows(4111, 288, "bf16", 3)
    check(lin(x), values(x) @ w.T + b, TOL["bf16", False])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize(("q", "N", "K"), [("Q4_0", 131077, 1024), ("Q4_K", 33001, 4096), ("Q4_1", 131072, 992),
                                           ("IQ4_NL", 40003, 3616), ("IQ4_XS", 16387, 8192)])
def test_tall(q: str, N: int, K: int, dtype: str) -> None:
    """Matrices of so many rows that a wave reads several tiles or parts of them (the rows those of 1009, a prime, over and
    over: each of a tile's places has each of them); a bias; x and the output with rows apart; the same bits again."""
    raw, w = dense.matrix(q, 1009, K, 3)
    raw = np.tile(raw.reshape(1009, -1), (-(-N // 1009), 1))[:N]
    b = np.random.default_rng(1).standard_normal(N).astype(np.float32)
    lin = QLinear(q, N, K)
    for bias in (None, b):
        lin.upload(raw, bias=bias)
        # (one large matrix: past 128 rows of bf16 by way of 16-bit weights)
        for M in (1, 4, 5, 11, 16) + ((128, 130) if N < 20000 else ()):
            data = x_rows(M, K, dtype, M)
            x, y = Rows(M, K, dtype, at=3, stride=K + 5, data=data), Rows(M, N, dtype, at=1, stride=N + 3)
            lin(x, y)
            got = y.numpy()
            check(got, np.tile(values(data) @ w.T, (1, -(-N // 1009)))[:, :N] + (0 if bias is None else b),
                  TOL[dtype, M <= 128])
            lin(x, y)
            assert np.array_equal(got, y.numpy())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize(("at", "pad", "out_at", "out_pad"), [(0, 0, 0, 0), (8, 8, 1, 3), (1, 0, 0, 4), (3, 5, 2, 2),
                                                              (8, 4, 4, 0), (0, 1, 0, 1)])
def test_strides(at: int, pad: int, out_at: int, out_pad: int, dtype: str) -> None:
    """Rows at any address and stride; what lies between and behind the output's rows stays."""
    N, K = 100, 160
    lin, w, _ = make("IQ4_NL", N, K, 2)
    for M in (1, 3, 16, 70, 300, 37500):
        data = x_rows(M, K, dtype, M)
        x = Rows(M, K, dtype, at=at, stride=K + pad, data=data)
        y = Rows(M, N, dtype, at=out_at, stride=N + out_pad)
        assert lin(x, y) is y
        check(y.numpy(), values(data) @ w.T, TOL[dtype, few(N, K, M, dtype)])


def test_one_row_for_all() -> None:
    """A row stride of 0: every output row is the one input row's."""
    lin, w, _ = make("Q4_0", 40, 256, 2)
    data = x_rows(1, 256, "bf16", 1)
    for M in (3, 80, 87400):
        x = Rows(1, 256, "bf16", data=data)
        x.shape, x.row = (M, 256), 0
        y = Rows(M, 40, "bf16")
        lin(x, y)
        check(y.numpy(), np.repeat(values(data) @ w.T, M, 0), TOL["bf16", few(40, 256, M, "bf16")])


def test_widest() -> None:
    """The most values a row may have, on every path (many rows: one for all of them)."""
    N, K = 20, 1 << 20
    lin, w, _ = make("Q4_0", N, K, 6)
    data = x_rows(1, K, "bf16", 1)
    want = values(data) @ w.T
    terms = np.sqrt(values(data) ** 2 @ (w ** 2).T)
    for M in (1, 7, 40, 100, 256, 257, 600):
        x = Rows(1, K, "bf16", data=data)
        x.shape, x.row = (M, K), 0
        y = Rows(M, N, "bf16")
        lin(x, y)
        check(y.numpy(), np.repeat(want, M, 0), TOL["bf16", few(N, K, M, "bf16")], np.repeat(terms, M, 0))
    with pytest.raises(_hip.Error, match="rows of 1048608 values"):
        QLinear("Q4_0", N, K + 32)


@pytest.mark.parametrize("M", [4, 90, 1300])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_values_out_of_the_ordinary(dtype: str, M: int) -> None:
    """Rows of zeros, of the type's smallest and largest sizes, with infinities and NaN: each row is its own, the others are
    unmoved."""
    N, K = 1600, 512
    lin, w, _ = make("Q4_K", N, K, 4)
    a = np.random.default_rng(1).standard_normal((M, K))
    a[0] = 0.0
    a[1] *= 1e-30
    a[2] *= 1e30
    base = encode(a, dtype)
    y0 = lin(base)
    check(y0[3:], values(base)[3:] @ w.T, TOL[dtype, few(N, K, M, dtype)])
    assert not values(y0)[0].any()
    for r in (1, 2):
        check(y0[r:r + 1], values(base)[r:r + 1] @ w.T, TOL[dtype, few(N, K, M, dtype)])
    a[3, 5] = np.nan
    bad = encode(a, dtype)
    bad[2, 7] = encode(np.array([np.inf]), dtype)[0]
    y1 = lin(bad)
    assert np.isnan(values(y1)[3]).all() and not np.isfinite(values(y1)[2]).any()
    assert np.array_equal(y1[:2], y0[:2]) and np.array_equal(y1[4:], y0[4:])


def test_zero_blocks_and_large_scales() -> None:
    """A matrix of zeros, and one whose scales are the largest fp16 ones, on both paths."""
    for M in (3, 70, 131100):
        x = x_rows(M, 64, "bf16", M)
        lin = QLinear("Q4_0", 20, 64)
        lin.upload(np.zeros((20, 36), np.uint8))
        assert not lin(x).any()
        raw, _ = dense.matrix("Q4_0", 20, 64, 1)
        raw = raw.reshape(20, 2, 18)
        raw[..., :2] = np.array([65504.0], np.float16).view(np.uint8)
        lin.upload(raw)
        w = dense.gguf_ref.dequantize("Q4_0", raw.reshape(20, 36), 64).astype(np.float64)
        check(lin(x), values(x) @ w.T, TOL["bf16", few(20, 64, M, "bf16")])


@pytest.mark.parametrize("q", ["Q4_0", "Q4_1", "IQ4_NL"])
def test_scales_beyond_their_values(q: str) -> None:
    """Groups whose values are zeros, or small differences, of large scales and offsets."""
    N, K, per = 1600, 512, {"Q4_0": 18, "Q4_1": 20, "IQ4_NL": 18}[q]
    raw, _ = dense.matrix(q, N, K, 3)
    raw = raw.reshape(N, K // 32, per).copy()
    big = np.array([100.0], np.float16).view(np.uint8)
    for r, at in ((5, 3), (800, 0), (1599, 15)):
        if q == "Q4_0":  # (c - 8 = 0)
            raw[r, at, :2], raw[r, at, 2:] = np.array([65504.0], np.float16).view(np.uint8), 0x88
        elif q == "Q4_1":  # (15 d + m = 0, and 1 for one value)
            raw[r, at, :2], raw[r, at, 2:4], raw[r, at, 4:] = big, np.array([-1500.0], np.float16).view(np.uint8), 0xFF
        else:
            raw[r, at, :2] = big
    lin = QLinear(q, N, K)
    lin.upload(raw.reshape(N, -1))
    w = dense.gguf_ref.dequantize(q, raw.reshape(N, -1), K).astype(np.float64)
    for M in (3, 90, 1300):
        x = x_rows(M, K, "bf16", M)
        check(lin(x), values(x) @ w.T, TOL["bf16", few(N, K, M, "bf16")], np.sqrt(values(x) ** 2 @ (w ** 2).T))


def test_no_rows_and_repeats() -> None:
    """0 rows write nothing; the same call twice gives the same bits, on every path."""
    lin, _, _ = make("IQ4_XS", 100, 512, 3)
    assert lin(np.empty((0, 512), np.uint16)).shape == (0, 100)
    for M in (1, 20, 65, 128, 129, 300, 18800):
        for dtype in ("bf16", "f32"):
            x = x_rows(M, 512, dtype, M)
            assert np.array_equal(lin(x), lin(x))


def test_refusals() -> None:
    lin, _, _ = make("Q4_0", 64, 64, 3)
    x, y = DeviceArray((280, 64), np.uint16), DeviceArray((280, 64), np.uint16)
    with pytest.raises(_hip.Error, match="out overlaps x"):
        lin(x, x)
    with pytest.raises(_hip.Error, match="for 64 rows of 64 values"):
        lin(x, DeviceArray((280, 64), np.float32))
    with pytest.raises(_hip.Error, match="for 64 rows of 64 values"):
        lin(x, DeviceArray((279, 64), np.uint16))
    with pytest.raises(_hip.Error, match="is no array"):
        lin(x)
    with pytest.raises(_hip.Error, match="a workspace of 1024 bytes, not"):
        make("Q4_0", 4096, 1024, 3)[0](DeviceArray((300, 1024), np.uint16), DeviceArray((300, 4096), np.uint16),
                                       work=Workspace(1024))

    class Host:  # (an address that is the host's)
        shape, dtype = (280, 64), np.dtype(np.uint16)
        mem = np.zeros((280, 64), np.uint16)

        def stride(self) -> tuple[int, int]:
            return 64, 1

        def data_ptr(self) -> int:
            return self.mem.ctypes.data

    with pytest.raises(_hip.Error, match="x: not device memory"):
        lin(Host(), y)
    x.close()
    with pytest.raises(_hip.Error, match="closed"):
        lin(x, y)
    lin.close()
    with pytest.raises(_hip.Error, match="closed"):
        lin(np.zeros((1, 64), np.uint16))
    empty = QLinear("Q4_0", 64, 64)
    with pytest.raises(_hip.Error, match="not uploaded"):
        empty(np.zeros((1, 64), np.uint16))
