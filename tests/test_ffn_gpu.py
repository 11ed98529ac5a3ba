"""``GatedFFN`` forward and backward against 64-bit math: few rows and the large tiles, formats, activations and widths of
partial units, strides, rows of nothing; its gradients against the formula's and against differences; a run of it between two
``QLinear``.

Tolerances (relative L2). bf16 outputs are rounded once (half a step 2^-8). Inside, each of the roundings to fp16 (weights, h;
backward also dg, du: half a step 2^-11 = an eighth of that) enters the output with a factor of about 1 and independently of
the others: at most 5 forward, 8 backward (gate and up weights in g, u and again in dx, down's, dg, du), so 2^-8 + 5 2^-11
and 2^-8 + 8 2^-11. fp32: fp32 sums of up to 3 (16384 / 32) steps (sqrt(n) 2^-24 = 2.4e-6 a product, two in a chain
forward, three backward), planes to 2^-22 a factor: 8e-6 and 1.2e-5."""

import numpy as np
import pytest

from artlite_amd import _hip
from artlite_amd.device import DeviceArray, Workspace
from artlite_amd.ffn import GatedFFN
from artlite_amd.gguf_model import TYPE_ID, GGUFFile
from artlite_amd.linear import QLinear
from oracle import dense

from .dense_helpers import DTYPE, Rows, check, encode, past_small, values
from .gguf_write import write_gguf

pytestmark = pytest.mark.gpu

FORWARD = {"bf16": 2.0 ** -8 + 5 * 2.0 ** -11, "f32": 8e-6}
BACKWARD = {"bf16": 2.0 ** -8 + 8 * 2.0 ** -11, "f32": 1.2e-5}
GRADS = ("dx", "dgate", "dup", "ddown")
# (hidden, ffn, formats): whole units and partial ones, widths that are no multiples of 64
SHAPES = [(256, 512, "Q4_K", "Q4_K"), (96, 160, "Q4_0", "Q4_1"), (288, 416, "Q4_1", "IQ4_NL"), (512, 1056, "IQ4_XS", "Q4_0"),
          (416, 256, "IQ4_NL", "IQ4_XS")]


def make(H: int, F: int, q: str, down: str, act: str = "silu", seed: int = 1) -> tuple[GatedFFN, list[np.ndarray]]:
    f = GatedFFN(hidden=H, ffn=F, gate_type=q, down_type=down, act=act)
    w = []
    for i, (name, t, r, c) in enumerate((("gate", q, F, H), ("up", q, F, H), ("down", down, H, F))):
        raw, v = dense.matrix(t, r, c, seed + i)
        f.upload("ffn_" + name, raw)
        w.append(v)
    return f, w


def rows(n: int, H: int, dtype: str, seed: int, size: float = 1.0) -> np.ndarray:
    return encode(size * np.random.default_rng(seed).standard_normal((n, H)), dtype)


def grads(f: GatedFFN, x: np.ndarray, dy: np.ndarray, names: tuple[str, ...] = GRADS) -> dict[str, np.ndarray]:
    shape = {"dx": x.shape, "dgate": (f.ffn, f.hidden), "dup": (f.ffn, f.hidden), "ddown": (f.hidden, f.ffn)}
    out = {k: np.full(shape[k], 7, x.dtype) for k in names}
    f.backward(x, dy, **out)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize(("H", "F", "q", "down"), SHAPES)
def test_forward(H: int, F: int, q: str, down: str, act: str, dtype: str) -> None:
    f, w = make(H, F, q, down, act)
    past = min(past_small(F, H, 1 if dtype == "bf16" else 3, True), past_small(H, F, 2))
    for n in (1, 3, 6, 16, 17, 40, 65, 128, 129, 192, 193, 240, 300, past):
        x = rows(n, H, dtype, n, 3.0)
        check(f(x), dense.ffn(act, values(x), *w), FORWARD[dtype])
    assert f(np.empty((0, H), DTYPE[dtype])).shape == (0, H)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize(("H", "F", "q", "down"), SHAPES)
def test_backward(H: int, F: int, q: str, down: str, act: str, dtype: str) -> None:
    """Every gradient, of rows of very different sizes with rows of zeros among them."""
    f, w = make(H, F, q, down, act)
    for n in (1, 2, 5, 16, 17, 31, 33, 64, 65, 128, 129, 192, 193, 240):
        x = rows(n, H, dtype, n, 3.0)
        size = 10.0 ** np.random.default_rng(n).uniform(-6, 1, (n, 1))
        size[2::5] = 0.0
        dy = encode(size * np.random.default_rng(n + 1).standard_normal((n, H)), dtype)
        want = dense.ffn_grad(act, values(x), values(dy), *w)
        got = grads(f, x, dy)
        for k in GRADS:
            check(got[k], want[k], BACKWARD[dtype])
        for r in range(n):  # (a row's gradient is as exact as the row is small)
            check(got["dx"][r:r + 1], want["dx"][r:r + 1], 1.5 * BACKWARD[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_tiles(dtype: str) -> None:
    """More tiles of 256 than CUs forward; sums over many rows backward."""
    f, w = make(256, 3200, "Q4_K", "Q4_0")
    n = 2821
    x, dy = rows(n, 256, dtype, 1, 2.0), rows(n, 256, dtype, 2)
    check(f(x), dense.ffn("silu", values(x), *w), FORWARD[dtype])
    want = dense.ffn_grad("silu", values(x), values(dy), *w)
    for k, g in grads(f, x, dy).items():
        check(g, want[k], BACKWARD[dtype])


def test_scales_beyond_their_values() -> None:
    """Matrices with groups whose values are small differences of their scales and offsets take the unpacked way."""
    H, F = 288, 416
    f, w = GatedFFN(hidden=H, ffn=F, gate_type="Q4_1", down_type="Q4_1"), []
    for i, (name, r, c) in enumerate((("gate", F, H), ("up", F, H), ("down", H, F))):
        raw, _ = dense.matrix("Q4_1", r, c, i)
        raw = raw.reshape(r, c // 32, 20).copy()
        raw[7, 2, :2], raw[7, 2, 2:4] = (np.array([v], np.float16).view(np.uint8) for v in (1.0, -15.0))
        raw[7, 2, 4:] = 0xFF  # (15 d + m = 0)
        f.upload("ffn_" + name, raw.reshape(r, -1))
        w.append(dense.gguf_ref.dequantize("Q4_1", raw.reshape(r, -1), c).astype(np.float64))
    for n in (9, 100, 240, 1500):
        x, dy = rows(n, H, "bf16", n, 3.0), rows(n, H, "bf16", n + 1)
        check(f(x), dense.ffn("silu", values(x), *w), FORWARD["bf16"])
        want = dense.ffn_grad("silu", values(x), values(dy), *w)
        for k, g in grads(f, x, dy).items():
            check(g, want[k], BACKWARD["bf16"])


def test_some_gradients() -> None:
    """Each set of outputs is what all of them together are; without rows the weights' gradients are zeros."""
    f, _ = make(96, 160, "Q4_0", "Q4_1")
    x, dy = rows(70, 96, "bf16", 1), rows(70, 96, "bf16", 2)
    full = grads(f, x, dy)
    for names in (("dx",), ("dgate",), ("dup",), ("ddown",), ("dx", "ddown"), ("dgate", "dup")):
        for k, g in grads(f, x, dy, names).items():
            assert np.array_equal(g, full[k]), names
    for dtype in ("bf16", "f32"):
        none = np.empty((0, 96), DTYPE[dtype])
        got = grads(f, none, none)
        assert got["dx"].shape == (0, 96) and not any(got[k].any() for k in GRADS)


def test_differences() -> None:
    """fp32 gradients against central differences of the operator itself. The operator is off by about 1e-6 of its size, a
    difference over a step of 2^-6 divides that by 2^-5: 3e-5 of y's norm; the third derivative's share is the step squared
    (2.4e-4) of a sum of order 1."""
    f, _ = make(96, 160, "Q4_0", "Q4_1")
    x, dy = rows(3, 96, "f32", 1), rows(3, 96, "f32", 2)
    dx = grads(f, x, dy, ("dx",))["dx"].astype(np.float64)
    rng = np.random.default_rng(3)
    for _ in range(4):
        v = rng.standard_normal(x.shape)
        v /= np.linalg.norm(v)
        hi, lo = (x + s * v for s in (2.0 ** -6, -2.0 ** -6))
        hi, lo = hi.astype(np.float32), lo.astype(np.float32)
        diff = ((f(hi).astype(np.float64) - f(lo)) * dy).sum() / np.sqrt(((hi.astype(np.float64) - lo) ** 2).sum())
        assert abs(diff - (dx * v).sum()) < 1e-3 * np.linalg.norm(dx) + 3e-5 * np.linalg.norm(dy) * np.linalg.norm(f(x))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides(dtype: str) -> None:
    """Rows at any address and stride; what surrounds the outputs stays; a broadcast dy."""
    H, F = 96, 160
    f, w = make(H, F, "IQ4_NL", "Q4_0")
    for n in (1, 5, 80, 200, 13200):
        for at, pad, oat, opad in ((0, 0, 0, 0), (1, 3, 2, 5), (8, 8, 1, 0)):
            xd, dyd = rows(n, H, dtype, 1), rows(n, H, dtype, 2)
            x, dy = (Rows(n, H, dtype, at=at, stride=H + pad, data=d) for d in (xd, dyd))
            y, dx = (Rows(n, H, dtype, at=oat, stride=H + opad) for _ in range(2))
            dw = [Rows(F, H, dtype, at=oat), Rows(F, H, dtype, at=oat), Rows(H, F, dtype, at=oat)]
            f(x, y)
            check(y.numpy(), dense.ffn("silu", values(xd), *w), FORWARD[dtype])
            f.backward(x, dy, dx=dx, dgate=dw[0], dup=dw[1], ddown=dw[2])
            want = dense.ffn_grad("silu", values(xd), values(dyd), *w)
            for k, g in zip(GRADS, [dx, *dw]):
                check(g.numpy(), want[k], BACKWARD[dtype])
        one = Rows(1, H, dtype, data=dyd[:1])
        one.shape, one.row = (n, H), 0
        dx = Rows(n, H, dtype)
        f.backward(x, one, dx=dx)
        want = dense.ffn_grad("silu", values(xd), np.repeat(values(dyd[:1]), n, 0), *w)
        check(dx.numpy(), want["dx"], BACKWARD[dtype])


def test_rows_are_their_own() -> None:
    """A row of infinities or NaN leaves the others' outputs and gradients as they are."""
    f, _ = make(96, 160, "Q4_0", "Q4_1")
    for n in (9, 80, 200, 13200):
        x, dy = rows(n, 96, "bf16", 1), rows(n, 96, "bf16", 2)
        y, dx = f(x), grads(f, x, dy, ("dx",))["dx"]
        bad = x.copy()
        bad[1, 3], bad[2, 4] = 0x7F80, 0x7FC0  # (inf, NaN)
        y2, dx2 = f(bad), grads(f, bad, dy, ("dx",))["dx"]
        keep = [i for i in range(n) if i not in (1, 2)]
        assert np.array_equal(y[keep], y2[keep]) and np.array_equal(dx[keep], dx2[keep])
        assert np.isnan(values(y2)[2]).all() and not np.isfinite(values(y2)[1]).any()


def test_refusals() -> None:
    f, _ = make(96, 160, "Q4_0", "Q4_1")
    x, y, dy = (DeviceArray((5, 96), np.uint16) for _ in range(3))
    with pytest.raises(_hip.Error, match="out overlaps x"):
        f(x, x)
    with pytest.raises(_hip.Error, match="device arrays need out"):
        f(x)
    with pytest.raises(_hip.Error, match="expected \\(5, 96\\)"):
        f(x, DeviceArray((5, 95), np.uint16))
    with pytest.raises(_hip.Error, match="out is .* of dtype 0"):
        f(x, DeviceArray((5, 96), np.float32))
    with pytest.raises(_hip.Error, match="dx overlaps dy"):
        f.backward(x, dy, dx=dy)
    with pytest.raises(_hip.Error, match="dgate is"):
        f.backward(x, dy, dgate=DeviceArray((96, 160), np.uint16))
    with pytest.raises(_hip.Error, match="rows are 97 values apart"):
        f.backward(x, dy, dgate=Rows(160, 96, "bf16", stride=97))
    with pytest.raises(_hip.Error, match="a workspace of 64 bytes, not"):
        f(x, y, work=Workspace(64))
    f.close()
    with pytest.raises(_hip.Error, match="closed"):
        f(x, y)
    g = GatedFFN(hidden=96, ffn=160, gate_type="Q4_0", down_type="Q4_1")
    with pytest.raises(_hip.Error, match="not uploaded"):
        g(x, y)


def test_blocks_of_a_file(tmp_path) -> None:
    """A projection, a dense block and a head of one file, one after another on the GPU, and the block's gradient."""
    H, F, V, n = 256, 512, 300, 70
    spec = [("blk.0.attn_output.weight", "IQ4_XS", H, H), ("blk.0.ffn_gate.weight", "Q4_K", F, H),
            ("blk.0.ffn_up.weight", "Q4_K", F, H), ("blk.0.ffn_down.weight", "Q4_0", H, F),
            ("output.weight", "Q4_1", V, H)]
    t, w = [], {}
    for i, (name, q, r, c) in enumerate(spec):
        raw, w[name] = dense.matrix(q, r, c, i)
        t.append((name, (c, r), TYPE_ID[q], raw))
    bias = np.random.default_rng(9).standard_normal(V).astype(np.float32)
    t.append(("output.bias", (V,), 0, bias))
    write_gguf(str(tmp_path / "m.gguf"), {"general.architecture": "qwen3moe"}, t)
    with GGUFFile(str(tmp_path / "m.gguf")) as file:
        proj = QLinear.from_gguf(file, "blk.0.attn_output.weight")
        block = GatedFFN.from_gguf(file, 0)
        head = QLinear.from_gguf(file, "output.weight", bias="output.bias")
        with pytest.raises(ValueError, match="no dense FFN"):
            GatedFFN.from_gguf(file, 1)
        with pytest.raises(ValueError, match="output.bias is F32, not one of"):
            QLinear.from_gguf(file, "output.bias")
    for m in (1, n):
        x = rows(m, H, "f32", 1)
        a, b, c = DeviceArray((m, H)), DeviceArray((m, H)), DeviceArray((m, V))
        d = DeviceArray.of(x)
        proj(d, a)
        block(a, b)
        head(b, c)
        p = values(x) @ w[spec[0][0]].T
        fw = [w[s[0]] for s in spec[1:4]]
        check(c.numpy(), dense.ffn("silu", p, *fw) @ w["output.weight"].T + bias, 2e-5)
        dx = DeviceArray((m, H))
        block.backward(a, d, dx=dx)
        check(dx.numpy(), dense.ffn_grad("silu", p, values(x), *fw)["dx"], 2e-5)
