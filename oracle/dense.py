"""The dense operators in 64 bits: one matrix's product, the gated feed-forward block and its gradients.

Test infrastructure only (see ``oracle/__init__.py``)."""

import numpy as np

from . import gguf_ref
from .tensors import random_blocks

FORMATS = ("Q4_0", "Q4_1", "Q4_K", "IQ4_NL", "IQ4_XS")
# fp16 scales that make values of about 0.02 to 0.1 whatever the format's codes are worth
SCALE = {"Q4_0": 0.01, "Q4_1": 0.01, "Q4_K": 4e-4, "IQ4_NL": 1e-3, "IQ4_XS": 4e-5}
GELU_K, GELU_C = np.sqrt(2.0 / np.pi), 0.044715


def matrix(q: str, rows: int, cols: int, seed: int) -> tuple[np.ndarray, np.ndarray]:
    """Random blocks and their values in 64 bits (exact: the fp32 values)."""
    raw = random_blocks(q, rows, cols, seed, scale=SCALE[q])
    return raw, gguf_ref.dequantize(q, raw, cols).astype(np.float64)


def act(name: str, g: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """The activation and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + np.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    t = np.tanh(GELU_K * (g + GELU_C * g ** 3))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * GELU_K * (1.0 + 3.0 * GELU_C * g * g)


def ffn(name: str, x: np.ndarray, gate: np.ndarray, up: np.ndarray, down: np.ndarray) -> np.ndarray:
    return (act(name, x @ gate.T)[0] * (x @ up.T)) @ down.T


def ffn_grad(name: str, x: np.ndarray, dy: np.ndarray, gate: np.ndarray, up: np.ndarray, down: np.ndarray
             ) -> dict[str, np.ndarray]:
    g, u = x @ gate.T, x @ up.T
    a, da = act(name, g)
    dh = dy @ down
    dg, du = dh * u * da, dh * a
    return {"dx": dg @ gate + du @ up, "dgate": dg.T @ x, "dup": du.T @ x, "ddown": dy.T @ (a * u)}
