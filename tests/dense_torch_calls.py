"""The dense operators beside torch: streams that arrays name, threads on their default streams, tensors that require grad,
columns of one tensor, gradients in graphs. A program of its own, which imports torch before the library loads. Run by test_dense_torch_calls_gpu.py.

TOL: a bf16 output's half step (2^-8) and the inner roundings' eighths of it (at most 8)."""

import sys
import threading
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from artlite_amd import _hip  # noqa: E402
from artlite_amd.device import Workspace  # noqa: E402
from artlite_amd.ffn import GatedFFN  # noqa: E402
from artlite_amd.linear import QLinear  # noqa: E402
from oracle import dense  # noqa: E402

TOL = 2.0 ** -8 + 8 * 2.0 ** -11
N, K = 2000, 512


def make() -> tuple[QLinear, torch.Tensor]:
    lin = QLinear("Q4_1", N, K)
    raw, w = dense.matrix("Q4_1", N, K, 8)
    lin.upload(raw)
    return lin, torch.from_numpy(w).cuda()


def near(y: torch.Tensor, x: torch.Tensor, w: torch.Tensor) -> None:
    want = x.double() @ w.T
    assert (y.double() - want).norm() <= TOL * want.norm()


class Interface:
    """A tensor's interface alone, with the stream that it was last written on."""

    def __init__(self, t: torch.Tensor, stream: int | None):
        self.__cuda_array_interface__ = {"shape": tuple(t.shape), "typestr": "<u2", "version": 3, "stream": stream,
                                         "data": (t.data_ptr(), False), "strides": tuple(2 * s for s in t.stride())}


def streams_of_interfaces() -> None:
    """x is written on another stream behind some work, which the call's stream has not waited for."""
    lin, w = make()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    for M in (1, 300, 1100):
        data = torch.randn(M, K, device="cuda").bfloat16()
        x, y = torch.zeros_like(data), torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            for _ in range(20):
                big @ big
            x.copy_(data)
        lin(Interface(x, a.cuda_stream), Interface(y, None), stream=b.cuda_stream)
        b.synchronize()
        near(y, data, w)


def per_thread_streams() -> None:
    """Threads that each name hipStreamPerThread (2) over the workspace that they share."""
    lin, w = make()
    xs = [torch.randn(1100 + i, K, device="cuda").bfloat16() for i in range(4)]
    ys = [torch.empty(x.shape[0], N, device="cuda", dtype=torch.bfloat16) for x in xs]
    torch.cuda.synchronize()

    def run(i: int) -> None:
        for _ in range(40):
            lin(xs[i], ys[i], stream=2)

    all_ = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in all_:
        t.start()
    for t in all_:
        t.join()
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        near(y, x, w)


def tensors_that_require_grad() -> None:
    """Read, and written under no_grad or inside a Function; refused as outputs while a graph is recorded."""
    H, F = 256, 512
    f = GatedFFN(hidden=H, ffn=F, gate_type="Q4_K", down_type="Q4_K")
    w = []
    for i, (name, r, c) in enumerate((("gate", F, H), ("up", F, H), ("down", H, F))):
        raw, v = dense.matrix("Q4_K", r, c, i)
        f.upload("ffn_" + name, raw)
        w.append(torch.from_numpy(v))

    def stream() -> int:
        return torch.cuda.current_stream().cuda_stream

    class Block(torch.autograd.Function):
        @staticmethod
        def forward(ctx: object, x: torch.Tensor) -> torch.Tensor:
            ctx.save_for_backward(x)
            return f(x, torch.empty_like(x), stream=stream())

        @staticmethod
        def backward(ctx: object, dy: torch.Tensor) -> torch.Tensor:
            x, = ctx.saved_tensors
            dx = torch.empty_like(x)
            f.backward(x, dy.contiguous(), dx=dx, stream=stream())
            return dx

    x = torch.randn(70, H, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(70, H, device="cuda").bfloat16()
    Block.apply(x).backward(dy)
    xd = x.detach().cpu().double().requires_grad_()
    g = xd @ w[0].T
    ((g * torch.sigmoid(g) * (xd @ w[1].T)) @ w[2].T).backward(dy.cpu().double())
    assert (x.grad.cpu().double() - xd.grad).norm() <= TOL * xd.grad.norm()
    out = torch.zeros_like(x).detach().requires_grad_()
    try:
        f(x, out)
    except _hip.Error as e:
        assert "ffn: out: requires grad" in str(e), e
    else:
        raise AssertionError("written")
    torch.cuda.synchronize()
    assert not out.any()
    with torch.no_grad():
        f(x, out)
    torch.cuda.synchronize()
    assert out.any()


def columns_of_one_tensor() -> None:
    lin, w = make()
    for M in (1, 40, 1100):
        whole = torch.randn(M, 3 * K + N, device="cuda").bfloat16()
        before = whole.clone()
        torch.cuda.synchronize()
        x, y = whole[:, K:2 * K], whole[:, 2 * K:2 * K + N]
        lin(x, y)
        torch.cuda.synchronize()
        near(y, before[:, K:2 * K], w)
        before[:, 2 * K:2 * K + N] = y
        assert torch.equal(whole, before)


def gradients_in_graphs() -> None:
    """Every gradient captured, replayed with inputs of other sizes and eager calls between: the eager call's bits each time
    (nothing of a replay's powers of two is left for the next)."""
    H, F = 256, 608
    f = GatedFFN(hidden=H, ffn=F, gate_type="Q4_0", down_type="IQ4_NL")
    for i, (name, q, r, c) in enumerate((("gate", "Q4_0", F, H), ("up", "Q4_0", F, H), ("down", "IQ4_NL", H, F))):
        f.upload("ffn_" + name, dense.matrix(q, r, c, i)[0])
    for n in (1, 30, 64, 65, 300, 1500):
        for dtype in (torch.bfloat16, torch.float32):
            x, dy = (torch.randn(n, H, device="cuda").to(dtype) for _ in range(2))
            shapes = {"dx": (n, H), "dgate": (F, H), "dup": (F, H), "ddown": (H, F)}
            out, eager = ({k: torch.empty(s, device="cuda", dtype=dtype) for k, s in shapes.items()} for _ in range(2))
            work = Workspace(f.workspace_bytes(n, "bf16" if dtype == torch.bfloat16 else "f32", weights=True))
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                f.backward(x, dy, **out, stream=torch.cuda.current_stream().cuda_stream, work=work)
            for size, grad in ((1.0, 1.0), (1e6, 1e-3), (1e-12, 1e4), (0.0, 1.0), (1.0, 1e-20), (1.0, 1.0)):
                x.copy_(size * torch.randn(n, H, device="cuda"))
                dy.copy_(grad * torch.randn(n, H, device="cuda"))
                for t in out.values():
                    t.fill_(7)
                g.replay()
                f.backward(x, dy, **eager)
                torch.cuda.synchronize()
                for k, t in out.items():
                    assert torch.equal(t, eager[k]), (n, dtype, size, k)
                assert all(t.isfinite().all() for t in out.values())


if __name__ == "__main__":
    for case in (streams_of_interfaces, per_thread_streams, tensors_that_require_grad, columns_of_one_tensor, gradients_in_graphs):
        case()
        print(case.__name__, "passed", flush=True)
