"""The dense operators on torch tensors, streams and graphs: a program of its own, since torch has to be imported before the
library loads (both then share torch's HIP runtime). Run by test_dense_torch_gpu.py.

TOL: a bf16 output's half step (2^-8) and the inner roundings' eighths of it (at most 8)."""

import sys
import threading
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from artlite_amd import _hip  # noqa: E402
from artlite_amd.device import Workspace  # noqa: E402
from artlite_amd.ffn import GatedFFN  # noqa: E402
from artlite_amd.linear import QLinear  # noqa: E402
from oracle import dense  # noqa: E402

TOL = 2.0 ** -8 + 8 * 2.0 ** -11


def refused(call: object) -> None:
    """A captured call on the workspace that a device's calls share (there already, or to be grown)."""
    try:
        call()
    except _hip.Error as e:
        assert "a captured call takes a workspace of its own" in str(e), e
    else:
        raise AssertionError("captured")


def linear_streams_and_graphs() -> None:
    """Torch tensors: calls that alternate between streams on one object's workspace; captured calls replayed with other
    inputs, beside eager ones on workspaces of their own."""
    N, K = 2000, 512
    lin = QLinear("Q4_1", N, K)
    raw, w = dense.matrix("Q4_1", N, K, 8)
    lin.upload(raw)
    w = torch.from_numpy(w)

    def ref(x: object) -> object:
        return x.cpu().double() @ w.T

    def near(y: object, x: object) -> None:
        want = ref(x)
        assert (y.cpu().double() - want).norm() <= 2.0 ** -7 * want.norm()

    streams = [torch.cuda.Stream() for _ in range(3)]
    xs = [torch.randn(1034 + i, K, device="cuda").bfloat16() for i in range(12)]
    ys = [torch.empty(x.shape[0], N, device="cuda", dtype=torch.bfloat16) for x in xs]
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(xs, ys)):
        lin(x, y, stream=streams[i % 3].cuda_stream)
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        near(y, x)
    graphs = []
    wide, out = (torch.empty(50000, c, device="cuda", dtype=torch.bfloat16) for c in (K, N))
    for M in (1, 100, 1100):
        x = torch.randn(M, K, device="cuda").bfloat16()
        y = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        work = Workspace(max(1, lin.workspace_bytes(M, "bf16")))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s = torch.cuda.current_stream().cuda_stream
            if lin.workspace_bytes(M, "bf16"):  # (nothing has been queued or allocated: the capture goes on)
                refused(lambda: lin(x, y, stream=s))
                refused(lambda: lin(wide, out, stream=s))
            lin(x, y, stream=s, work=work)
        graphs.append((g, x, y, work))
    for _ in range(3):
        for g, x, y, _ in graphs:
            x.copy_(torch.randn_like(x))
            y.zero_()
            g.replay()
        lin(xs[0], ys[0])
        torch.cuda.synchronize()
        for _, x, y, _ in graphs:
            near(y, x)
        near(ys[0], xs[0])


def ffn_streams_and_graphs() -> None:
    """Torch tensors on several streams over one workspace; forward and backward captured and replayed with other inputs,
    beside eager calls on other workspaces."""
    H, F = 256, 512
    f, w = GatedFFN(hidden=H, ffn=F, gate_type="Q4_K", down_type="Q4_K"), []
    for i, (name, r, c) in enumerate((("gate", F, H), ("up", F, H), ("down", H, F))):
        raw, v = dense.matrix("Q4_K", r, c, i)
        f.upload("ffn_" + name, raw)
        w.append(v)

    def near(got: object, want: np.ndarray, tol: float) -> None:
        assert np.linalg.norm(got.double().cpu().numpy() - want) <= tol * np.linalg.norm(want)

    def host(t: object) -> np.ndarray:
        return t.double().cpu().numpy()

    def rand(n: int) -> object:
        return torch.randn(n, H, device="cuda").bfloat16()

    streams = [torch.cuda.Stream() for _ in range(3)]
    xs = [rand(n) for n in (5, 4200, 64, 129, 1, 33)]
    ys = [torch.empty_like(x) for x in xs]
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(xs, ys)):
        f(x, y, stream=streams[i % 3].cuda_stream)
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        near(y, dense.ffn("silu", host(x), *w), TOL)
    graphs = []
    for n in (4, 150, 220, 4200):
        x, dy = rand(n), rand(n)
        out = {"y": torch.empty_like(x), "dx": torch.empty_like(x),
               "dgate": torch.empty(F, H, device="cuda", dtype=torch.bfloat16)}
        work = Workspace(max(f.workspace_bytes(n), f.workspace_bytes(n, weights=True)))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s = torch.cuda.current_stream().cuda_stream
            f(x, out["y"], stream=s, work=work)
            f.backward(x, dy, dx=out["dx"], dgate=out["dgate"], stream=s, work=work)
        graphs.append((g, x, dy, out, work))
    for _ in range(3):
        for g, x, dy, out, _ in graphs:
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(dy))
            for t in out.values():
                t.zero_()
            g.replay()
        f(xs[1], ys[1])
        torch.cuda.synchronize()
        near(ys[1], dense.ffn("silu", host(xs[1]), *w), TOL)
        for _, x, dy, out, _ in graphs:
            want = {"y": dense.ffn("silu", host(x), *w), **dense.ffn_grad("silu", host(x), host(dy), *w)}
            for k, t in out.items():
                near(t, want[k], TOL)


def far_rows() -> None:
    """Rows whose offsets pass 32 bits, in values and in bytes."""
    N, K = 1600, 512
    lin = QLinear("Q4_K", N, K)
    raw, w = dense.matrix("Q4_K", N, K, 8)
    lin.upload(raw)
    w = torch.from_numpy(w)
    f, fw = GatedFFN(hidden=256, ffn=512, gate_type="Q4_0", down_type="IQ4_NL"), []
    for i, (name, q, r, c) in enumerate((("gate", "Q4_0", 512, 256), ("up", "Q4_0", 512, 256), ("down", "IQ4_NL", 256, 512))):
        raw, v = dense.matrix(q, r, c, i)
        f.upload("ffn_" + name, raw)
        fw.append(v)

    def rows(n: int, cols: int, stride: int) -> object:
        return torch.empty((n - 1) * stride + cols, device="cuda", dtype=torch.bfloat16).as_strided((n, cols), (stride, 1))

    def near(y: object, want: np.ndarray) -> None:
        assert np.linalg.norm(y.double().cpu().numpy() - want) <= TOL * np.linalg.norm(want)

    for M, stride in ((3, 2_200_000_001), (90, 50_000_001), (1300, 3_400_003)):
        x, y = rows(M, K, stride), rows(M, N, stride)
        x.copy_(torch.randn(M, K, device="cuda"))
        torch.cuda.synchronize()
        lin(x, y)
        near(y, (x.cpu().double() @ w.T).numpy())
        del x, y
        x, dy, y, dx = (rows(M, 256, stride) for _ in range(4))
        for t in (x, dy):
            t.copy_(torch.randn(M, 256, device="cuda"))
        torch.cuda.synchronize()
        f(x, y)
        f.backward(x, dy, dx=dx)
        xs, dys = (t.double().cpu().numpy() for t in (x, dy))
        near(y, dense.ffn("silu", xs, *fw))
        near(dx, dense.ffn_grad("silu", xs, dys, *fw)["dx"])
        del x, dy, y, dx
        torch.cuda.empty_cache()


def threads_and_shared_workspaces() -> None:
    """Threads on streams of their own, over one object and the workspace that they share; graphs that share a workspace,
    replayed in turn on one stream."""
    N, K, M = 2000, 512, 1100
    lin = QLinear("Q4_1", N, K)
    raw, w = dense.matrix("Q4_1", N, K, 8)
    lin.upload(raw)
    w = torch.from_numpy(w).cuda()
    xs = [torch.randn(M + i, K, device="cuda").bfloat16() for i in range(4)]
    ys = [torch.empty(M + i, N, device="cuda", dtype=torch.bfloat16) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()

    def near(y: object, x: object) -> None:
        want = x.double() @ w.T
        assert (y.double() - want).norm() <= TOL * want.norm()

    def run(i: int) -> None:
        for _ in range(40):
            lin(xs[i], ys[i], stream=streams[i].cuda_stream)

    all_ = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in all_:
        t.start()
    for t in all_:
        t.join()
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        near(y, x)
    work = Workspace(max(lin.workspace_bytes(x.shape[0]) for x in xs))
    graphs = []
    for x, y in zip(xs, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lin(x, y, stream=torch.cuda.current_stream().cuda_stream, work=work)
        graphs.append(g)
    for _ in range(3):
        for x, y, g in zip(xs, ys, graphs):
            x.copy_(torch.randn_like(x))
            y.zero_()
            g.replay()
        torch.cuda.synchronize()
        for x, y in zip(xs, ys):
            near(y, x)


if __name__ == "__main__":
    for case in (linear_streams_and_graphs, ffn_streams_and_graphs, far_rows, threads_and_shared_workspaces):
        case()
        print(case.__name__, "passed", flush=True)
