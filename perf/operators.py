"""Dense products over the blocks of a GGUF file: one matrix's product (an attention projection, the output head) and the
gated feed-forward block with its backward pass, from single tokens to training batches.

``linear``: y = x W^T + b with W (N, K) in a 4-bit format (codes and a scale, or scale and min, for each 32 values).
``ffn``: y = (act(x Wg^T) (x Wu^T)) Wd^T; ``ffn_grad``: from x and dy the gradient of x and, with "weights", those of the
three matrices' values. Activations, outputs and gradients are bf16 or fp32. Sizes are generic ones and the tests'."""

import math

import torch

own = False

# format: values per block, bytes per block, byte offsets of its fp16 fields (the scale, then the min's scale)
BLOCK = {"Q4_0": (32, 18, (0,)), "Q4_1": (32, 20, (0, 2)), "IQ4_NL": (32, 18, (0,)), "Q4_K": (256, 144, (0, 2)),
         "IQ4_XS": (256, 136, (0,))}
# what one code step is worth as a share of a block's fp16 scale, about (K-quants' 6-bit scales, IQ4's wider steps)
STEP = {"Q4_0": 1.0, "Q4_1": 1.0, "IQ4_NL": 15.0, "Q4_K": 32.0, "IQ4_XS": 15.0 * 16.0}
IQ4 = (-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113)
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST_FLOPS = 3.3e12  # the largest listed pass


def listed():
    def linear(name, M, N, K, q, x="bf16", bias=False):
        return dict(name=name, kind="linear", M=M, N=N, K=K, q=q, x=x, bias=bias)

    def ffn(name, T, H, F, q, down, x="bf16", act="silu"):
        return dict(name=name, kind="ffn", T=T, H=H, F=F, q=q, down=down, x=x, act=act)

    def grad(name, T, H, F, q, down, x="bf16", act="silu", weights=False):
        return dict(name=name, kind="ffn_grad", T=T, H=H, F=F, q=q, down=down, x=x, act=act, weights=weights)

    return [
        # an attention projection for one token: a call is a launch and its latency
        linear("linear 1", 1, 2048, 2048, "Q4_0"),
        # the output head of a vocabulary for one token, in a K-quant
        linear("linear 1 head", 1, 131072, 2048, "Q4_K"),
        # a wide projection for a batch of sequences that decode together
        linear("linear 16", 16, 8192, 4096, "IQ4_XS"),
        # fp32 activations, an odd number of outputs, a width of no whole 256 values, a bias
        linear("linear 5 f32", 5, 1531, 2880, "Q4_1", x="f32", bias=True),
        # drafted or chunked tokens: between single tokens and prompts
        linear("linear 77", 77, 4096, 4096, "Q4_K"),
        # a chunk of a prompt through a projection
        linear("linear 1000", 1000, 6144, 2048, "IQ4_NL"),
        # a dense block for one token
        ffn("ffn 1", 1, 2048, 8192, "Q4_K", "Q4_K"),
        # a dense block for a batch of sequences, another activation
        ffn("ffn 24 gelu", 24, 2880, 7680, "Q4_0", "Q4_1", act="gelu_tanh"),
        # a prompt of no round length
        ffn("ffn 3001", 3001, 4096, 11008, "Q4_K", "Q4_K"),
        # training adapters below or beside frozen blocks: the input's gradient alone
        grad("ffn grad 2048", 2048, 2048, 8192, "Q4_0", "Q4_0"),
        # a few fp32 tokens with the weights' gradients: sensitivities of a small block
        grad("ffn grad 45 f32", 45, 1024, 2816, "IQ4_NL", "Q4_K", x="f32", act="gelu_tanh", weights=True),
        # a training batch, every gradient
        grad("ffn grad 4096 weights", 4096, 4096, 8192, "Q4_K", "Q4_K", weights=True),
    ]


def _flops(case):
    if case["kind"] == "linear":
        return 2.0 * case["M"] * case["N"] * case["K"]
    one = 2.0 * case["T"] * case["H"] * case["F"]  # one product of the block
    return one * {"ffn": 3, "ffn_grad": 8 if case.get("weights") else 5}[case["kind"]]


def draw(rng):
    def spread(lo, hi, step=1):
        return max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step

    kind = rng.choice(["linear", "linear", "ffn", "ffn_grad"])
    x = rng.choice(["bf16", "bf16", "bf16", "f32"])
    q, down = (rng.choice(list(BLOCK)) for _ in range(2))
    while True:
        if kind == "linear":
            case = dict(kind=kind, M=spread(1, 4096), N=spread(256, 32768), K=spread(512, 12288, BLOCK[q][0]), q=q, x=x,
                        bias=rng.random() < 0.3)
        else:
            case = dict(kind=kind, T=spread(1, 4096), H=spread(512, 6144, max(BLOCK[q][0], 32)),
                        F=spread(1024, 16384, max(BLOCK[down][0], 32)), q=q, down=down, x=x,
                        act=rng.choice(["silu", "silu", "gelu_tanh"]))
            if kind == "ffn_grad":
                case["weights"] = rng.random() < 0.5
        # (fp32 takes several products of 16 bits for each of its own)
        if _flops(case) * (4 if x == "f32" else 1) <= MOST_FLOPS:
            return case


# ---- inputs


def _blocks(g, q, rows, cols):
    """Random blocks (rows, row bytes) of about unit-gain weights: codes uniform, fp16 scales |N| about the size that gives
    |w| about 1 / sqrt(cols), mins that about centre the codes."""
    per, nb, f16 = BLOCK[q]
    n = rows * (cols // per)
    raw = torch.randint(0, 256, (n, nb), dtype=torch.uint8, device="cuda", generator=g)
    size = 0.2 / (STEP[q] * math.sqrt(cols))
    for i, o in enumerate(f16):
        d = torch.randn(n, device="cuda", generator=g).abs() * size
        if i:  # (w = d q + m: m about -7.5 d; K: w = d sc q - dmin m)
            d = d * (-7.5 if q == "Q4_1" else 7.5)
        raw[:, o:o + 2] = d.to(torch.float16).view(torch.uint8).view(n, 2)
    return raw.view(rows, -1)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPE[case["x"]]
    if case["kind"] == "linear":
        N, K = case["N"], case["K"]
        s = {"w": _blocks(g, case["q"], N, K), "x": torch.randn(case["M"], K, device="cuda", generator=g).to(dt)}
        s["b"] = torch.randn(N, device="cuda", generator=g) if case["bias"] else None
        return s
    T, H, F = case["T"], case["H"], case["F"]
    s = {"gate": _blocks(g, case["q"], F, H), "up": _blocks(g, case["q"], F, H), "down": _blocks(g, case["down"], H, F),
         "x": (2.0 * torch.randn(T, H, device="cuda", generator=g)).to(dt)}
    if case["kind"] == "ffn_grad":
        # (a loss's gradients: small, of another size for every token, and none for a padded one)
        size = 1e-3 * torch.exp(torch.randn(T, 1, device="cuda", generator=g))
        if T > 8:
            size[-(T // 8):] = 0.0
        s["dy"] = (size * torch.randn(T, H, device="cuda", generator=g)).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    dt = DTYPE[case["x"]]
    empty = lambda *shape: torch.empty(shape, dtype=dt, device="cuda")  # noqa: E731
    if case["kind"] == "linear":
        s["y"] = empty(case["M"], case["N"])
    else:
        T, H, F = case["T"], case["H"], case["F"]
        if case["kind"] == "ffn":
            s["y"] = empty(T, H)
        else:
            s["grads"] = {"dx": empty(T, H)}
            if case["weights"]:
                s["grads"].update(dgate=empty(F, H), dup=empty(F, H), ddown=empty(H, F))
    if own:  # (a program keeps its uploaded matrices)
        if case["kind"] == "linear":
            from artlite_amd.linear import QLinear

            s["op"] = QLinear(case["q"], case["N"], case["K"])
            s["op"].upload(s["w"].cpu().numpy(), bias=None if s["b"] is None else s["b"].cpu().numpy())
        else:
            from artlite_amd.ffn import GatedFFN

            s["op"] = GatedFFN(hidden=H, ffn=F, gate_type=case["q"], down_type=case["down"], act=case["act"])
            for name in ("gate", "up", "down"):
                s["op"].upload("ffn_" + name, s[name].cpu().numpy())
    return s


# ---- a pass


def _dequant(q, raw, cols, dt=torch.float32):
    """The weights (rows, cols) of rows of blocks."""
    rows = raw.shape[0]
    per, nb, f16 = BLOCK[q]
    b = raw.view(rows, cols // per, nb)
    n = b.shape[1]
    d, *m = (b[..., o:o + 2].contiguous().view(torch.float16).to(dt) for o in f16)
    if q == "Q4_K":
        lo, hi, top = b[..., 4:8], b[..., 8:12], b[..., 12:16]
        sc = torch.cat([lo & 63, (top & 15) | ((lo >> 6) << 4)], -1).to(dt)
        mn = torch.cat([hi & 63, (top >> 4) | ((hi >> 6) << 4)], -1).to(dt)
        c = b[..., 16:].reshape(rows, n, 4, 32)
        c = torch.stack([c & 15, c >> 4], 3).reshape(rows, n, 8, 32).to(dt)
        return ((d * sc)[..., None] * c - (m[0] * mn)[..., None]).reshape(rows, cols)
    if q == "IQ4_XS":
        high = (b[..., 2:4].to(torch.int32) * torch.tensor([1, 256], device=b.device, dtype=torch.int32)).sum(-1, keepdim=True)
        at = torch.arange(8, device=b.device, dtype=torch.int32)
        low = torch.stack([b[..., 4:8] & 15, b[..., 4:8] >> 4], -1).reshape(rows, n, 8)
        ls = low.to(torch.int32) | (((high >> (2 * at)) & 3) << 4)
        c = b[..., 8:].reshape(rows, n, 8, 16)
        c = torch.cat([c & 15, c >> 4], -1)
        values = torch.tensor(IQ4, dtype=dt, device=b.device)
        return ((d * (ls - 32).to(dt))[..., None] * values[c.long()]).reshape(rows, cols)
    c = b[..., nb - 16:]
    c = torch.cat([c & 15, c >> 4], -1)
    if q == "IQ4_NL":
        w = d * torch.tensor(IQ4, dtype=dt, device=b.device)[c.long()]
    elif q == "Q4_1":
        w = d * c.to(dt) + m[0]
    else:
        w = d * (c.to(dt) - 8.0)
    return w.reshape(rows, cols)


GELU = math.sqrt(2.0 / math.pi), 0.044715


def _act(act, g):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(GELU[0] * (g + GELU[1] * g * g * g)))


def _act_grad(act, g):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    t = torch.tanh(GELU[0] * (g + GELU[1] * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * GELU[0] * (1.0 + 3.0 * GELU[1] * g * g)


def run(state):
    case = state["case"]
    dt = DTYPE[case["x"]]
    if case["kind"] == "linear":
        if own:
            return {"y": state["op"](state["x"], out=state["y"])}
        y = state["x"].float() @ _dequant(case["q"], state["w"], case["K"]).T
        return {"y": (y if state["b"] is None else y + state["b"]).to(dt)}
    if case["kind"] == "ffn":
        if own:
            return {"y": state["op"](state["x"], out=state["y"])}
        x = state["x"].float()
        h = _act(case["act"], x @ _dequant(case["q"], state["gate"], case["H"]).T)
        h = h * (x @ _dequant(case["q"], state["up"], case["H"]).T)
        return {"y": (h @ _dequant(case["down"], state["down"], case["F"]).T).to(dt)}
    if own:
        state["op"].backward(state["x"], state["dy"], **state["grads"])
        return state["grads"]
    x, dy = state["x"].float(), state["dy"].float()
    gate, up = (_dequant(case["q"], state[n], case["H"]) for n in ("gate", "up"))
    down = _dequant(case["down"], state["down"], case["F"])
    g, u = x @ gate.T, x @ up.T
    dh, a = dy @ down, _act(case["act"], g)
    dg, du = dh * u * _act_grad(case["act"], g), dh * a
    out = {"dx": (dg @ gate + du @ up).to(dt)}
    if case["weights"]:
        out.update(dgate=(dg.T @ x).to(dt), dup=(du.T @ x).to(dt), ddown=(dy.T @ (a * u)).to(dt))
    return out


# ---- what a pass cannot do without


def work(case):
    v = 2.0 if case["x"] == "bf16" else 4.0

    def blocks(q, n):
        return n * BLOCK[q][1] / BLOCK[q][0]

    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": blocks(case["q"], float(N) * K) + v * M * (N + K) + 4.0 * N * case["bias"], "flops": _flops(case)}
    T, H, F = case["T"], case["H"], case["F"]
    nbytes = 2 * blocks(case["q"], float(H) * F) + blocks(case["down"], float(H) * F) + v * 2 * T * H
    if case["kind"] == "ffn_grad":
        nbytes += v * T * H + (3 * v * H * F if case["weights"] else 0.0)
    return {"bytes": nbytes, "flops": _flops(case)}


# ---- results in 64 bits


def _blockwise(q, raw, cols):
    """The weights in 64 bits, a block's fields taken one value of the block at a time."""
    per, nb, _ = BLOCK[q]
    rows = raw.shape[0]
    b = raw.view(rows, cols // per, nb)
    half = lambda o: (b[..., o].to(torch.int32) | (b[..., o + 1].to(torch.int32) << 8)).to(torch.int16).view(torch.float16).double()  # noqa: E731
    d = half(0)
    table = torch.tensor(IQ4, dtype=torch.float64, device=raw.device)
    w = torch.empty(rows, cols // per, per, dtype=torch.float64, device=raw.device)
    for j in range(per):
        g, i = j // 32, j % 32
        if q == "Q4_K":
            byte = b[..., 16 + 32 * (g // 2) + i].int()
            c = (byte >> 4 if g % 2 else byte & 15).double()
            if g < 4:
                sc, mn = b[..., 4 + g].int() & 63, b[..., 8 + g].int() & 63
            else:
                sc = (b[..., 8 + g].int() & 15) + 16 * (b[..., g].int() >> 6)
                mn = (b[..., 8 + g].int() >> 4) + 16 * (b[..., 4 + g].int() >> 6)
            w[..., j] = d * sc * c - half(2) * mn
            continue
        first = {"Q4_0": 2, "IQ4_NL": 2, "Q4_1": 4, "IQ4_XS": 8 + 16 * g}[q]
        byte = b[..., first + i % 16].int()
        c = byte & 15 if i < 16 else byte >> 4
        if q == "Q4_0":
            w[..., j] = d * (c.double() - 8)
        elif q == "Q4_1":
            w[..., j] = d * c.double() + half(2)
        elif q == "IQ4_NL":
            w[..., j] = d * table[c.long()]
        else:
            low = b[..., 4 + g // 2].int()
            low = low >> 4 if g % 2 else low & 15
            high = (b[..., 2 + g // 4].int() >> (2 * (g % 4))) & 3
            w[..., j] = d * (low + 16 * high - 32).double() * table[c.long()]
    return w.view(rows, cols)


def exact(case, seed):
    s = _inputs(case, seed)
    x = s["x"].double()
    if case["kind"] == "linear":
        y = x @ _blockwise(case["q"], s["w"], case["K"]).T
        return {"y": y if s["b"] is None else y + s["b"].double()}
    gate, up = (_blockwise(case["q"], s[n], case["H"]) for n in ("gate", "up"))
    down = _blockwise(case["down"], s["down"], case["F"])
    g, u = x @ gate.T, x @ up.T
    if case["act"] == "silu":
        p = torch.sigmoid(g)
        a, slope = g * p, p + g * p * (1 - p)
    else:
        k, c = GELU
        p = torch.sigmoid(2 * k * (g + c * g ** 3))  # ((1 + tanh z) / 2 is sigmoid(2 z))
        a, slope = g * p, p + g * p * (1 - p) * 2 * k * (1 + 3 * c * g ** 2)
    if case["kind"] == "ffn":
        return {"y": (a * u) @ down.T}
    dy = s["dy"].double()
    dh = dy @ down
    dg, du = dh * u * slope, dh * a
    out = {"dx": dg @ gate + du @ up}
    if case["weights"]:
        out.update(dgate=dg.T @ x, dup=du.T @ x, ddown=dy.T @ (a * u))
    return out
