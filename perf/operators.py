"""Cases and plain forms of the dense operators that stand beside the routed layer.

linear     y = x . W^T, W in NVFP4 (E2M1 codes, an e4m3 scale for 16 of them, one fp32 scale);
           gated: the rows of W are gate rows and up rows, and y = silu(gate) * up; add: a tensor
           of y's shape is added (the routed experts' output, a residual stream)
ffn        y = (silu(x . Wg^T) * (x . Wu^T)) . W2^T (+ add), 16-bit weights: a shared expert
ffn_train  the same forward pass, and from dy the gradients of x, w13 = [Wg; Wu] and w2

`own` false: the plain form, in elementary torch operations and 32 bits; true: the framework's calls.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _linear(name, T, K, N, gated, dtype, add):
    return {"name": name, "op": "linear", "T": T, "K": K, "N": N, "gated": gated, "dtype": dtype, "add": add}


def _ffn(name, op, T, H, I, dtype, add):
    return {"name": name, "op": op, "T": T, "H": H, "I": I, "dtype": dtype, "add": add}


def listed():
    return [
        # one token through the first half of a small 4-bit shared expert: latency counts
        _linear("linear 1 small", 1, 1024, 1024, True, "bf16", False),
        # one token through the first half of a large 4-bit shared expert: weight streaming
        _linear("linear 1 gated", 1, 7168, 4096, True, "bf16", False),
        # a small decode batch through its second half, onto the routed experts' output
        _linear("linear 13 down", 13, 2048, 7168, False, "fp16", True),
        # a decode batch of 32 through a wide gated projection
        _linear("linear 32 gated", 32, 4096, 8192, True, "bf16", False),
        # ragged: sizes that end inside every tile, more tokens than a decode batch
        _linear("linear 77 odd", 77, 1008, 1001, False, "bf16", True),
        # a prompt of 4096 tokens through a square projection
        _linear("linear 4096", 4096, 4096, 4096, False, "bf16", False),
        # one token through a 16-bit shared expert of a large layer, added to the routed output
        _ffn("ffn 1", "ffn", 1, 7168, 2048, "bf16", True),
        # a decode batch through the shared expert of a small layer
        _ffn("ffn 24", "ffn", 24, 2048, 768, "fp16", False),
        # a short prompt of odd length, inner size off the tiles
        _ffn("ffn 509 odd", "ffn", 509, 4096, 1288, "bf16", False),
        # a prompt of 8192 tokens through the large layer's shared expert
        _ffn("ffn 8192", "ffn", 8192, 7168, 2048, "bf16", True),
        # a training step on a small batch of odd length
        _ffn("ffn_train 257", "ffn_train", 257, 2048, 768, "fp16", False),
        # a training step on 4096 tokens of the large layer
        _ffn("ffn_train 4096", "ffn_train", 4096, 7168, 2048, "bf16", False),
    ]


def _between(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step, max(-(-lo // step), round(v / step))) * step


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 50


def draw(rng):
    op = rng.choice(("linear", "ffn", "ffn_train"))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        dtype, add = rng.choice(("bf16", "fp16")), rng.random() < 0.5
        if op == "linear":
            gated = rng.random() < 0.5
            N = 2 * _between(rng, 64, 4096) if gated else _between(rng, 128, 8192)
            case = _linear("", _between(rng, 1, 4096), _between(rng, 256, 8192, 16), N, gated, dtype, add)
        else:
            T = _between(rng, 1 if op == "ffn" else 16, 8192)
            case = _ffn("", op, T, _between(rng, 256, 8192, 8), _between(rng, 128, 4096, 8), dtype, add)
            case["add"] = add and op == "ffn"
        if _cost(case) <= most:
            del case["name"]
            return case


def _quantised(w):
    """NVFP4 of an fp32 matrix: codes two to a byte (the even element in the low nibble), block
    scales, global scale."""
    n, k = w.shape
    blocks = w.view(n, k // 16, 16)
    gs = w.abs().amax() / (6.0 * 448.0)
    sf = (blocks.abs().amax(-1) / 6.0 / gs).to(torch.float8_e4m3fn)
    scale = sf.float() * gs
    q = torch.where(scale[..., None] > 0, blocks / scale[..., None], 0.0).view(n, k)
    mids = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=w.device)
    code = torch.bucketize(q.abs(), mids).to(torch.uint8)
    code |= (q < 0).to(torch.uint8) << 3
    return {"w": code[:, 0::2] | (code[:, 1::2] << 4), "w_sf": sf, "w_gs": gs}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale)

    T = case["T"]
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        out = N // 2 if case["gated"] else N
        state = {"case": case, "x": normal(T, K).to(dt), "weight": _quantised(normal(N, K, scale=0.02))}
        state["add"] = normal(T, out).to(dt) if case["add"] else None
        if own:  # the weights as the layer keeps them after loading a model
            state["linear"] = _package().prepare_linear(state["weight"], gated=case["gated"])
        return state
    H, I = case["H"], case["I"]
    state = {"case": case, "x": normal(T, H).to(dt), "w13": normal(2 * I, H, scale=0.02).to(dt),
             "w2": normal(H, I, scale=0.02).to(dt)}
    state["add"] = normal(T, H).to(dt) if case["add"] else None
    if case["op"] == "ffn_train":
        state["dy"] = normal(T, H).to(dt)
        for name in ("x", "w13", "w2"):
            state[name].requires_grad_(True)
    return state


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_linear(state) if op == "linear" else _plain_ffn(state) if op == "ffn" else _plain_train(state)


def _run_own(state):
    pkg = _package()
    op = state["case"]["op"]
    if op == "linear":
        return {"y": pkg.linear_w4(state["x"], state["linear"], add=state["add"])}
    if op == "ffn":
        return {"y": pkg.gated_ffn(state["x"], state["w13"], state["w2"], add=state["add"])}
    leaves = (state["x"], state["w13"], state["w2"])
    y = pkg.gated_ffn(*leaves)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, state["dy"])
    return {"y": y, "dx": dx, "dw13": dw13, "dw2": dw2}


def _plain_linear(state):
    w, x = state["weight"], state["x"]
    grid = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0),
                        device=x.device)
    n, half = w["w"].shape
    codes = torch.stack((w["w"] & 15, w["w"] >> 4), dim=-1).view(n, 2 * half)
    scale = w["w_sf"].float() * w["w_gs"]
    full = (grid[codes.int()].view(n, half // 8, 16) * scale[..., None]).view(n, 2 * half)
    y = x.float() @ full.t()
    if state["case"]["gated"]:
        gate, up = y[:, :n // 2], y[:, n // 2:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    if state["add"] is not None:
        y = y + state["add"].float()
    return {"y": y.to(x.dtype)}


def _plain_ffn(state):
    x, w13, w2 = (state[k].float() for k in ("x", "w13", "w2"))
    ab = x @ w13.t()
    a, b = ab[:, :w2.shape[1]], ab[:, w2.shape[1]:]
    y = (a / (1.0 + torch.exp(-a)) * b) @ w2.t()
    if state["add"] is not None:
        y = y + state["add"].float()
    return {"y": y.to(state["x"].dtype)}


def _plain_train(state):
    dt = state["x"].dtype
    x, w13, w2, dy = (state[k].detach().float() for k in ("x", "w13", "w2", "dy"))
    inner = w2.shape[1]
    ab = x @ w13.t()
    a, b = ab[:, :inner], ab[:, inner:]
    s = 1.0 / (1.0 + torch.exp(-a))
    h = a * s * b
    y = h @ w2.t()
    dh = dy @ w2
    dab = torch.cat((dh * b * (s * (1.0 + a * (1.0 - s))), dh * a * s), dim=1)
    out = {"y": y, "dx": dab @ w13, "dw13": dab.t() @ x, "dw2": dy.t() @ h}
    return {k: v.to(dt) for k, v in out.items()}


def work(case):
    T = case["T"]
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        out = N // 2 if case["gated"] else N
        return {"bytes": N * K // 2 + N * K // 16 + 4 + 2 * T * K + 2 * T * out * (2 if case["add"] else 1),
                "flops": 2 * T * N * K}
    H, I = case["H"], case["I"]
    if case["op"] == "ffn":
        return {"bytes": 6 * H * I + 2 * T * H * (3 if case["add"] else 2), "flops": 6 * T * H * I}
    return {"bytes": 2 * 6 * H * I + 4 * 2 * T * H, "flops": 18 * T * H * I}


def exact(case, seed):
    state = prepare(case, seed)
    silu = torch.nn.functional.silu
    if case["op"] == "linear":
        w = state["weight"]
        byte = w["w"].to(torch.int64)
        code = torch.empty(byte.shape[0], 2 * byte.shape[1], dtype=torch.int64, device=byte.device)
        code[:, 0::2], code[:, 1::2] = byte % 16, byte // 16
        exponent, odd = code % 8 // 2, code % 2
        size = torch.where(exponent == 0, 0.5 * odd, torch.exp2(exponent.double() - 1) * (1.0 + 0.5 * odd))
        value = torch.where(code >= 8, -size, size)
        value *= w["w_sf"].double().repeat_interleave(16, dim=1) * w["w_gs"].double()
        y = torch.einsum("tk,nk->tn", state["x"].double(), value)
        if case["gated"]:
            first, second = y.chunk(2, dim=1)
            y = silu(first) * second
        return {"y": y if state["add"] is None else y + state["add"].double()}
    x, w13, w2 = (state[k].detach().double() for k in ("x", "w13", "w2"))
    if case["op"] == "ffn":
        first, second = torch.nn.functional.linear(x, w13).chunk(2, dim=1)
        y = torch.nn.functional.linear(silu(first) * second, w2)
        return {"y": y if state["add"] is None else y + state["add"].double()}
    for t in (x, w13, w2):
        t.requires_grad_(True)
    first, second = torch.nn.functional.linear(x, w13).chunk(2, dim=1)
    y = torch.nn.functional.linear(silu(first) * second, w2)
    dx, dw13, dw2 = torch.autograd.grad(y, (x, w13, w2), state["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}
