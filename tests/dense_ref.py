"""Plain 64-bit forms of the dense operators and the bounds their tests use.

u = finfo(dtype).eps / 2 is half a step of a 16-bit rounding, relative to the value. A product's
fp32 sum of K terms is off by at most (K / 8 + 32) * 2^-23 * sum |terms|: the tensor core adds at
least eight products per accumulation (at most K / 8 accumulations in a row) and each, like each of
the at most 32 further additions across warps, ranks and splits, loses at most one fp32 step
(2^-23, as a tensor core may truncate) of a sum that is at most sum |terms|.
"""

from __future__ import annotations

import torch


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def sum_error(k: int) -> float:
    return (k / 8 + 32) * 2.0 ** -23


# __expf, the division and the products of silu and its derivative: each within 2^-21 of its value
# for the arguments tested (|a| < 64: __expf's error is 2 + floor(1.16 |a|) steps of 2^-23, which at
# |a| = 64 is 76 steps, under 2^-16; it is the largest of the terms).
ACTIVATION = 2.0 ** -16


def dequant64(w: torch.Tensor, sf: torch.Tensor, gs: torch.Tensor) -> torch.Tensor:
    code = torch.stack((w & 15, w >> 4), -1).flatten(-2).to(torch.int64)
    grid = torch.tensor((0, .5, 1, 1.5, 2, 3, 4, 6), dtype=torch.float64, device=w.device)
    val = grid[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    scale = sf.view(torch.float8_e4m3fn).double().repeat_interleave(16, dim=1)
    return val * scale * gs.double()


def random_w4(n: int, k: int, seed: int, dev="cpu") -> dict:
    """Every code and a wide range of scales (zero and the smallest subnormal among them)."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    sf = torch.exp2(torch.randint(-6, 5, (n, k // 16), generator=g).float()) * (1 + torch.rand((n, k // 16), generator=g))
    sf = sf.to(torch.float8_e4m3fn)
    sf.view(torch.uint8)[0, 0] = 1
    sf.view(torch.uint8)[-1, -1] = 0
    return {"w": w.to(dev), "w_sf": sf.to(dev), "w_gs": torch.tensor(0.0023, device=dev)}


def linear64(x, weight, gated: bool, add=None):
    """(y, bound): the product in 64 bits and how far a kernel's 16-bit result may be from it."""
    full = dequant64(weight["w"], weight["w_sf"], weight["w_gs"])
    u, k = half_step(x.dtype), full.shape[1]
    x64 = x.double()
    y = x64 @ full.t()
    err = sum_error(k) * (x64.abs() @ full.abs().t())
    if gated:
        a, b = y.chunk(2, dim=-1)
        ea, eb = err.chunk(2, dim=-1)
        y = a * torch.sigmoid(a) * b
        # |silu'| <= 1.1
        err = 1.1 * ea * (b.abs() + eb) + (a * torch.sigmoid(a)).abs() * eb + ACTIVATION * y.abs()
    if add is not None:
        y = y + add.double()
        err = err + 2.0 ** -23 * (y.abs() + err)
    # one rounding to 16 bits, of at least the type's smallest subnormal step
    return y, err + u * (y.abs() + err) + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps


def ffn64(x, w13, w2, add=None):
    a, b = (x.double() @ w13.double().t()).chunk(2, dim=-1)
    y = (a * torch.sigmoid(a) * b) @ w2.double().t()
    return y if add is None else y + add.double()


def ffn_bounds(x, w13, w2, dy=None, add=None):
    """64-bit y (and dx, dw13, dw2 if dy is given) with elementwise bounds, {name: (value, bound)}.
    The 16-bit roundings counted: h, da, db (operands) and each result."""
    u = half_step(x.dtype)
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    x, w13, w2 = x.double(), w13.double(), w2.double()
    T, H = x.shape
    inner = w2.shape[1]
    ab = x @ w13.t()
    eab = sum_error(H) * (x.abs() @ w13.abs().t())
    (a, b), (ea, eb) = ab.chunk(2, dim=-1), eab.chunk(2, dim=-1)
    s = torch.sigmoid(a)
    h = a * s * b
    eh = 1.1 * ea * (b.abs() + eb) + (a * s).abs() * eb + ACTIVATION * h.abs()
    eh = eh + u * (h.abs() + eh) + tiny

    def product(p, ep, q, k):  # p @ q with p off by ep, then one rounding
        v = p @ q
        e = ep @ q.abs() + sum_error(k) * ((p.abs() + ep) @ q.abs())
        return v, e

    def rounded(v, e):
        return v, e + u * (v.abs() + e) + tiny

    y, ey = product(h, eh, w2.t(), inner)
    if add is not None:
        y = y + add.double()
        ey = ey + 2.0 ** -23 * (y.abs() + ey)
    out = {"y": rounded(y, ey)}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ w2
    edh = sum_error(H) * (dy.abs() @ w2.abs())
    ds = s * (1 + a * (1 - s))
    da, db = dh * b * ds, dh * a * s
    # |silu''| <= 0.5
    eda = edh * b.abs() * 1.1 + dh.abs() * (eb * 1.1 + b.abs() * 0.5 * ea) + ACTIVATION * (dh * b).abs()
    edb = edh * (a * s).abs() + dh.abs() * 1.1 * ea + ACTIVATION * db.abs()
    dab = torch.cat((da, db), dim=1)
    edab = torch.cat((eda, edb), dim=1) * 1.01   # second-order terms
    edab = edab + u * (dab.abs() + edab) + tiny
    out["dx"] = rounded(*product(dab, edab, w13, 2 * inner))
    out["dw13"] = rounded(*product(dab.t(), edab.t(), x, T))
    v, e = product(h.t(), eh.t(), dy, T)
    out["dw2"] = rounded(v.t(), e.t())
    return out


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst at " \
        f"{torch.nonzero(bad)[0].tolist()}: got {got[tuple(torch.nonzero(bad)[0])].item()}, " \
        f"want {want[tuple(torch.nonzero(bad)[0])].item()} +- {bound[tuple(torch.nonzero(bad)[0])].item()}"


def check_norm(got: torch.Tensor, want: torch.Tensor, dtype: torch.dtype, roundings: int, what: str = "") -> None:
    """Independent roundings, each at most u of its value: their combined 2-norm is at most
    u * sqrt(roundings) of the result's (their root mean square is below u / sqrt 3, which leaves
    room for the fp32 sums)."""
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel <= half_step(dtype) * roundings ** 0.5, f"{what}: relative 2-norm error {rel:.3g}"
