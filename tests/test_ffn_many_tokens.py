"""gated_ffn with a million tokens: element offsets past 32 bits in every tensor of the tokens, sums of
the weights' gradients over all of them, and the same bits from a repeat."""

from __future__ import annotations

import pytest
import torch

from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_a_million_tokens(pkg):
    T, H, I = (1 << 20) + 77, 2064, 1032
    g = torch.Generator(device=DEV).manual_seed(3)
    normal = lambda *s, scale=1.0: (torch.randn(s, generator=g, device=DEV, dtype=torch.float32) * scale).bfloat16()  # noqa: E731
    x, dy, add = (torch.empty((T, H), dtype=torch.bfloat16, device=DEV).normal_(generator=g) for _ in range(3))
    w13, w2 = normal(2 * I, H, scale=H ** -0.5), normal(H, I, scale=I ** -0.5)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    y = pkg.gated_ffn(*leaves, add=add)
    grads = torch.autograd.grad(y, leaves, dy)
    x, w13, w2, y = (t.detach() for t in (*leaves, y))
    assert torch.equal(pkg.gated_ffn(x, w13, w2, add=add), y)
    for first in (0, T // 2, T - 40):
        rows = slice(first, first + 40)
        b = ref.ffn_bounds(x[rows], w13, w2, dy[rows], add=add[rows])
        ref.check(y[rows], *b["y"], f"y from {first}")
        ref.check(grads[0][rows], *b["dx"], f"dx from {first}")
    # the weights' gradients: 64-bit sums over chunks of tokens. Their fp32 sums of T terms have the loose
    # worst-case bound, so the 2-norm is held to the roundings' as well.
    want = {"dw13": 0.0, "dw2": 0.0}
    for first in range(0, T, 1 << 17):
        rows = slice(first, first + (1 << 17))
        xs, dys = x[rows].double(), dy[rows].double()
        a, b = (xs @ w13.double().t()).chunk(2, dim=-1)
        s = torch.sigmoid(a)
        dh = dys @ w2.double()
        want["dw2"] = want["dw2"] + dys.t() @ (a * s * b)
        dab = torch.cat((dh * b * s * (1 + a * (1 - s)), dh * a * s), dim=1)
        want["dw13"] = want["dw13"] + dab.t() @ xs
        del a, b, s, dh, dab, xs, dys
    for name, got in zip(("dw13", "dw2"), grads[1:]):
        ref.check_norm(got, want[name], torch.bfloat16, 2, name)
    again = torch.autograd.grad(pkg.gated_ffn(*leaves, add=add), leaves, dy)
    for got, first in zip(again, grads):
        assert torch.equal(got, first)
