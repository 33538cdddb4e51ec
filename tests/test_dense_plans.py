"""Every way a dense product is laid out on the chip, against 64 bits: several tiles per group of
CTAs (alternating accumulators), whole tiles with a split tail, K split alone -- the plans of
prompts and training steps, at the smallest sizes that reach them. `test_plan_*` (CPU) holds each
size to the plan that it stands for, so that a changed rule does not drop one from the tests."""

from __future__ import annotations

import pytest
import torch

from tests import dense_ref as ref
from tests.test_gated_ffn import make

DEV = torch.device("cuda:0")
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
PAIRS, SMS = 74, 148


def describe(p: dict) -> str:
    """kernel and layout of a plan in a word or two"""
    if p["kernel"] == 0:
        return "few"
    kernel = {1: "weights", 2: "tokens"}[p["kernel"]]
    if p["splits"] > 1:
        return f"{kernel}, {'tail split' if p['whole'] else 'split'}"
    if p["per_group"] == 1:
        return f"{kernel}, one wave"
    if p["kernel"] == 1 and p["per_group"] == -(-p["tiles"] // SMS):
        return f"{kernel}, several tiles of a CTA"
    return f"{kernel}, several tiles of a pair"


# (kind, tokens, rows, cols): layout
LINEAR = {
    ("linear", 271, 6310, 16): "weights, several tiles of a pair",
    ("linear", 3393, 1286, 1040): "weights, several tiles of a pair",
    ("linear", 4096, 2064, 256): "weights, several tiles of a pair",
    ("linear", 3982, 1054, 64): "weights, several tiles of a CTA",
    ("linear", 2108, 132, 1952): "weights, split",
    ("gated", 271, 6310, 16): "weights, several tiles of a pair",
    ("gated", 3393, 1286, 1040): "weights, several tiles of a pair",
    ("gated", 2000, 4096, 7168): "weights, several tiles of a pair",
    ("gated", 3982, 1054, 64): "weights, several tiles of a CTA",
    ("gated", 2108, 132, 1952): "weights, split",
}

# (tokens, hidden, inter): layouts of the products that the size stands for
FFN = {
    (134, 64, 3120): {"gate": "weights, several tiles of a pair"},
    (200, 4784, 64): {"down": "weights, several tiles of a pair"},
    (35, 1544, 64): {"gate": "tokens, split"},
    (539, 64, 3432): {"gate": "tokens, several tiles of a pair"},
    (543, 6216, 64): {"down": "tokens, several tiles of a pair", "dx": "tokens, several tiles of a pair"},
    (2001, 4096, 1288): {"gate": "weights, several tiles of a pair", "down": "weights, several tiles of a pair",
                         "dx": "tokens, several tiles of a pair", "dw13": "tokens, several tiles of a pair",
                         "dw2": "tokens, several tiles of a pair"},
    (6314, 72, 520): {"dgate": "tokens, several tiles of a pair"},
    (6233, 1632, 272): {"gate": "tokens, tail split"},
    (6266, 560, 1512): {"down": "tokens, tail split"},
    (1261, 848, 3784): {"dgate": "tokens, tail split"},
    (1200, 3808, 432): {"dx": "tokens, tail split"},
    (890, 3792, 560): {"dw13": "tokens, tail split"},
    (1021, 6240, 752): {"dw2": "tokens, tail split"},
    (1501, 7168, 2048): {"gate": "tokens, tail split", "dx": "tokens, tail split", "dw13": "tokens, tail split",
                         "dw2": "tokens, tail split"},
    (4093, 7168, 2048): {"gate": "tokens, tail split", "down": "tokens, several tiles of a pair",
                         "dgate": "tokens, several tiles of a pair"},
}


@pytest.mark.parametrize("case", LINEAR, ids=str)
def test_plan_linear(pkg, case):
    from muse_moe_w4a16_b200 import _lib
    assert describe(_lib.dense_plan(*case)) == LINEAR[case]


@pytest.mark.parametrize("size", FFN, ids=str)
def test_plan_ffn(pkg, size):
    from muse_moe_w4a16_b200 import _lib
    for product, layout in FFN[size].items():
        assert describe(_lib.dense_plan(product, *size)) == layout, product


def test_plan_refusals(pkg):
    from muse_moe_w4a16_b200 import _lib
    for args, code in ((("linear", 0, 8, 16), -1), (("linear", 1, 8, 24), -2), (("gated", 1, 7, 16), -1),
                       (("gate", 0, 64, 64), -1), (("dx", 1, 60, 64), -2), (("dw2", -1, 64, 64), -1),
                       (("linear", (1 << 28) + 1, 8, 16), -2)):
        with pytest.raises(pkg.MuseError) as e:
            _lib.dense_plan(*args)
        assert e.value.code == code, args
    assert pkg.load_library().muse_moe_ffn_plan(6, 1, 64, 64, None) == -1
    assert describe(_lib.dense_plan("linear", 1, 8, 16)) == "few" == describe(_lib.dense_plan("down", 8, 64, 64))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", LINEAR, ids=str)
def test_linear(pkg, case, dtype):
    """All rows, with and without an addend, and the same bits again."""
    kind, T, N, K = case
    gated = kind == "gated"
    weight = ref.random_w4(N, K, T, DEV)
    state = pkg.prepare_linear(weight, gated=gated)
    g = torch.Generator().manual_seed(N)
    x = torch.randn((T, K), generator=g).to(dtype).to(DEV)
    add = torch.randn((T, state["n_out"]), generator=g).to(dtype).to(DEV)
    for extra in (None, add):
        y = pkg.linear_w4(x, state, add=extra)
        ref.check(y, *ref.linear64(x, weight, gated, extra), "y")
        assert torch.equal(pkg.linear_w4(x, state, add=extra), y)
    both = add.clone()
    assert torch.equal(pkg.linear_w4(x, state, add=both, out=both), y)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", FFN, ids=str)
def test_ffn(pkg, size, dtype):
    """The block with and without an addend, and its gradients, all elements."""
    x, w13, w2, dy, add = make(*size, dtype, seed=2)
    want = ref.ffn_bounds(x, w13, w2, dy)
    y = pkg.gated_ffn(x, w13, w2)
    ref.check(y, *want["y"], "y")
    ref.check_norm(y, want["y"][0], dtype, 2, "y")
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    kept = pkg.gated_ffn(*leaves)
    assert torch.equal(kept.detach(), y)
    grads = torch.autograd.grad(kept, leaves, dy)
    for name, got in zip(("dx", "dw13", "dw2"), grads):
        ref.check(got, *want[name], name)
        ref.check_norm(got, want[name][0], dtype, 2, name)
    again = torch.autograd.grad(pkg.gated_ffn(*leaves), leaves, dy)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)
    del want, leaves, grads, again
    ref.check(pkg.gated_ffn(x, w13, w2, add=add), *ref.ffn_bounds(x, w13, w2, add=add)["y"], "y + add")
