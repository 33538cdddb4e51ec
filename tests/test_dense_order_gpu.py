"""linear_w4 sees its weight as it is at the call's place in the stream, whatever wrote it: also a
kernel that lets its successor start early, as this library's dense products do."""

from __future__ import annotations

import pytest
import torch

from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [1, 12, 70, 400])
def test_weight_written_by_a_product(pkg, T, gated):
    """The prepared bytes are written as a 16-bit output (0 . W + add), and the next launch reads them."""
    N, K = 384, 1024
    states = [pkg.prepare_linear(ref.random_w4(N, K, seed, DEV), gated=gated) for seed in (1, 2)]
    copier = pkg.prepare_linear(ref.random_w4(512, 64, 3, DEV))
    words = [s["w"].view(torch.bfloat16).view(-1, 512) for s in states]
    zeros = torch.zeros((words[0].shape[0], 64), dtype=torch.bfloat16, device=DEV)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
    # what the copies hold (an addition rewrites -0 and NaN patterns) and the products with them
    want = []
    for w in words:
        held = pkg.linear_w4(zeros, copier, add=w)
        torch.cuda.synchronize()
        want.append(pkg.linear_w4(x, dict(states[0], w=held.view(torch.uint8).view(-1))).view(torch.int16).clone())
        torch.cuda.synchronize()
    assert not torch.equal(*want)
    buffer = torch.empty_like(words[0])
    state = dict(states[0], w=buffer.view(torch.uint8).view(-1))
    outs = []
    torch.cuda.synchronize()
    for i in range(40):
        pkg.linear_w4(zeros, copier, add=words[i % 2], out=buffer)
        outs.append(pkg.linear_w4(x, state))
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        assert torch.equal(got.view(torch.int16), want[i % 2]), i


@pytest.mark.parametrize("T", [1, 12, 70, 400])
def test_prepare_and_call_at_once(pkg, T):
    """prepare_linear with the product right behind it, over memory that held another weight."""
    N, K = 640, 2048
    weights = [ref.random_w4(N, K, seed, DEV) for seed in (4, 5)]
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
    want = []
    for w in weights:
        state = pkg.prepare_linear(w)
        torch.cuda.synchronize()
        want.append(pkg.linear_w4(x, state))
        torch.cuda.synchronize()
    outs = []
    for i in range(40):   # the state is freed at once: the next one's memory is this one's
        outs.append(pkg.linear_w4(x, pkg.prepare_linear(weights[i % 2])))
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        assert torch.equal(got, want[i % 2]), i


@pytest.mark.parametrize("T", [1, 12, 70, 400])
def test_scale_rewritten_in_place(pkg, T):
    """The global scale changes between calls, with nothing between the launches."""
    state = pkg.prepare_linear(ref.random_w4(384, 1024, 7, DEV))
    x = torch.randn((T, 1024), generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
    first = state["w_gs"].clone()
    scales = [first, first * 4]
    want = []
    for s in scales:
        torch.cuda.synchronize()
        want.append(pkg.linear_w4(x, dict(state, w_gs=s)))
    # a factor of four is exact, in fp32 and in bf16
    assert torch.equal(want[1], want[0] * 4)
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        torch.mul(first, 4.0 if i % 2 else 1.0, out=state["w_gs"])
        outs += [pkg.linear_w4(x, state), pkg.linear_w4(x, state)]
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        assert torch.equal(got, want[i // 2 % 2]), i
