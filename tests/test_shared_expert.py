"""The dense operators as a layer uses them: a shared expert beside the routed ones, in 4 and in 16
bits, on the routed output, in one captured step; and a shared expert trained in 16 bits."""

from __future__ import annotations

import pytest
import torch

from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def layer(pkg):
    from muse_moe_w4a16_b200 import synth
    shape = synth.MoEShape(256, 8, 256, 256, local_start=0, local_count=32, router="reference-normal")
    w = synth.reference_weights(shape, device="cpu")
    return shape, pkg.prepare({k: v.to(DEV) for k, v in w.items()})


def inputs(shape, T, seed):
    from muse_moe_w4a16_b200 import synth
    x, scores = synth.reference_scores(shape, T, seed=seed)
    return x.to(DEV), scores.to(DEV), synth.make_config(shape, T)


def quantised(w):
    from muse_moe_w4a16_b200 import synth
    packed, sf, gs = synth.quantize_nvfp4(w)
    return {"w": packed, "w_sf": sf, "w_gs": gs}


@pytest.mark.parametrize("T", [1, 12, 48, 300])
def test_step_with_a_shared_expert(pkg, layer, T):
    """router -> routed experts -> 4-bit and 16-bit shared expert on top, eager and captured; the parts
    on their own give the same bits, and the sum is the 64-bit one within the operators' bounds."""
    shape, routed = layer
    H, I = 256, 200
    x, scores, cfg = inputs(shape, T, 5)
    g = torch.Generator().manual_seed(T)
    w13, w2 = torch.randn((2 * I, H), generator=g) * 0.05, torch.randn((H, 208), generator=g) * 0.05
    w2[:, I:] = 0    # K is a multiple of 16: the inner size is padded with zero weights
    q13, q2 = ({k: v.to(DEV) for k, v in quantised(w).items()} for w in (w13, w2))
    s13, s2 = pkg.prepare_linear(q13, gated=True), pkg.prepare_linear(q2)
    f13, f2 = w13.to(torch.bfloat16).to(DEV), w2[:, :I].to(torch.bfloat16).to(DEV)
    inner = torch.zeros((T, 208), dtype=torch.bfloat16, device=DEV)

    def step():
        ids, wts = pkg.route_topk(scores, 8)
        y = pkg.kernel_fn({"hidden_states": x, "topk_ids": ids, "topk_weights": wts, "config": cfg}, routed)
        inner[:, :I] = pkg.linear_w4(x, s13)
        return y, pkg.linear_w4(inner, s2, add=y), pkg.gated_ffn(x, f13, f2, add=y)

    with torch.no_grad():
        y, four, sixteen = step()
        h, bound = ref.linear64(x, q13, True)
        ref.check(inner[:, :I], h, bound, "inner")
        ref.check(four, *ref.linear64(inner, q2, False, y), "4-bit shared expert")
        ref.check(sixteen, *ref.ffn_bounds(x, f13, f2, add=y)["y"], "16-bit shared expert")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, (y, four, sixteen)):
        assert torch.equal(a, b)


def test_shared_expert_gradients_through_the_sum(pkg, layer):
    """The shared expert's gradients with the routed output as its addend, which gets dy."""
    shape, routed = layer
    x, scores, cfg = inputs(shape, 40, 6)
    ids, wts = pkg.route_topk(scores, 8)
    y = pkg.kernel_fn({"hidden_states": x, "topk_ids": ids, "topk_weights": wts, "config": cfg}, routed)
    g = torch.Generator().manual_seed(1)
    w13, w2 = (torch.randn(s, generator=g).mul(0.05).to(torch.bfloat16).to(DEV) for s in ((272, 256), (256, 136)))
    dy = torch.randn(x.shape, generator=g).to(torch.bfloat16).to(DEV)
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2, y)]
    pkg.gated_ffn(*leaves[:3], add=leaves[3]).backward(dy)
    want = ref.ffn_bounds(x, w13, w2, dy)
    for name, leaf in zip(("dx", "dw13", "dw2"), leaves):
        ref.check(leaf.grad, *want[name], name)
    assert torch.equal(leaves[3].grad, dy)


def test_trained_in_sixteen_bits_served_in_four(pkg):
    """One step of plain descent on the block's weights, then the same weights quantised: the 4-bit pair
    computes the product of the quantised weights, the 16-bit block that of the weights."""
    g = torch.Generator().manual_seed(2)
    T, H, I = 24, 256, 128
    x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(DEV)
    w13 = (torch.randn((2 * I, H), generator=g) * 0.06).to(torch.bfloat16).to(DEV).requires_grad_()
    w2 = (torch.randn((H, I), generator=g) * 0.06).to(torch.bfloat16).to(DEV).requires_grad_()
    pkg.gated_ffn(x, w13, w2).float().square().mean().backward()
    with torch.no_grad():
        for w in (w13, w2):
            assert w.grad.isfinite().all() and w.grad.any()
            w -= 0.1 * w.grad
        ref.check(pkg.gated_ffn(x, w13, w2), *ref.ffn_bounds(x, w13, w2)["y"], "16 bits")
        q13, q2 = quantised(w13.float()), quantised(w2.float())
        h = pkg.linear_w4(x, pkg.prepare_linear(q13, gated=True))
        ref.check(h, *ref.linear64(x, q13, True), "4 bits, inner")
        ref.check(pkg.linear_w4(h, pkg.prepare_linear(q2)), *ref.linear64(h, q2, False), "4 bits")


@pytest.mark.parametrize("T", [2, 14, 70, 300])
def test_long_chains_on_two_streams(pkg, T):
    """Hundreds of dependent calls with nothing between them, their temporaries' memory handed from call
    to call, in place on an addend, on two streams at once: every repeat gives the first one's bits."""
    H, I = 384, 256
    g = torch.Generator().manual_seed(T)
    q1 = quantised(torch.randn((2 * I, H), generator=g) * H ** -0.5)
    q2 = quantised(torch.randn((H, I), generator=g) * I ** -0.5)
    s13 = pkg.prepare_linear({k: v.to(DEV) for k, v in q1.items()}, gated=True)
    s2 = pkg.prepare_linear({k: v.to(DEV) for k, v in q2.items()})
    f13 = (torch.randn((2 * I, H), generator=g) * H ** -0.5).to(torch.bfloat16).to(DEV)
    f2 = (torch.randn((H, I), generator=g) * I ** -0.5).to(torch.bfloat16).to(DEV)
    x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(DEV)

    @torch.no_grad()
    def chain():
        y = x.clone()
        for _ in range(4):
            pkg.linear_w4(pkg.linear_w4(y, s13), s2, add=y, out=y)
            y = pkg.gated_ffn(y, f13, f2, add=y)
            y = y / y.float().square().mean().sqrt().to(y.dtype)
        return y

    def gradients():
        leaves = [t.detach().requires_grad_() for t in (x, f13, f2)]
        return torch.autograd.grad(pkg.gated_ffn(*leaves), leaves, x)

    want, want_g = chain(), gradients()
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((chain(), gradients()))
    torch.cuda.synchronize()
    for y, grads in outs:
        assert torch.equal(y, want)
        for a, b in zip(grads, want_g):
            assert torch.equal(a, b)
