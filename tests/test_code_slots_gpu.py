"""Weight slots of the expert GEMM go back to the copies only after their values were used: a
copy that overtook the reads would change some rows of some repeats. Many tokens, with the
epilogue's accesses and another stream's copies filling the memory pipelines, must repeat their
bits."""

from __future__ import annotations

import pytest
import torch

from oracle import moe_oracle as orc
from tests import torch_ref
from tests.gpu_util import bits

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("T,top_k,H,I", [(1, 2, 1024, 512), (24, 4, 1024, 512), (700, 4, 1024, 512),
                                         (9000, 4, 1024, 512), ((1 << 17) + 77, 4, 1024, 512)])
def test_routed_layer_repeats_under_memory_traffic(pkg, T, top_k, H, I):
    from muse_moe_w4a16_b200 import _lib, synth
    shape = synth.MoEShape(16, top_k, H, I, router="zipf")
    w = synth.baseline_weights(shape, seed=11, device="cuda")
    state = pkg.prepare(w)
    data = synth.baseline_input(shape, T, seed=T, device="cuda")
    alone = pkg.kernel_fn(data, state)
    torch.cuda.synchronize()
    rows = torch.linspace(0, T - 1, min(T, 64), device=DEV).long()
    want = torch_ref.layer(data["hidden_states"][rows], data["topk_ids"][rows], data["topk_weights"][rows], w, 0, 16, I)
    ok, msg, err, _ = orc.compare(bits(alone[rows]), bits(want), 1.5e-2)
    assert ok and err < 5e-3, msg

    side = torch.cuda.Stream()
    a = torch.zeros(256 << 20, dtype=torch.uint8, device=DEV)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    outs = []
    for _ in range(6):
        with torch.cuda.stream(side):
            for _ in range(8):
                b.copy_(a)
        outs.append(pkg.kernel_fn(data, state))
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for i, out in enumerate(outs):
        assert torch.equal(out.view(torch.int16), alone.view(torch.int16)), i
