"""Weights with very many rows: whatever size the library gives for a prepared weight, it prepares."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests import dense_ref as ref

DEV = torch.device("cuda:0")


def test_sizes_at_the_limits(pkg):
    size = lambda *a: pkg.load_library().muse_moe_linear_prepared_size(*a, ctypes.byref(n))  # noqa: E731
    n = ctypes.c_size_t()
    assert size(1 << 24, 16, 0) == 0 and n.value == (1 << 17) * 9216
    assert size(16, 1 << 24, 0) == 0 and n.value == (1 << 17) * 9216
    assert size((1 << 24) + 1, 16, 0) == -2 and size(16, (1 << 24) + 16, 0) == -2
    # 2^17 row tiles of 2^14 chunks are one tile too many for a launch
    assert size(1 << 24, (1 << 21) - 128, 0) == 0 and size(1 << 24, 1 << 21, 0) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("gated,T", [(False, 2), (False, 20), (True, 2), (True, 20)])
def test_more_than_65535_row_tiles(pkg, gated, T):
    N, K = 65536 * 128 + 2, 16
    weight = ref.random_w4(N, K, 3, DEV)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
    y = pkg.linear_w4(x, pkg.prepare_linear(weight, gated=gated))
    want, bound = ref.linear64(x, weight, gated)
    ref.check(y, want, bound, "y")
