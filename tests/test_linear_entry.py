"""linear_w4's C entry refuses pointers that a kernel could only fault on, before any launch."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("bad", [dict(gs=258), dict(out=257), dict(add=257, ld_add=32), dict(wp=264)])
def test_misaligned_pointers(pkg, bad):
    good = dict(x=256, ldx=64, dtype=0, tokens=2, rows=32, cols=64, gated=0, wp=256, gs=256, add=None, ld_add=0, out=256,
                ldo=32, stream=None)
    assert pkg.load_library().muse_moe_linear_w4(*{**good, **bad}.values()) == -1
