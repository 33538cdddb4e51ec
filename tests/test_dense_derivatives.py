"""Derivatives that the dense operators do not have are refused, not dropped."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from tests import dense_ref as ref

DEV = torch.device("cuda:0")
gpu = pytest.mark.gpu


def linear_arguments(device):
    return {"x": torch.ones((2, 64), dtype=torch.bfloat16, device=device),
            "gs": torch.ones(1, device=device),
            "add": torch.ones((2, 32), dtype=torch.bfloat16, device=device),
            "out": torch.ones((2, 32), dtype=torch.bfloat16, device=device)}


def ffn_arguments(device):
    one = lambda *s: torch.ones(s, dtype=torch.bfloat16, device=device)  # noqa: E731
    return {"x": one(2, 64), "w13": one(144, 64), "w2": one(64, 72), "add": one(2, 64)}


def refused(pkg, call, arguments, which, grad):
    """`call` with a tangent on one argument raises, with gradients on or off."""
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        a = dict(arguments)
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(pkg.MuseError, match="forward-mode") as e:
            call(a)
        assert e.value.code == -1


# On the CPU the device check is taken out: the refusal comes before anything touches a device.
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["x", "gs", "add", "out"])
def test_linear_refuses_tangents(pkg, monkeypatch, which, grad):
    from muse_moe_w4a16_b200 import dense
    monkeypatch.setattr(dense, "_require_cuda", lambda t, name: None)
    state = {"cols": 64, "rows": 32, "n_out": 32, "gated": False, "w": torch.zeros(1024, dtype=torch.uint8)}
    refused(pkg, lambda a: pkg.linear_w4(a["x"], dict(state, w_gs=a["gs"]), add=a["add"], out=a["out"]),
            linear_arguments("cpu"), which, grad)


@pytest.mark.parametrize("which", ["x", "gs", "add", "out"])
def test_linear_refuses_gradients(pkg, monkeypatch, which):
    """Every floating-point tensor of a call, the global scale among them."""
    from muse_moe_w4a16_b200 import dense
    monkeypatch.setattr(dense, "_require_cuda", lambda t, name: None)
    a = linear_arguments("cpu")
    a[which] = a[which].requires_grad_()
    state = {"cols": 64, "rows": 32, "n_out": 32, "gated": False, "w": torch.zeros(1024, dtype=torch.uint8), "w_gs": a["gs"]}
    with pytest.raises(pkg.MuseError, match="gradient") as e:
        pkg.linear_w4(a["x"], state, add=a["add"], out=a["out"])
    assert e.value.code == -1


@gpu
def test_linear_with_a_trained_scale(pkg):
    """A scale that wants a gradient: refused while gradients are on, served without."""
    weight = ref.random_w4(32, 64, 1, DEV)
    x = torch.ones((2, 64), dtype=torch.bfloat16, device=DEV)
    want = pkg.linear_w4(x, pkg.prepare_linear(weight))
    state = pkg.prepare_linear(dict(weight, w_gs=weight["w_gs"].clone().requires_grad_()))
    with pytest.raises(pkg.MuseError):
        pkg.linear_w4(x, state)
    with torch.no_grad():
        assert torch.equal(pkg.linear_w4(x, state), want)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["x", "w13", "w2", "add"])
def test_ffn_refuses_tangents(pkg, monkeypatch, which, grad):
    from muse_moe_w4a16_b200 import dense
    monkeypatch.setattr(dense, "_require_cuda", lambda t, name: None)
    refused(pkg, lambda a: pkg.gated_ffn(**a), ffn_arguments("cpu"), which, grad)


@gpu
@pytest.mark.parametrize("which", ["x", "gs", "add", "out"])
def test_linear_refuses_tangents_on_the_device(pkg, which):
    state = pkg.prepare_linear(ref.random_w4(32, 64, 1, DEV))
    call = lambda a: pkg.linear_w4(a["x"], dict(state, w_gs=a["gs"]), add=a["add"], out=a["out"])  # noqa: E731
    refused(pkg, call, linear_arguments(DEV), which, True)
    with forward_ad.dual_level():   # no tangent, no refusal
        a = linear_arguments(DEV)
        y = call(a)
    assert torch.equal(y, call(linear_arguments(DEV)))


@gpu
@pytest.mark.parametrize("which", ["x", "w13", "w2", "add"])
def test_ffn_refuses_tangents_on_the_device(pkg, which):
    refused(pkg, lambda a: pkg.gated_ffn(**a), ffn_arguments(DEV), which, True)
    with forward_ad.dual_level():
        y = pkg.gated_ffn(**ffn_arguments(DEV))
    assert torch.equal(y, pkg.gated_ffn(**ffn_arguments(DEV)))
    with forward_ad.dual_level(), torch.inference_mode():   # forward mode is off, as in torch
        a = ffn_arguments(DEV)
        assert torch.equal(pkg.gated_ffn(**a), y)
