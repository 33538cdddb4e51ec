"""gated_ffn: refusals (CPU), parity of the block and its gradients with 64 bits (GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests import dense_ref as ref

DEV = torch.device("cuda:0")
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def make(T, H, I, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + T * 31 + H + I)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(dtype).to(DEV)  # noqa: E731
    return r(T, H), r(2 * I, H, scale=H ** -0.5), r(H, I, scale=I ** -0.5), r(T, H), r(T, H)


# ------------------------------------------------------------------ refusals, no device

def test_cpu_tensors_are_refused(pkg):
    z = torch.zeros(16, 8, dtype=torch.bfloat16)
    with pytest.raises(pkg.MuseError) as e:
        pkg.gated_ffn(z[:2], z, z[:8])
    assert e.value.code == -4


@pytest.mark.parametrize("args,code", [((-1, 64, 64, 0), -1), ((1, 0, 64, 0), -1), ((1, 64, 0, 1), -1),
                                       ((1, 60, 64, 0), -2), ((1, 64, 60, 0), -2)])
def test_workspace_size_refuses(pkg, args, code):
    n = ctypes.c_size_t()
    assert pkg.load_library().muse_moe_ffn_workspace_size(*args, ctypes.byref(n)) == code


def test_workspace_size(pkg):
    n = ctypes.c_size_t()
    lib = pkg.load_library()
    assert lib.muse_moe_ffn_workspace_size(0, 64, 64, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.muse_moe_ffn_workspace_size(100, 64, 128, 0, ctypes.byref(n)) == 0 and n.value >= 100 * 128 * 2
    fwd = n.value
    assert lib.muse_moe_ffn_workspace_size(100, 64, 128, 1, ctypes.byref(n)) == 0 and n.value >= fwd + 100 * 256 * 2


def test_entries_refuse_before_any_launch(pkg):
    lib = pkg.load_library()
    good = dict(x=256, ldx=64, dtype=0, tokens=2, hidden=64, inter=64, w13=256, ld13=64, w2=256, ld2=64, add=None,
                ld_add=0, out=256, ab=None, ws=256, bytes=1 << 30, stream=None)
    call = lambda **k: lib.muse_moe_ffn_forward(*{**good, **k}.values())  # noqa: E731
    assert call(tokens=0) == 0
    for bad in (dict(x=None), dict(x=264), dict(ldx=60), dict(ldx=56), dict(dtype=3), dict(w13=None), dict(ld13=63),
                dict(w2=258), dict(ld2=32), dict(add=264, ld_add=64), dict(add=256, ld_add=8), dict(out=None),
                dict(ab=8), dict(ws=None), dict(ws=128)):
        assert call(**bad) == -1, bad
    assert call(bytes=16) == -3
    good = dict(dy=256, ldy=64, x=256, ldx=64, dtype=0, tokens=2, hidden=64, inter=64, w13=256, ld13=64, w2=256,
                ld2=64, ab=256, dx=256, dw13=256, dw2=256, ws=256, bytes=1 << 30, stream=None)
    call = lambda **k: lib.muse_moe_ffn_backward(*{**good, **k}.values())  # noqa: E731
    assert call(dx=None, dw13=None, dw2=None) == 0
    for bad in (dict(tokens=0), dict(dy=None), dict(ldy=60), dict(x=None), dict(w13=None), dict(w2=None), dict(ab=None),
                dict(dx=8), dict(dw13=8), dict(dw2=8), dict(ws=None)):
        assert call(**bad) == -1, bad
    assert call(bytes=16) == -3


# ------------------------------------------------------------------ parity

SIZES = [(1, 8, 8), (1, 128, 64), (2, 72, 200), (7, 264, 136), (8, 1024, 512), (9, 64, 1032), (16, 2048, 768),
         (17, 200, 72), (31, 512, 264), (33, 1000, 128), (64, 128, 1000), (100, 640, 384), (128, 264, 520),
         (129, 1032, 64), (255, 136, 136), (256, 512, 512), (257, 768, 328), (509, 520, 1288), (1025, 256, 320),
         (20, 4104, 2056), (32, 3080, 1368), (40, 8, 8), (600, 2056, 24), (2100, 72, 520)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,I", SIZES)
def test_forward(pkg, T, H, I, dtype):
    x, w13, w2, _, add = make(T, H, I, dtype)
    for extra in (None, add):
        y = pkg.gated_ffn(x, w13, w2, add=extra)
        want, bound = ref.ffn_bounds(x, w13, w2, add=extra)["y"]
        ref.check(y, want, bound, "y")
        ref.check_norm(y, want, dtype, 2, "y")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,I", SIZES)
def test_gradients(pkg, T, H, I, dtype):
    x, w13, w2, dy, add = make(T, H, I, dtype, seed=1)
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2, add)]
    y = pkg.gated_ffn(*leaves[:3], add=leaves[3])
    assert torch.equal(y.detach(), pkg.gated_ffn(x, w13, w2, add=add))
    grads = torch.autograd.grad(y, leaves, dy)
    want = ref.ffn_bounds(x, w13, w2, dy)
    for name, got in zip(("dx", "dw13", "dw2"), grads):
        assert got.dtype == dtype
        ref.check(got, *want[name], name)
        ref.check_norm(got, want[name][0], dtype, 2, name)
    assert torch.equal(grads[3], dy)


@gpu
@pytest.mark.parametrize("T,H,I", [(5, 64, 72), (40, 264, 128), (300, 128, 136)])
def test_gradients_against_differences(pkg, T, H, I):
    """<gradient, v> against a central difference of the 64-bit block along v. The difference is
    off by O(step^2) of the third derivative (1e-8 here); the gradient's elements by their bounds."""
    x, w13, w2, dy, _ = make(T, H, I, torch.float16, seed=3)
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    grads = torch.autograd.grad(pkg.gated_ffn(*leaves), leaves, dy)
    bounds = ref.ffn_bounds(x, w13, w2, dy)
    f = lambda *p: (ref.ffn64(*p) * dy.double()).sum()  # noqa: E731
    for i, name in enumerate(("dx", "dw13", "dw2")):
        v = torch.randn_like(leaves[i], dtype=torch.float64)
        at = [t.double() for t in (x, w13, w2)]
        step = 1e-4
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + step * v, at[i] - step * v
        slope = (f(*plus) - f(*minus)) / (2 * step)
        room = (bounds[name][1] * v.abs()).sum() + 1e-5 * (bounds[name][0] * v).abs().sum()
        assert abs((grads[i].double() * v).sum() - slope) <= room, name


@gpu
@pytest.mark.parametrize("which", range(1, 8))
def test_only_wanted_gradients(pkg, which):
    x, w13, w2, dy, _ = make(48, 256, 128, torch.bfloat16, seed=4)
    full = [t.clone().requires_grad_() for t in (x, w13, w2)]
    want = torch.autograd.grad(pkg.gated_ffn(*full), full, dy)
    some = [t.clone().requires_grad_(bool(which >> i & 1)) for i, t in enumerate((x, w13, w2))]
    pkg.gated_ffn(*some).backward(dy)
    for i, t in enumerate(some):
        assert (t.grad is None) if not which >> i & 1 else torch.equal(t.grad, want[i])


@gpu
def test_gradient_of_the_addend_alone(pkg):
    x, w13, w2, dy, add = make(20, 64, 72, torch.bfloat16)
    leaf = add.clone().requires_grad_()
    y = pkg.gated_ffn(x, w13, w2, add=leaf)
    y.backward(dy)
    assert torch.equal(leaf.grad, dy) and torch.equal(y.detach(), pkg.gated_ffn(x, w13, w2, add=add))
    # one tensor as input and addend: both gradients reach it
    both = x.clone().requires_grad_()
    pkg.gated_ffn(both, w13, w2, add=both).backward(dy)
    only = x.clone().requires_grad_()
    pkg.gated_ffn(only, w13, w2).backward(dy)
    assert torch.equal(both.grad, only.grad + dy)


@gpu
def test_empty(pkg):
    _, w13, w2, _, _ = make(1, 64, 72, torch.bfloat16)
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w13.requires_grad_(), w2.requires_grad_()
    y = pkg.gated_ffn(x, w13, w2)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and not w13.grad.any() and not w2.grad.any()


@gpu
@pytest.mark.parametrize("T", [3, 40, 300])
def test_strides_and_shapes(pkg, T):
    x, w13, w2, dy, add = make(T, 256, 136, torch.bfloat16, seed=5)
    full = [t.clone().requires_grad_() for t in (x, w13, w2)]
    y = pkg.gated_ffn(*full, add=add)
    want = torch.autograd.grad(y, full, dy)

    def strided(t, pad):  # the same values inside a NaN frame, rows `pad` elements apart
        f = torch.full((t.shape[0] + 2, t.shape[1] + pad), float("nan"), dtype=t.dtype, device=DEV)
        v = f[1:-1, pad // 2:pad // 2 + t.shape[1]]
        v.copy_(t)
        return v

    for pad in (16, 6):
        a = [strided(t, pad).detach().requires_grad_() for t in (x, w13, w2)]
        out = pkg.gated_ffn(*a, add=strided(add, pad))
        assert torch.equal(out, y)
        for g, w in zip(torch.autograd.grad(out, a, strided(dy, pad)), want):
            assert torch.equal(g, w)
    t = [v.t().contiguous().t().detach().requires_grad_() for v in (x, w13, w2)]
    out = pkg.gated_ffn(t[0].view(1, T, 256), t[1], t[2], add=add.view(1, T, 256))
    assert out.shape == (1, T, 256) and torch.equal(out[0], y)
    for g, w in zip(torch.autograd.grad(out, t, dy.view(1, T, 256)), want):
        assert torch.equal(g, w)
    # a broadcast dy (as a sum's backward pass gives) and a broadcast x row
    leaf = full[0]
    g1 = torch.autograd.grad(pkg.gated_ffn(leaf, w13, w2).sum(), leaf)[0]
    g2 = torch.autograd.grad(pkg.gated_ffn(leaf, w13, w2), leaf, torch.ones_like(x))[0]
    assert torch.equal(g1, g2)
    one = x[:1].clone().requires_grad_()
    got = torch.autograd.grad(pkg.gated_ffn(one.expand(T, 256), w13, w2), one, dy)[0]
    each = x[:1].expand(T, 256).contiguous().requires_grad_()
    rows = torch.autograd.grad(pkg.gated_ffn(each, w13, w2), each, dy)[0]
    torch.testing.assert_close(got, rows.sum(0, keepdim=True), rtol=0.02, atol=0.05)


@gpu
@pytest.mark.parametrize("T", [2, 40, 300])
def test_non_finite_tokens_stay_in_their_rows(pkg, T):
    x, w13, w2, dy, _ = make(T, 256, 136, torch.float16, seed=6)
    y = pkg.gated_ffn(x, w13, w2)
    z = x.clone()
    z[1] = float("nan")
    got = pkg.gated_ffn(z, w13, w2)
    keep = torch.arange(T, device=DEV) != 1
    assert torch.equal(got[keep], y[keep]) and got[1].isnan().all()


@gpu
def test_extreme_activations(pkg):
    """Gates far out on both sides: silu and its derivative stay finite and keep their limits."""
    T, H, I = 32, 64, 64
    x = torch.zeros((T, H), dtype=torch.bfloat16, device=DEV)
    x[:, 0] = torch.linspace(-300, 300, T, device=DEV)
    w13 = torch.zeros((2 * I, H), dtype=torch.bfloat16, device=DEV)
    w13[:I, 0] = 1.0
    w13[I:, 0] = 0.25
    w2 = torch.eye(H, I, dtype=torch.bfloat16, device=DEV)
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    y = pkg.gated_ffn(*leaves)
    want = ref.ffn64(x, w13, w2)
    torch.testing.assert_close(y.double(), want, rtol=3 * 2.0 ** -8, atol=1e-30)
    l64 = [t.double().requires_grad_() for t in (x, w13, w2)]
    w64 = torch.autograd.grad(ref.ffn64(*l64), l64, torch.ones_like(want))
    g = torch.autograd.grad(y, leaves, torch.ones_like(y))
    for a, b in zip(g, w64):
        assert a.isfinite().all()
        ref.check_norm(a, b, torch.bfloat16, 4)


@gpu
def test_refusals(pkg):
    x, w13, w2, _, _ = make(4, 64, 72, torch.bfloat16)
    for call, code in ((lambda: pkg.gated_ffn(x.float(), w13, w2), -1), (lambda: pkg.gated_ffn(x, w13.half(), w2), -1),
                       (lambda: pkg.gated_ffn(x, w13, w2.cpu()), -1), (lambda: pkg.gated_ffn(x, w13[:-1], w2), -1),
                       (lambda: pkg.gated_ffn(x[:, :56], w13, w2), -1), (lambda: pkg.gated_ffn(x, w13, w2, add=x[:2]), -1),
                       (lambda: pkg.gated_ffn(x, w13[:140], w2[:, :70]), -2),
                       (lambda: pkg.gated_ffn(x[:, :60], w13[:, :60], w2[:60]), -2)):
        with pytest.raises(pkg.MuseError) as e:
            call()
        assert e.value.code == code
    leaf = x.clone().requires_grad_()
    g = torch.autograd.grad(pkg.gated_ffn(leaf, w13, w2).sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu
@pytest.mark.parametrize("T", [1, 24, 300])
def test_graphs_streams_and_repeats(pkg, T):
    """Forward and backward captured and replayed on new contents, two graphs at once, another
    stream: the same bits as the eager call."""
    x, w13, w2, dy, add = make(T, 512, 264, torch.bfloat16, seed=7)

    def step(xs):
        leaves = [t.detach().requires_grad_() for t in (xs, w13, w2)]
        y = pkg.gated_ffn(*leaves, add=add)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(step(x), first):
            assert torch.equal(a, b)
    side.synchronize()
    static = x.clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(static))
        graphs.append(g)
    x2 = torch.randn_like(x)
    want = step(x2)
    static.copy_(x2)
    torch.cuda.synchronize()
    for g, s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
