"""linear_w4: refusals (CPU) and parity with a 64-bit product (GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests import dense_ref as ref

DEV = torch.device("cuda:0")
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


# ------------------------------------------------------------------ refusals, no device

def test_cpu_tensors_are_refused(pkg):
    with pytest.raises(pkg.MuseError) as e:
        pkg.prepare_linear(ref.random_w4(32, 64, 0))
    assert e.value.code == -4
    with pytest.raises(pkg.MuseError) as e:
        pkg.linear_w4(torch.zeros(2, 64, dtype=torch.bfloat16), {})
    assert e.value.code == -4


@pytest.mark.parametrize("rows,cols,gated,code", [(0, 64, 0, -1), (8, 0, 0, -1), (7, 64, 1, -1), (8, 64, 2, -1),
                                                  (8, 24, 0, -2), (1 << 25, 64, 0, -2)])
def test_prepared_size_refuses(pkg, rows, cols, gated, code):
    n = ctypes.c_size_t()
    assert pkg.load_library().muse_moe_linear_prepared_size(rows, cols, gated, ctypes.byref(n)) == code


@pytest.mark.parametrize("rows,cols,gated,n", [(1, 16, 0, 128 * 128), (128, 128, 0, 128 * 128), (129, 144, 0, 256 * 256),
                                               (2, 16, 1, 128 * 128), (130, 16, 1, 256 * 128)])
def test_prepared_size(pkg, rows, cols, gated, n):
    size = ctypes.c_size_t()
    assert pkg.load_library().muse_moe_linear_prepared_size(rows, cols, gated, ctypes.byref(size)) == 0
    assert size.value == n // 2 + n // 16


def test_entry_refuses_before_any_launch(pkg):
    lib = pkg.load_library()
    call = lambda **k: lib.muse_moe_linear_w4(*[{**dict(  # noqa: E731
        x=256, ldx=64, dtype=0, tokens=2, rows=32, cols=64, gated=0, wp=256, gs=256, add=None, ld_add=0,
        out=256, ldo=32, stream=None), **k}[n] for n in ("x", "ldx", "dtype", "tokens", "rows", "cols", "gated", "wp",
                                                        "gs", "add", "ld_add", "out", "ldo", "stream")])
    assert call(tokens=0) == 0
    for bad in (dict(tokens=-1), dict(dtype=2), dict(x=None), dict(wp=None), dict(gs=None), dict(out=None),
                dict(x=264), dict(ldx=68), dict(ldx=56), dict(ldo=31), dict(add=256, ld_add=31)):
        assert call(**bad) == -1, bad
    assert call(cols=40) == -2
    assert call(tokens=(1 << 28) + 1) == -2


# ------------------------------------------------------------------ parity

def run(pkg, T, N, K, gated, dtype, with_add, seed=0):
    weight = ref.random_w4(N, K, seed, DEV)
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn((T, K), generator=g).to(dtype).to(DEV)
    add = torch.randn((T, N // 2 if gated else N), generator=g).to(dtype).to(DEV) if with_add else None
    state = pkg.prepare_linear(weight, gated=gated)
    y = pkg.linear_w4(x, state, add=add)
    want, bound = ref.linear64(x, weight, gated, add)
    assert y.dtype == dtype and y.shape == want.shape
    ref.check(y, want, bound, f"T={T} N={N} K={K}")
    return x, state, add, y


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,K,gated,add", [
    (1, 1, 16, False, False), (1, 2, 16, True, True), (1, 128, 128, False, False), (1, 256, 2048, True, False),
    (2, 129, 144, False, True), (3, 34, 1008, True, True), (4, 512, 4096, False, False), (5, 130, 272, True, False),
    (8, 1001, 1008, False, True), (9, 200, 528, False, False), (13, 384, 2048, False, True), (16, 254, 400, True, False),
    (17, 640, 1024, False, False), (31, 66, 80, True, True), (32, 1024, 512, True, False), (33, 300, 336, False, True),
    (64, 128, 7168, False, False), (77, 1001, 1008, False, True), (128, 258, 640, True, False),
    (129, 96, 2064, False, False), (200, 510, 256, True, True), (257, 130, 128, False, False)])
def test_parity(pkg, T, N, K, gated, add, dtype):
    run(pkg, T, N, K, gated, dtype, add, seed=T * 31 + N)


@gpu
@pytest.mark.parametrize("T,N,K,gated", [(513, 1001, 1008, False), (1000, 1288, 2048, True), (2049, 640, 528, False),
                                         (2500, 66, 4112, True), (4096, 16, 16, False)])
def test_parity_many_tokens(pkg, T, N, K, gated):
    run(pkg, T, N, K, gated, torch.bfloat16, True, seed=T)


@gpu
def test_every_code_and_scale_decodes(pkg):
    """One-hot rows of x read single weights back: all 16 codes with every finite scale."""
    K, N = 128, 256
    code = torch.arange(16, dtype=torch.uint8).repeat(N * K // 16).view(N, K)
    w = (code[:, 0::2] | (code[:, 1::2] << 4)).to(DEV)
    byte = torch.arange(N, dtype=torch.uint8).view(N, 1).repeat(1, K // 16)
    byte[(byte & 0x7F) == 0x7F] = 0
    weight = {"w": w, "w_sf": byte.view(torch.float8_e4m3fn).to(DEV), "w_gs": torch.ones((), device=DEV)}
    state = pkg.prepare_linear(weight)
    full = ref.dequant64(w, weight["w_sf"], weight["w_gs"])
    for dtype in DTYPES:
        for T in (16, 128):
            x = torch.eye(K, dtype=dtype, device=DEV)[:T]
            y = pkg.linear_w4(x, state)
            assert torch.equal(y.double(), full.t()[:T].to(dtype).double()), (dtype, T)


@gpu
@pytest.mark.parametrize("T", [3, 40, 300])
def test_strides_shapes_and_out(pkg, T):
    x, state, add, y = run(pkg, T, 300, 512, False, torch.bfloat16, True, seed=5)
    wide = torch.full((T, 512 + 24), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, 8:520] = x
    wide_add = torch.full((T, 333), float("nan"), dtype=x.dtype, device=DEV)
    wide_add[:, 3:303] = add
    assert torch.equal(pkg.linear_w4(wide[:, 8:520], state, add=wide_add[:, 3:303]), y)
    assert torch.equal(pkg.linear_w4(x.t().contiguous().t(), state, add=add.t().contiguous().t()), y)
    odd = torch.empty(T * 512 + 1, dtype=x.dtype, device=DEV)[1:].view(T, 512).copy_(x)
    out = torch.full((T + 2, 300), 7.0, dtype=x.dtype, device=DEV)
    got = pkg.linear_w4(odd.view(1, T, 512), state, add=add.view(1, T, 300), out=out[1:T + 1].view(1, T, 300))
    assert got.shape == (1, T, 300) and torch.equal(out[1:T + 1], y)
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    # out may be add itself, and overlaps nothing else
    both = add.clone()
    assert pkg.linear_w4(x, state, add=both, out=both) is both and torch.equal(both, y)
    room = torch.empty((T + 1, 300), dtype=x.dtype, device=DEV)
    room[:-1] = add
    for bad in (lambda: pkg.linear_w4(x, state, add=room[:-1], out=room[1:]),
                lambda: pkg.linear_w4(x, state, out=x.view(-1)[:T * 300].view(T, 300))):
        with pytest.raises(pkg.MuseError):
            bad()
    assert torch.equal(pkg.linear_w4(x[0], state, add=add[0]), y[0]) or T > 8   # (fewer rows, another kernel)
    assert pkg.linear_w4(x[0], state).shape == (300,)
    one = x[:1].expand(T, 512)
    assert torch.equal(pkg.linear_w4(one, state), pkg.linear_w4(one.contiguous(), state))


@gpu
@pytest.mark.parametrize("T", [1, 20, 300])
def test_non_finite_tokens_stay_in_their_rows(pkg, T):
    x, state, _, y = run(pkg, T, 200, 1008, False, torch.float16, False, seed=9)
    if T > 1:
        z = x.clone()
        z[1] = float("nan")
        got = pkg.linear_w4(z, state)
        keep = torch.arange(T, device=DEV) != 1
        assert torch.equal(got[keep], y[keep]) and got[1].isnan().all()
    x[0, 0] = float("inf")
    assert not pkg.linear_w4(x, state)[0].isfinite().all()


@gpu
def test_empty(pkg):
    state = pkg.prepare_linear(ref.random_w4(64, 64, 1, DEV), gated=True)
    assert pkg.linear_w4(torch.empty((0, 64), dtype=torch.float16, device=DEV), state).shape == (0, 32)
    assert pkg.linear_w4(torch.empty((2, 0, 64), dtype=torch.float16, device=DEV), state).shape == (2, 0, 32)


@gpu
def test_refusals(pkg):
    weight = ref.random_w4(64, 64, 1, DEV)
    state = pkg.prepare_linear(weight)
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device=DEV)
    half = torch.zeros((2, 64), dtype=torch.float16, device=DEV)
    for call in (lambda: pkg.linear_w4(x.float(), state), lambda: pkg.linear_w4(x[:, :48], state),
                 lambda: pkg.linear_w4(x, state, add=half), lambda: pkg.linear_w4(x, state, add=x[:1]),
                 lambda: pkg.linear_w4(x, state, add=x.cpu()), lambda: pkg.linear_w4(x, state, out=half),
                 lambda: pkg.linear_w4(x, state, out=x.t().contiguous().t()),
                 lambda: pkg.linear_w4(x.clone().requires_grad_(), state),
                 lambda: pkg.prepare_linear(dict(weight, w_sf=weight["w_sf"][:, :2])),
                 lambda: pkg.prepare_linear(dict(weight, w=weight["w"][:63], w_sf=weight["w_sf"][:63]), gated=True),
                 lambda: pkg.prepare_linear(dict(weight, w=weight["w"][:, :4], w_sf=weight["w_sf"][:, :1])),
                 lambda: pkg.prepare_linear(dict(weight, w_gs=torch.ones(2, device=DEV)))):
        with pytest.raises(pkg.MuseError) as e:
            call()
        assert e.value.code == -1
    with torch.no_grad():
        pkg.linear_w4(x.clone().requires_grad_(), state)


@gpu
@pytest.mark.parametrize("T", [1, 12, 70, 400])
def test_graph_stream_and_repeat(pkg, T):
    """Captured and replayed on new contents, on another stream, twice at once: the same bits."""
    x, state, add, y = run(pkg, T, 384, 1024, True, torch.bfloat16, True, seed=2)
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(pkg.linear_w4(static, state, add=add), y)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.linear_w4(static, state, add=add))
        graphs.append(g)
    x2 = torch.randn_like(x)
    want = pkg.linear_w4(x2, state, add=add)
    static.copy_(x2)
    torch.cuda.synchronize()
    for g, s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@gpu
@pytest.mark.parametrize("T", [1, 12, 70, 400])
def test_weights_rewritten_in_place(pkg, T):
    """A kernel rewrites the prepared weight between calls, with nothing between the launches: each call
    sees the weight as it is at its place in the stream."""
    x, state, _, y = run(pkg, T, 384, 1024, True, torch.bfloat16, False, seed=5)
    other = pkg.prepare_linear(ref.random_w4(384, 1024, 6, DEV), gated=True)
    z = pkg.linear_w4(x, dict(other, w_gs=state["w_gs"]))
    flip = state["w"] ^ other["w"]
    torch.cuda.synchronize()
    outs = []
    for _ in range(40):
        state["w"].bitwise_xor_(flip)
        outs += [pkg.linear_w4(x, state), pkg.linear_w4(x, state)]
    torch.cuda.synchronize()
    assert not torch.equal(y, z)
    for i, got in enumerate(outs):
        assert torch.equal(got, y if i // 2 % 2 else z), i


@gpu
def test_out_and_autograd(pkg):
    """A leaf that wants a gradient is refused as out; writing over what a backward pass keeps is noticed."""
    state = pkg.prepare_linear(ref.random_w4(64, 64, 1, DEV))
    x = torch.ones((2, 64), dtype=torch.bfloat16, device=DEV)
    out = torch.ones_like(x)
    leaf = torch.ones_like(x).requires_grad_()
    with pytest.raises(pkg.MuseError) as e:
        pkg.linear_w4(x, state, out=leaf)
    assert e.value.code == -1
    y = leaf * out
    pkg.linear_w4(x, state, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.no_grad():
        pkg.linear_w4(x, state, out=leaf)
    assert torch.equal(out, leaf)


@gpu
def test_scale_on_another_device_is_refused(pkg):
    state = pkg.prepare_linear(ref.random_w4(64, 64, 1, DEV))
    with pytest.raises(pkg.MuseError) as e:
        pkg.linear_w4(torch.zeros((2, 64), dtype=torch.bfloat16, device=DEV), dict(state, w_gs=state["w_gs"].cpu()))
    assert e.value.code == -1


@gpu
def test_a_million_tokens_repeat(pkg):
    """Offsets past 32 bits, and the same bits from repeats and in place on the addend: copies and waits
    take longest at this size."""
    T, N, K = (1 << 20) + 77, 2064, 2048
    weight = ref.random_w4(N, K, 1, DEV)
    state = pkg.prepare_linear(weight)
    x = torch.randn((T, K), dtype=torch.bfloat16, device=DEV)
    add = torch.randn((T, N), dtype=torch.bfloat16, device=DEV)
    y = pkg.linear_w4(x, state, add=add)
    for _ in range(3):
        assert torch.equal(pkg.linear_w4(x, state, add=add), y)
    for first in (0, T // 2, T - 40):
        rows = slice(first, first + 40)
        ref.check(y[rows], *ref.linear64(x[rows], weight, False, add[rows]), f"rows from {first}")
    pkg.linear_w4(x, state, add=add, out=add)
    assert torch.equal(add, y)
