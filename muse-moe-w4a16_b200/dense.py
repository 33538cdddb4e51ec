"""Dense products beside the routed experts: linear_w4 (NVFP4 weights) and gated_ffn (16-bit
weights, with gradients).

Both are what a layer with routed experts needs next to them: its dense projections and its
shared expert, whose output is added to the routed one (`add`). Same rules as kernel_fn: CUDA
tensors only, the current stream, memory from torch's caching allocator, no host
synchronisation; so calls can be captured in a CUDA graph after one eager call of the same sizes.
"""

from __future__ import annotations

import ctypes
import functools
import types
from typing import TypedDict

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from .layer import _require_cuda

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_MAX_ROWS = 1 << 28   # rows of x in one call


class LinearWeights(TypedDict):
    w: torch.Tensor      # uint8 [N, K/2], packed E2M1, element 2i in the low nibble
    w_sf: torch.Tensor   # float8_e4m3fn [N, K/16]
    w_gs: torch.Tensor   # float32, one element


def _bad(message: str) -> _lib.MuseError:
    return _lib.MuseError(_lib.MUSE_ERR_INVALID_ARGUMENT, message)


# Handle of a device's current stream, without the Stream object that torch.cuda.current_stream
# builds (2 us of a call's host time, as much as its launch) where torch has the direct form.
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(index: int, name: str, *args) -> None:
    """An entry point on device `index` and its current stream (kernels launch on the current device)."""
    if torch.cuda.current_device() == index:
        _lib.call(name, *args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _current_stream(index))


def _scratch(n: int, device: torch.device) -> torch.Tensor:
    return torch.empty_strided((n,), (1,), dtype=torch.uint8, device=device)


def _same(t: torch.Tensor, name: str, device: torch.device, dtype: torch.dtype) -> None:
    if t.device != device:
        raise _bad(f"{name} is on {t.device}, x on {device}")
    if t.dtype != dtype:
        raise _bad(f"{name} is {t.dtype}, x {dtype}")


# Where no dual level is open (_current_level < 0) no tensor has a tangent, and a call need not look.
_duals = forward_ad if hasattr(forward_ad, "_current_level") else types.SimpleNamespace(_current_level=0)


def _refuse_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """A forward-mode tangent would be lost without an error: the kernels see the values alone."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _bad(f"{name} has no forward-mode derivative: give it tensors without a tangent")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the byte ranges of two tensors' elements meet."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _rows(t: torch.Tensor, width: int) -> tuple[torch.Tensor, int]:
    """`t` [..., width] as 16-byte aligned rows and their stride: in place where its strides
    allow it, else a contiguous copy."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if t.is_contiguous() and not t.data_ptr() % 16:
        return t, width
    ld = t.stride(0) if t.shape[0] > 1 else width
    if t.stride(1) != 1 or ld % 8 or ld < width or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        ld = width
    return t, ld


def prepare_linear(weight: LinearWeights, gated: bool = False) -> dict:
    """Repack an NVFP4 matrix [N, K] for linear_w4 (once, untimed): any N, K a multiple of 16.
    gated: rows [0, N/2) are gate rows and the rest the matching up rows (a w13).

    The state's tensors may be copied and rewritten in place like any others."""
    w, sf, gs = weight["w"], weight["w_sf"], weight["w_gs"]
    _require_cuda(w, "w")
    if w.dtype != torch.uint8 or w.dim() != 2 or 0 in w.shape:
        raise _bad("w must be a uint8 matrix of packed codes [N, K/2]")
    N, K = w.shape[0], 2 * w.shape[1]
    if K % 16:
        raise _bad(f"K = {K} is not a multiple of 16")
    if gated and N % 2:
        raise _bad(f"a gated weight has gate and up rows in equal number, got {N} rows")
    if sf.dtype not in (torch.float8_e4m3fn, torch.uint8) or tuple(sf.shape) != (N, K // 16):
        raise _bad(f"w_sf must be float8_e4m3fn {(N, K // 16)}, got {sf.dtype} {tuple(sf.shape)}")
    if gs.numel() != 1 or not gs.is_floating_point():
        raise _bad("w_gs must be one floating-point value")
    dev = w.device
    if sf.device != dev:
        raise _bad(f"w_sf is on {sf.device}, w on {dev}")
    codes, scales = w.contiguous(), sf.contiguous().view(torch.uint8)
    if codes.data_ptr() % 8:
        codes = codes.clone()
    size = ctypes.c_size_t(0)
    _lib.call("muse_moe_linear_prepared_size", N, K, int(gated), ctypes.byref(size))
    out = torch.empty(size.value, dtype=torch.uint8, device=dev)
    _call(dev.index, "muse_moe_prepare_linear", codes.data_ptr(), scales.data_ptr(), N, K, int(gated), out.data_ptr())
    return {"w": out, "w_gs": gs.to(device=dev, dtype=torch.float32).reshape(1).clone(),
            "rows": N, "cols": K, "gated": bool(gated), "n_out": N // 2 if gated else N}


def linear_w4(x: torch.Tensor, state: dict, add: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] times a prepared NVFP4 matrix: [..., N], or silu(gate) * up [..., N/2] for a gated
    one, plus `add` (same shape) if given. x is bf16 or fp16, and so are add and the result; any
    number of rows. Sums in fp32, one rounding. `out` receives the result if given; it may be `add`
    itself. Inference only: it has no gradient, and refuses tensors that want one or carry a
    forward-mode tangent."""
    _require_cuda(x, "x")
    K, n_out, w, dev = state["cols"], state["n_out"], state["w"], x.device
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise _bad(f"x must be bfloat16 or float16, got {x.dtype}")
    shape = x.shape
    if not shape or shape[-1] != K:
        raise _bad(f"x {tuple(shape)} does not end in the weight's {K} columns")
    gs = state["w_gs"]
    if w.device != dev or gs.device != dev:
        raise _bad(f"the weight is on {w.device} and its scale on {gs.device}, x on {dev}")
    if torch.is_grad_enabled() and (x.requires_grad or gs.requires_grad or (add is not None and add.requires_grad)):
        raise _bad("linear_w4 has no gradient: call it under torch.no_grad()")
    if _duals._current_level >= 0:
        _refuse_tangents("linear_w4", x, gs, add, out)
    x2, ldx = _rows(x, K)
    T = x2.shape[0]
    if T > _MAX_ROWS:
        raise _lib.MuseError(_lib.MUSE_ERR_UNSUPPORTED_SHAPE, f"{T} rows in one call, at most {_MAX_ROWS}")
    if len(shape) == 2:
        shape = (T, n_out)
    else:
        shape = shape[:-1] + (n_out,)
    add_ptr, ld_add = None, 0
    if add is not None:
        _same(add, "add", dev, x.dtype)
        if add.shape != shape:
            raise _bad(f"add must be {tuple(shape)}, got {tuple(add.shape)}")
        add2 = add if add.dim() == 2 else add.reshape(-1, n_out)
        if not add2.is_contiguous() and (add2.stride(1) != 1 or (T > 1 and add2.stride(0) < n_out)):
            add2 = add2.contiguous()
        add_ptr, ld_add = add2.data_ptr(), add2.stride(0)
    if out is None:
        out = x.new_empty(shape)
    elif out.shape != shape or out.dtype != x.dtype or out.device != dev or not out.is_contiguous():
        raise _bad(f"out must be a contiguous {x.dtype} {tuple(shape)} on {dev}")
    elif _overlap(out, x) or (add is not None and _overlap(out, add)
                              and (add.data_ptr() != out.data_ptr() or not add.is_contiguous())):
        raise _bad("out may be add itself, but overlaps no input otherwise")
    elif out.requires_grad and torch.is_grad_enabled():
        raise _bad("out requires a gradient, which linear_w4 does not have")
    else:
        increment_version(out)   # autograd sees the write: a backward pass that kept out's old values refuses
    _call(dev.index, "muse_moe_linear_w4", x2.data_ptr(), ldx, dtype, T, state["rows"], K, 1 if state["gated"] else 0,
          w.data_ptr(), gs.data_ptr(), add_ptr, ld_add, out.data_ptr(), n_out)
    return out


@functools.lru_cache(maxsize=4096)
def _ffn_workspace(tokens: int, hidden: int, inter: int, backward: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.call("muse_moe_ffn_workspace_size", tokens, hidden, inter, backward, ctypes.byref(n))
    return n.value


def _ffn_forward(x, w13, w2, add, keep: bool):
    """(out, ab): the block's output and, with `keep`, its fp32 pre-activations [T, 2I]."""
    H, I = w2.shape
    dev, dtype = x.device, x.dtype
    x2, ldx = _rows(x, H)
    T = x2.shape[0]
    out = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    ab = torch.empty((T, 2 * I), dtype=torch.float32, device=dev) if keep else None
    if T == 0:
        return out, ab
    w13, ld13 = _rows(w13, H)
    w2, ld2 = _rows(w2, I)
    add2, ld_add = (None, 0) if add is None else _rows(add, H)
    n = _ffn_workspace(T, H, I, 0)
    ws = _scratch(n, dev)
    _call(dev.index, "muse_moe_ffn_forward", x2.data_ptr(), ldx, _DTYPES[dtype], T, H, I, w13.data_ptr(), ld13,
          w2.data_ptr(), ld2, None if add is None else add2.data_ptr(), ld_add, out.data_ptr(),
          ab.data_ptr() if keep else None, ws.data_ptr(), n)
    return out, ab


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, add):
        keep = any(ctx.needs_input_grad[:3])
        out, ab = _ffn_forward(x, w13, w2, add, keep)
        if keep:
            ctx.save_for_backward(x, w13, w2, ab)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_13, need_2, need_add = ctx.needs_input_grad
        dx = dw13 = dw2 = None
        if need_x or need_13 or need_2:
            x, w13, w2, ab = ctx.saved_tensors
            H, I = w2.shape
            T, dev = ab.shape[0], x.device
            make = torch.zeros if T == 0 else torch.empty
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
            dw13 = make((2 * I, H), dtype=x.dtype, device=dev) if need_13 else None
            dw2 = make((H, I), dtype=x.dtype, device=dev) if need_2 else None
            if T:
                dy2, ldy = _rows(dy, H)
                x2, ldx = _rows(x, H)
                w13, ld13 = _rows(w13, H)
                w2, ld2 = _rows(w2, I)
                n = _ffn_workspace(T, H, I, 1)
                ws = _scratch(n, dev)
                _call(dev.index, "muse_moe_ffn_backward", dy2.data_ptr(), ldy, x2.data_ptr(), ldx, _DTYPES[x.dtype], T,
                      H, I, w13.data_ptr(), ld13, w2.data_ptr(), ld2, ab.data_ptr(),
                      dx.data_ptr() if need_x else None, dw13.data_ptr() if need_13 else None,
                      dw2.data_ptr() if need_2 else None, ws.data_ptr(), n)
        return dx, dw13, dw2, dy if need_add else None


def gated_ffn(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, add: torch.Tensor | None = None) -> torch.Tensor:
    """The gated feed-forward block (silu(x Wg^T) * (x Wu^T)) W2^T (+ add), 16-bit weights.

    x [..., H], w13 [2I, H] (gate rows, then up rows, as the routed experts' w13), w2 [H, I], add of
    x's shape; all bf16 or all fp16; H and I multiples of 8. Sums in fp32; the inner activation and the
    gradients of the pre-activations are rounded to the tensors' type (fp16 ones overflow past
    65504). Differentiable once in every tensor, in reverse mode (a forward-mode tangent is refused); a pass that needs gradients keeps the
    pre-activations in fp32 (8 T I bytes). Equal inputs give equal bits, with or without gradients."""
    _require_cuda(x, "x")
    dev = x.device
    if x.dtype not in _DTYPES:
        raise _bad(f"x must be bfloat16 or float16, got {x.dtype}")
    _same(w13, "w13", dev, x.dtype)
    _same(w2, "w2", dev, x.dtype)
    if w13.dim() != 2 or w2.dim() != 2 or x.dim() == 0:
        raise _bad("gated_ffn needs x [..., H], w13 [2I, H] and w2 [H, I]")
    H, I = w2.shape
    if x.shape[-1] != H or tuple(w13.shape) != (2 * I, H):
        raise _bad(f"inconsistent shapes: x {tuple(x.shape)}, w13 {tuple(w13.shape)}, w2 {tuple(w2.shape)}")
    if H == 0 or I == 0 or H % 8 or I % 8:
        raise _lib.MuseError(_lib.MUSE_ERR_UNSUPPORTED_SHAPE, f"H = {H} and I = {I} must be multiples of 8")
    if x.numel() // H > _MAX_ROWS:
        raise _lib.MuseError(_lib.MUSE_ERR_UNSUPPORTED_SHAPE, f"{x.numel() // H} rows in one call, at most {_MAX_ROWS}")
    if add is not None:
        _same(add, "add", dev, x.dtype)
        if add.shape != x.shape:
            raise _bad(f"add must be {tuple(x.shape)}, got {tuple(add.shape)}")
    if _duals._current_level >= 0:
        _refuse_tangents("gated_ffn", x, w13, w2, add)
    if torch.is_grad_enabled() and (x.requires_grad or w13.requires_grad or w2.requires_grad
                                    or (add is not None and add.requires_grad)):
        return _GatedFfn.apply(x, w13, w2, add)
    return _ffn_forward(x, w13, w2, add, False)[0]
