"""Group normalisation with an activation over channels-last images.

The rasteriser blends ``custom_features`` into feature images ``[B, H, W, C]``; ``group_norm_act`` is the
normalisation layer of a network that decodes such images, in their own layout and with its gradient.  The
reference has no counterpart.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib
from ._recording import refuse_recording

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"none": 0, "silu": 1, "gelu": 2}
_DESC = struct.Struct("6q5if")   # GroupNorm; filled through ctypes it takes the host twice as long
assert _DESC.size == C.sizeof(_lib.GroupNorm)


def _pixel_strides(t: torch.Tensor):
    """(image stride, pixel stride) of [B, *spatial, C] when its channels are dense and its pixels evenly spaced,
    else None."""
    shape = t.shape
    if t.is_contiguous():
        n = t.numel()
        return (n // shape[0] if n else 0), shape[-1]
    stride = t.stride()
    if t.numel() == 0:
        return 0, shape[-1]
    if shape[-1] > 1 and stride[-1] != 1:
        return None
    pixel, span = None, 1
    for n, s in zip(reversed(shape[1:-1]), reversed(stride[1:-1])):
        if n == 1:
            continue
        if pixel is None:
            pixel = s
        elif s != pixel * span:
            return None
        span *= n
    return (stride[0] if shape[0] > 1 else 0), (pixel if pixel is not None else shape[-1])


def _prepared(t: torch.Tensor):
    strides = _pixel_strides(t)
    if strides is None:
        t = t.contiguous()
        strides = _pixel_strides(t)
    return t, strides


def _workspace_bytes(lib, d, backward: int) -> int:
    n = lib.d3gs_group_norm_workspace_bytes(C.byref(d), backward)
    if n == 0:
        raise RuntimeError(f"d3gs_group_norm_workspace_bytes: {_lib.last_error()}")
    return n


def _forward(x, groups, weight, bias, eps, act, keep: bool):
    """The input as it was read, the result, and for the backward (``keep``) the statistics and the arguments."""
    device = x.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _forward(x, groups, weight, bias, eps, act, keep)
    lib = _lib.load()
    x, (image, pixel) = _prepared(x)
    shape = x.shape
    batch, channels, values = shape[0], shape[-1], x.numel()
    wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
    args = bytearray(_DESC.pack(batch, values // (batch * channels) if values else 0, image, pixel, 0, 0, channels, groups,
                                _DTYPES[x.dtype], _DTYPES[wdtype], act, eps))
    d = _lib.GroupNorm.from_buffer(args)
    y = torch.empty(shape, dtype=x.dtype, device=device)
    n = _workspace_bytes(lib, d, 0)
    ws = torch.empty(n if keep else n + batch * groups * 8, dtype=torch.uint8, device=device)
    at = ws.data_ptr()
    stats = torch.empty((batch, groups, 2), dtype=torch.float32, device=device) if keep else None
    _lib.check(lib.d3gs_group_norm_forward(C.byref(d), x.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(),
                                           stats.data_ptr() if keep else at + n, at, n, _lib.raw_stream(device.index)),
               "d3gs_group_norm_forward")
    return x, y, stats, args


def _other(t, what: str) -> RuntimeError:
    return RuntimeError(f"group_norm_act: a saved tensor came back as {tuple(t.shape)} {t.dtype} on {t.device}: not the {what} "
                        "that the forward saved")


def _came_back(x, weight, bias, stats, dy, d):
    """The saved tensors as the library reads them.  Hooks of the caller (``save_on_cpu``) may have put copies in their
    place, laid out anew; ``d`` gets the strides of ``x`` as it is now."""
    index, channels, wdtype = dy.get_device(), d.channels, d.weight_dtype
    if x.shape != dy.shape or x.dtype is not dy.dtype or x.get_device() != index:
        raise _other(x, "x")
    if weight is not None:
        if weight.numel() != channels or _DTYPES.get(weight.dtype) != wdtype or weight.get_device() != index:
            raise _other(weight, "weight")
        weight = weight.contiguous()
    if bias is not None:
        if bias.numel() != channels or _DTYPES.get(bias.dtype) != wdtype or bias.get_device() != index:
            raise _other(bias, "bias")
        bias = bias.contiguous()
    if stats.numel() != 2 * d.batch * d.groups or stats.dtype is not torch.float32 or stats.get_device() != index:
        raise _other(stats, "statistics")
    x, (d.x_batch_stride, d.x_pixel_stride) = _prepared(x)
    return x, weight, bias, stats.contiguous()


def _backward(args, x, weight, bias, stats, dy, need_x: bool, need_w: bool, need_b: bool):
    device = dy.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _backward(args, x, weight, bias, stats, dy, need_x, need_w, need_b)
    lib = _lib.load()
    d = _lib.GroupNorm.from_buffer_copy(args)
    x, weight, bias, stats = _came_back(x, weight, bias, stats, dy, d)
    dy, (d.dy_batch_stride, d.dy_pixel_stride) = _prepared(dy)
    empty = x.numel() == 0
    dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_x else None
    make = torch.zeros_like if empty else torch.empty_like
    dw = make(weight) if need_w else None
    db = make(bias) if need_b else None
    if not empty and (need_x or need_w or need_b):
        n = _workspace_bytes(lib, d, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        _lib.check(lib.d3gs_group_norm_backward(C.byref(d), x.data_ptr(), _lib.ptr(weight), _lib.ptr(bias),
                                                stats.data_ptr(), dy.data_ptr(), _lib.ptr(dx), _lib.ptr(dw),
                                                _lib.ptr(db), ws.data_ptr(), n, _lib.raw_stream(device.index)),
                   "d3gs_group_norm_backward")
    return dx, dw, db


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, how):   # how: groups, eps, act
        groups, eps, act = how
        x, y, stats, ctx.args = _forward(x, groups, weight, bias, eps, act, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        # the wrapper that refuses a second derivative takes the host 14 us, as long as the kernels of a small image
        return (_differentiable_once if torch.is_grad_enabled() else _gradients)(ctx, dy)


def _gradients(ctx, dy):
    return (*_backward(ctx.args, *ctx.saved_tensors, dy, *ctx.needs_input_grad[:3]), None)


_differentiable_once = torch.autograd.function.once_differentiable(_gradients)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5, act: str = "silu") -> torch.Tensor:
    """``act(weight * (x - mean) / sqrt(var + eps) + bias)`` of a channels-last image ``x`` ``[B, *spatial, C]``.

    Mean and (biased) variance go over the pixels and the ``C / num_groups`` channels of a group, per image.
    ``act`` is ``"none"``, ``"silu"`` or ``"gelu"`` (the erf form).  ``x`` is float32, bfloat16 or float16; ``weight``
    and ``bias`` ``[C]`` share one of these types, not necessarily that of ``x``.  Sums and statistics are float32.
    Channels that are not dense, or pixels that are not evenly spaced, are copied first.  The result is dense and has
    the type of ``x``; gradients flow to ``x``, ``weight`` and ``bias`` (once).  Under ``torch.jit.trace`` or with inputs
    that carry a forward-mode tangent the call is refused."""
    refuse_recording("group_norm_act", x, weight, bias)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("group_norm_act: x must be a CUDA tensor")
    if x.dim() < 2 or x.dtype not in _DTYPES:
        raise ValueError(f"group_norm_act: x must be [B, ..., C] in float32, bfloat16 or float16, got {tuple(x.shape)} "
                         f"{x.dtype}")
    if act not in _ACTS:
        raise ValueError(f"group_norm_act: act must be one of {sorted(_ACTS)}, got {act!r}")
    c = x.shape[-1]
    num_groups = int(num_groups)
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"group_norm_act: {num_groups} groups do not divide {c} channels")
    if not 0.0 <= eps <= 1e30:
        raise ValueError(f"group_norm_act: eps must be in [0, 1e30], got {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dim() != 1 or t.shape[0] != c or t.device != x.device or t.dtype not in _DTYPES):
            raise ValueError(f"group_norm_act: {name} must be [{c}] on {x.device} in float32, bfloat16 or float16, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("group_norm_act: weight and bias must have one type")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNormAct.apply(x, weight, bias, (num_groups, float(eps), _ACTS[act]))
    return _forward(x, num_groups, weight, bias, float(eps), _ACTS[act], False)[1]
