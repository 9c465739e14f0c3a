"""Orthogonalised updates of weight matrices, and the optimizer that takes them.

``GaussianAdam`` steps the per-Gaussian parameters.  The hidden matrices of a network that decodes rendered feature
images are better served by an update whose singular values are all near one: the momentum, orthogonalised by a few
Newton-Schulz products.  ``orthogonalize`` is that product chain, ``muon_step`` the whole update of a list of
parameters in a handful of launches, ``GaussianMuon`` the optimizer around it.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
from bisect import bisect_left
from typing import Sequence

import torch

from . import _lib
from ._recording import refuse_recording

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=64)
def _coefficients(what: str, coefficients: tuple, steps: int):
    """a, b, c of every step as the library takes them."""
    if not 1 <= steps <= _lib.NS_MAX_STEPS:
        raise ValueError(f"{what}: ns_steps must be 1 to {_lib.NS_MAX_STEPS}, got {steps}")
    if len(coefficients) == 3 and not isinstance(coefficients[0], tuple):
        coefficients = (coefficients,) * steps
    if len(coefficients) != steps or any(len(c) != 3 for c in coefficients):
        raise ValueError(f"{what}: ns_coefficients must be (a, b, c), or one such triple for each of {steps} steps")
    if not all(math.isfinite(v) for c in coefficients for v in c):
        raise ValueError(f"{what}: ns_coefficients must be finite")
    return (C.c_float * (3 * steps))(*[v for c in coefficients for v in c])


def _config(what: str, dtype: int, coefficients, eps: float, steps: int) -> _lib.OrthoConfig:
    values = _coefficients(what, tuple([tuple(map(float, c)) if isinstance(c, (tuple, list)) else float(c) for c in coefficients]),
                           int(steps))
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"{what}: eps must be finite and positive, got {eps}")
    cfg = _lib.OrthoConfig()
    cfg.dtype, cfg.steps, cfg.eps = dtype, steps, eps
    C.memmove(cfg.coefficients, values, C.sizeof(values))
    return cfg


def _run(entry: str, mats, count: int, cfg: _lib.OrthoConfig, device):
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _run(entry, mats, count, cfg, device)
    lib = _lib.load()
    n = lib.d3gs_orthogonalize_workspace_bytes(mats, count, C.byref(cfg))
    if n == 0:
        raise RuntimeError(f"{entry}: {_lib.last_error()}")
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    _lib.check(getattr(lib, entry)(mats, count, C.byref(cfg), ws.data_ptr(), n, _lib.raw_stream(device.index)), entry)


@torch.no_grad()
def orthogonalize(update: torch.Tensor, ns_coefficients: Sequence = NS_COEFFICIENTS, eps: float = 1e-7,
                  ns_steps: int = 5) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of a matrix ``[m, n]`` or of each matrix of a stack ``[..., m, n]``.

    ``X = U / max(|U|_F, eps)``, then ``ns_steps`` times ``X = a X + (b A + c A A) X`` with ``A = X X^T``.
    ``ns_coefficients`` is ``(a, b, c)``, or one such triple per step.  float32 or bfloat16 in, a dense tensor of the
    same type out; every product is summed in 32 bits.  float32 results are off by some 1e-6 of their norm; bfloat16 ones by
    their own rounding, and with a short side above 384 by up to 1.5e-3 more (products of fp16 operands).  Rows that are not
    dense are copied first.  No gradient.
    Coefficients with which singular values in [0, 1] grow past 1024, or with ``0 < 1024 |c| < |b|``, are refused, and so
    are calls under ``torch.jit.trace`` or with a forward-mode tangent."""
    refuse_recording("orthogonalize", update)
    if not isinstance(update, torch.Tensor) or not update.is_cuda:
        raise ValueError("orthogonalize: update must be a CUDA tensor")
    if update.dim() < 2 or update.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"orthogonalize: update must be [..., m, n] in float32 or bfloat16, got {tuple(update.shape)} "
                         f"{update.dtype}")
    cfg = _config("orthogonalize", 0 if update.dtype == torch.float32 else 1, ns_coefficients, eps, ns_steps)
    out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    if update.numel() == 0:
        return out
    m, n = update.shape[-2:]
    if (n > 1 and update.stride(-1) != 1) or update.dim() > 3:
        update = update.contiguous()
    src = update.reshape(-1, m, n)
    count, step, size = src.shape[0], src.stride(0) * src.element_size(), src.element_size()
    mats = (_lib.OrthoMatrix * count)()
    for k in range(count):
        mats[k] = (src.data_ptr() + k * step, None, out.data_ptr() + k * m * n * size, m, n, src.stride(1), 0.0, 0)
    _run("d3gs_orthogonalize", mats, count, cfg, update.device)
    return out


def _dense_rows(t: torch.Tensor) -> bool:
    """Whether the first axis is the outermost of a gapless layout (contiguous or channels last): flattening the
    rest gives the same columns, in some order, for every tensor of these strides."""
    return (t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last))
            or (t.dim() == 5 and t.is_contiguous(memory_format=torch.channels_last_3d)))


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal strides wherever an axis has more than one value."""
    return all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _adjusted_lr(lr: float, rows: int, cols: int, adjust_lr_fn: str | None) -> float:
    if adjust_lr_fn == "match_rms_adamw":
        return lr * 0.2 * math.sqrt(max(rows, cols))
    return lr * math.sqrt(max(1.0, rows / cols))


_MATRIX = struct.Struct("PPPqqqfi")   # OrthoMatrix; a struct filled through ctypes takes three times as long
assert _MATRIX.size == C.sizeof(_lib.OrthoMatrix)
_ADJUST = (None, "original", "match_rms_adamw")


@torch.no_grad()
def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momentum_buffers: Sequence[torch.Tensor], *,
              lr: float, weight_decay: float = 0.1, momentum: float = 0.95, nesterov: bool = True,
              ns_coefficients: Sequence = NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
              adjust_lr_fn: str | None = None) -> None:
    """One optimizer step of a list of float32 parameters, in place, all of them through the same launches::

        buffer = momentum * buffer + (1 - momentum) * grad
        update = momentum * buffer + (1 - momentum) * grad   if nesterov else   buffer
        param  = (1 - lr * weight_decay) * param - lr * ratio * orthogonalize(update)

    A parameter of more than two axes (a convolution's filters) is taken as ``[size(0), the rest]``.  ``ratio`` is
    ``sqrt(max(1, rows / columns))``, or with ``adjust_lr_fn="match_rms_adamw"`` ``0.2 sqrt(max(rows, columns))``.
    Parameters and buffers must be dense (contiguous or channels last) and must not overlap one another or a gradient."""
    params, grads, momentum_buffers = list(params), list(grads), list(momentum_buffers)
    refuse_recording("muon_step", params, grads, momentum_buffers)
    if not len(params) == len(grads) == len(momentum_buffers):
        raise ValueError(f"muon_step: {len(params)} params, {len(grads)} grads, {len(momentum_buffers)} momentum_buffers")
    if adjust_lr_fn not in _ADJUST:
        raise ValueError(f"muon_step: adjust_lr_fn must be one of {_ADJUST}, got {adjust_lr_fn!r}")
    lr, weight_decay, momentum = float(lr), float(weight_decay), float(momentum)
    for name, v in (("lr", lr), ("weight_decay", weight_decay)):
        if not 0.0 <= v <= 1e30:
            raise ValueError(f"muon_step: {name} must be in [0, 1e30], got {v}")
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"muon_step: momentum must be in [0, 1), got {momentum}")
    cfg = _config("muon_step", 0, ns_coefficients, eps, ns_steps)
    cfg.momentum, cfg.decay, cfg.nesterov = momentum, 1.0 - lr * weight_decay, int(nesterov)
    table = bytearray(C.sizeof(_lib.OrthoMatrix) * len(params))
    keep, spans, read, count, device, f32 = [], [], [], 0, None, torch.float32
    for p, g, buf in zip(params, grads, momentum_buffers):
        at_device, shape = p.device, p.shape
        if not (p.is_cuda and p.dtype is f32 and g.dtype is f32 and buf.dtype is f32 and len(shape) >= 2
                and g.device == at_device and buf.device == at_device and g.shape == shape and buf.shape == shape
                and g.layout is torch.strided):
            raise ValueError("muon_step: params, grads and momentum_buffers must be float32 CUDA tensors of two or more axes "
                             f"with equal shapes and devices, got {tuple(p.shape)} {p.dtype} {p.device}, {tuple(g.shape)} "
                             f"{g.dtype} {g.device}, {tuple(buf.shape)} {buf.dtype} {buf.device}")
        if device is None:
            device = at_device
        if at_device != device:
            raise ValueError(f"muon_step: parameters on {device} and {p.device} in one call")
        size = p.numel()
        if size == 0:
            continue
        plain = p.is_contiguous()
        if not (plain and buf.is_contiguous()) and (not _dense_rows(p) or not _same_order(p, buf)):
            raise ValueError(f"muon_step: a parameter of strides {p.stride()} or its buffer of strides {buf.stride()} is not "
                             "dense (contiguous or channels last, the two alike)")
        rows = shape[0]
        row_stride = cols = size // rows
        if not (plain and g.is_contiguous()) and not _same_order(p, g):
            if g.dim() == 2 and (cols == 1 or g.stride(1) == 1) and plain:
                row_stride = g.stride(0)
            else:
                g = torch.empty_like(p).copy_(g)
                keep.append(g)
        src, state, at, size = g.data_ptr(), buf.data_ptr(), p.data_ptr(), 4 * size
        _MATRIX.pack_into(table, count * _MATRIX.size, src, state, at, rows, cols, row_stride,
                          _adjusted_lr(lr, rows, cols, adjust_lr_fn), 0)
        spans.append((state, state + size))
        spans.append((at, at + size))
        read.append((src, src + ((rows - 1) * row_stride + cols) * 4))
        count += 1
    if count == 0:
        return
    spans.sort()
    if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
        raise ValueError("muon_step: parameters or buffers overlap (is one given twice?)")
    ends = [end for _, end in spans]
    for first, last in read:
        k = bisect_left(ends, first + 1)   # the first span that ends behind the gradient's start
        if k < len(spans) and spans[k][0] < last:
            raise ValueError("muon_step: a gradient overlaps a parameter or a buffer")
    _run("d3gs_muon_step", (_lib.OrthoMatrix * len(params)).from_buffer(table), count, cfg, device)
    torch.autograd.graph.increment_version([*params, *momentum_buffers])


class GaussianMuon(torch.optim.Optimizer):
    """Optimizer over ``muon_step``: one call per parameter group.  Takes float32 CUDA parameters of two or more axes;
    biases and per-Gaussian parameters belong to ``GaussianAdam``.  The state of a parameter is ``momentum_buffer``.
    Hyper-parameters are those of ``muon_step``."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients: Sequence = NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
                 adjust_lr_fn: str | None = None):
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps,
                                      adjust_lr_fn=adjust_lr_fn))
        for group in self.param_groups:
            _config("GaussianMuon", 0, group["ns_coefficients"], group["eps"], group["ns_steps"])
            for p in group["params"]:
                if p.dim() < 2 or p.dtype != torch.float32:
                    raise ValueError(f"GaussianMuon: parameters must be float32 with two or more axes, got {tuple(p.shape)} "
                                     f"{p.dtype}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                state = self.state[p]
                if len(state) == 0:
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            if params:
                muon_step(params, [p.grad for p in params], [self.state[p]["momentum_buffer"] for p in params],
                          **{k: v for k, v in group.items() if k in _HYPER})
        return loss


_HYPER = ("lr", "weight_decay", "momentum", "nesterov", "ns_coefficients", "eps", "ns_steps", "adjust_lr_fn")
