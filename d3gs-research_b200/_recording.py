"""Calls that a kernel cannot take part in are refused here."""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as forward_ad

_tracing = torch._C._get_tracing_state
_mode = torch._C._get_dispatch_mode
_mode_before = torch._ops._get_dispatch_mode_pre_dispatch
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def refuse_recording(what: str, tensors):
    """Refuses a call that is being traced, or whose inputs carry a tangent.  What a kernel computes is seen by neither
    ``torch.jit.trace`` (nor ``make_fx``), which would keep the allocation of the result alone, nor forward-mode
    differentiation, which would go on without the tangent."""
    if _tracing() is not None or _mode(_PROXY) is not None or _mode_before(_PROXY) is not None:
        raise RuntimeError(f"{what}: cannot be traced (torch.jit.trace, make_fx): its kernels would not be in the trace")
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise RuntimeError(f"{what}: has no forward-mode derivative, and an input carries a tangent")
