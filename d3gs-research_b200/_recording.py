"""Calls that a kernel cannot take part in are refused here."""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as forward_ad

# looked up once: with small tensors a call is bound by the host
_tracing, _mode, _mode_before = torch._C._get_tracing_state, torch._C._get_dispatch_mode, torch._ops._get_dispatch_mode_pre_dispatch
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def refuse_recording(what: str, *tensors):
    """Refuses a call that is being traced, or whose inputs (tensors, or lists of them) carry a tangent.  What a kernel
    computes is seen by neither ``torch.jit.trace`` (nor ``make_fx``), which would keep the allocation of the result alone,
    nor forward-mode differentiation, which would go on without the tangent."""
    if _tracing() is not None or _mode(_PROXY) is not None or _mode_before(_PROXY) is not None:
        raise RuntimeError(f"{what}: cannot be traced (torch.jit.trace, make_fx): its kernels would not be in the trace")
    if forward_ad._current_level >= 0:
        for t in tensors:
            for u in t if isinstance(t, list) else (t,):
                if isinstance(u, torch.Tensor) and forward_ad.unpack_dual(u).tangent is not None:
                    raise RuntimeError(f"{what}: has no forward-mode derivative, and an input carries a tangent")
