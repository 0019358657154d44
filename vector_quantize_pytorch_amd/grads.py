"""The global norm of many gradients and their clipping, without a host read: `clip_grads` on tensors, `clip_grad_norm_` on parameters.
`VectorQuantize(in_place_codebook_max_grad_norm=)` clips the gradients of its in-place optimizer with it."""
from __future__ import annotations

import ctypes
from typing import Iterable, Optional, Sequence

import torch

from . import _lib as L

_EPS = 1e-6                                               # torch.nn.utils.clip_grad_norm_'s


class _Grad(ctypes.Structure):                            # vqhip_grad_t
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("n", ctypes.c_int64), ("dtype", ctypes.c_int64)]


@L._on_device
def _clip(first, grads, outs, max_norm):
    codes = L._ELEM_CODES
    dst = [None] * len(grads) if outs is None else [o.data_ptr() for o in outs]              # None: the norm alone
    table = (_Grad * len(grads))(*[(g.data_ptr(), d, g.numel(), codes[g.dtype]) for g, d in zip(grads, dst)])
    norm = torch.empty((), dtype=torch.float32, device=first.device)
    nws = L.lib().vqhip_clip_grads_workspace_bytes(table, len(grads))
    ws = torch.empty(nws, dtype=torch.uint8, device=first.device)
    L._check(L.lib().vqhip_clip_grads(table, len(grads), max_norm, _EPS, norm.data_ptr(), ws.data_ptr(), nws, L._stream()), "vqhip_clip_grads")
    return norm


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, *, out: Optional[Sequence[torch.Tensor]] = None):
    """-> (clipped, norm): norm = the 2-norm over all elements of all tensors (a 0-dim float32 tensor, summed in 64 bits), clipped =
    every tensor times min(1, max_norm / (norm + 1e-6)), rounded once to its type.

    grads: contiguous float32 / bfloat16 / float16 tensors of one device, none twice; out: contiguous tensors that take the result, of
    the same shapes and types -- a gradient itself, or memory that no other tensor of the call shares; None: new tensors.  A norm that is
    not finite is not hidden: infinite, it makes every finite gradient 0, NaN makes all of them NaN.  No gradient passes through."""
    grads = list(grads)
    if not max_norm >= 0.0:
        raise L.VQHipError(f"clip_grads: max_norm {max_norm}")
    if not grads:
        return [], torch.zeros((), dtype=torch.float32)
    dev = grads[0].device
    for g in grads:
        if g.dtype not in L._ELEM_CODES:
            L._elem_code(g, "clip_grads")
        if not g.is_contiguous():
            raise L.VQHipError(f"clip_grads: tensor {tuple(g.shape)} with strides {g.stride()}, expected a contiguous one")
        if g.device != dev:
            raise L.VQHipError(f"clip_grads: tensors on different devices ({dev} and {g.device})")
    if len({g.data_ptr() for g in grads if g.numel()}) != sum(1 for g in grads if g.numel()):
        raise L.VQHipError("clip_grads: a tensor occurs twice")
    if out is None:
        L._need_gpu(*grads[:1])
        out = [torch.empty_like(g) for g in grads]
    else:
        out = list(out)
        if len(out) != len(grads):
            raise L.VQHipError(f"clip_grads: {len(out)} results for {len(grads)} tensors")
        for g, o in zip(grads, out):
            if o.shape != g.shape or o.dtype != g.dtype or o.device != dev or not o.is_contiguous():
                raise L.VQHipError(f"clip_grads: out {tuple(o.shape)} {o.dtype}, expected contiguous {tuple(g.shape)} {g.dtype} on {dev}")
        _check_memory(grads, out)
        L._need_gpu(*grads[:1])
    norm = _clip(grads[0], grads, out, float(max_norm))
    L._written(out)
    return out, norm


def _check_memory(grads, outs):
    """every result is its own gradient's memory, or shares none with any tensor of the call"""
    spans = [(g.data_ptr(), g.data_ptr() + g.numel() * g.element_size(), 0) for g in grads if g.numel()]
    spans += [(o.data_ptr(), o.data_ptr() + o.numel() * o.element_size(), 1) for g, o in zip(grads, outs)
              if o.numel() and o.data_ptr() != g.data_ptr()]
    inside = {g.data_ptr() for g, o in zip(grads, outs) if o.data_ptr() == g.data_ptr()}       # gradients that are written themselves
    spans.sort()
    end = end_out = -1
    for first, behind, is_out in spans:
        written = is_out or first in inside
        if first < (end if written else end_out):
            raise L.VQHipError("clip_grads: a result shares memory with another tensor")
        end = max(end, behind)
        if written:
            end_out = max(end_out, behind)


def clip_grad_norm_(parameters: Iterable[torch.Tensor], max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of `parameters` in place to a global 2-norm of max_norm and returns the norm before (0-dim float32, on the
    device; nothing is read back unless error_if_nonfinite asks).  Parameters without a gradient are passed over; a gradient that is not
    contiguous is clipped through a contiguous copy."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = list({id(p.grad): p.grad.detach() for p in parameters if p.grad is not None}.values())      # a shared one counts once
    work = [g if g.is_contiguous() else g.contiguous() for g in grads]
    if error_if_nonfinite and work:
        L._need_gpu(*work[:1])
        if not torch.isfinite(_clip(work[0], work, None, 0.0)).item():
            raise RuntimeError("clip_grad_norm_: the total norm of the gradients is not finite")
    _, norm = clip_grads(work, max_norm, out=work)
    for g, w in zip(grads, work):
        if w is not g:
            g.copy_(w)
    return norm
