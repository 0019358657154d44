"""The global norm of many gradients and their clipping, without a host read: `clip_grads` on tensors, `clip_grad_norm_` on parameters.
`VectorQuantize(in_place_codebook_max_grad_norm=)` clips the gradients of its in-place optimizer with it."""
from __future__ import annotations

import array
import ctypes
from typing import Iterable, Optional, Sequence

import torch

from . import _lib as L

_EPS = 1e-6                                               # torch.nn.utils.clip_grad_norm_'s


class _Grad(ctypes.Structure):                            # vqhip_grad_t
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("n", ctypes.c_int64), ("dtype", ctypes.c_int64)]


@L._on_device
def _clip(first, grads, outs, max_norm):
    lib, count = L.lib(), len(grads)
    src = [g.data_ptr() for g in grads]
    dst = [0] * count if outs is None else [o.data_ptr() for o in outs]                      # 0: the norm alone
    rows = zip(src, dst, [g.numel() for g in grads], [L._ELEM_CODES[g.dtype] for g in grads])
    table = array.array("q", [v for row in rows for v in row])                               # vqhip_grad_t [count]
    at = table.buffer_info()[0]
    norm = torch.empty((), dtype=torch.float32, device=first.device)
    nws = lib.vqhip_clip_grads_workspace_bytes(at, count)
    ws = torch.empty(nws, dtype=torch.uint8, device=first.device)
    L._check(lib.vqhip_clip_grads(at, count, max_norm, _EPS, norm.data_ptr(), ws.data_ptr(), nws, L._stream()), "vqhip_clip_grads")
    return norm


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, *, out: Optional[Sequence[torch.Tensor]] = None):
    """-> (clipped, norm): norm = the 2-norm over all elements of all tensors (a 0-dim float32 tensor, summed in 64 bits), clipped =
    every tensor times min(1, max_norm / (norm + 1e-6)), rounded once to its type.

    grads: contiguous float32 / bfloat16 / float16 tensors of one device; out: contiguous tensors of the same types and numbers of
    elements that take the result -- a gradient itself, or memory that no other tensor of the call shares; None: new tensors.  A norm that
    is not finite is not hidden: infinite, it makes every finite gradient 0, NaN makes all of them NaN.  No gradient passes through."""
    grads = list(grads)
    if not max_norm >= 0.0:
        raise L.VQHipError(f"clip_grads: max_norm {max_norm}")
    if not grads:
        return [], torch.zeros((), dtype=torch.float32)
    dev = grads[0].get_device()
    for g in grads:
        if g.dtype not in L._ELEM_CODES:
            L._elem_code(g, "clip_grads")
        if not g.is_contiguous():
            raise L.VQHipError(f"clip_grads: tensor {tuple(g.shape)} with strides {g.stride()}, expected a contiguous one")
        if g.get_device() != dev:
            raise L.VQHipError(f"clip_grads: tensors on different devices ({grads[0].device} and {g.device})")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise L.VQHipError(f"clip_grads: {len(out)} results for {len(grads)} tensors")
        for g, o in zip(grads, out):
            if o is not g and (o.numel() != g.numel() or o.dtype != g.dtype or o.get_device() != dev or not o.is_contiguous()):
                raise L.VQHipError(f"clip_grads: out {tuple(o.shape)} {o.dtype}, expected {g.numel()} contiguous elements of {g.dtype} on {g.device}")
    L._need_gpu(grads[0])
    if out is None:
        out = [torch.empty_like(g) for g in grads]
    norm = _clip(grads[0], grads, out, float(max_norm))
    L._written(out)
    return out, norm


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
