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
def _clip(first, table, max_norm):
    """table: array('q') of vqhip_grad_t rows"""
    lib, (at, fields) = L.lib(), table.buffer_info()
    norm = torch.empty((), dtype=torch.float32, device=first.device)
    nws = lib.vqhip_clip_grads_workspace_bytes(at, fields // 4)
    ws = torch.empty(nws, dtype=torch.uint8, device=first.device)
    L._check(lib.vqhip_clip_grads(at, fields // 4, max_norm, _EPS, norm.data_ptr(), ws.data_ptr(), nws, L._stream()), "vqhip_clip_grads")
    return norm


def _check(grads, out):
    """raises what is wrong with a tensor or its result, if anything is"""
    dev = grads[0].get_device()
    for g, o in zip(grads, out):
        L._elem_code(g, "clip_grads")
        if not g.is_contiguous():
            raise L.VQHipError(f"clip_grads: tensor {tuple(g.shape)} with strides {g.stride()}, expected a contiguous one")
        if g.get_device() != dev:
            raise L.VQHipError(f"clip_grads: tensors on different devices ({grads[0].device} and {g.device})")
        if o.numel() != g.numel() or o.dtype != g.dtype or not o.is_contiguous() or o.get_device() != dev:
            raise L.VQHipError(f"clip_grads: out {tuple(o.shape)} {o.dtype}, expected {g.numel()} contiguous elements of {g.dtype} on {g.device}")


def _unflagged(grads, out):
    """grads with a pending negation carried out where the result has none (the imaginary part of a conjugate only sets a flag; its strides are
    even, so of contiguous tensors single elements alone have one)"""
    grads = list(grads)
    for i, g in enumerate(grads):
        if out is not None and out[i].is_neg() and not g.is_neg():
            raise L.VQHipError("clip_grads: out with a pending negation")
        if g.is_neg() and (out is None or not out[i].is_neg()):
            grads[i] = g.resolve_neg()
    return grads


def _table(grads, out):
    """the checked rows of vqhip_grad_t, and the tensors that they point to; out None: the norm alone.  A pass over all tensors for each
    property: a model has hundreds, and `map` takes two thirds of the time of a loop over them (311 tensors with results of their own: a
    call 205 us instead of 250)"""
    T, codes = torch.Tensor, L._ELEM_CODES
    dtypes, sizes = [t.dtype for t in grads], list(map(T.numel, grads))
    if 1 in sizes and out is not grads:
        grads = _unflagged(grads, out)
    fine = all(map(T.is_contiguous, grads)) and len(set(map(T.get_device, grads))) == 1 and all(map(codes.__contains__, set(dtypes)))
    if out is not None and out is not grads:
        fine = fine and sizes == list(map(T.numel, out)) and dtypes == [t.dtype for t in out] and all(map(T.is_contiguous, out)) \
            and set(map(T.get_device, out)) == {grads[0].get_device()}
    if not fine:
        _check(grads, grads if out is None else out)
    flat = [0] * (4 * len(grads))
    flat[::4] = map(T.data_ptr, grads)
    if out is not None:
        flat[1::4] = map(T.data_ptr, out)
    flat[2::4] = sizes
    flat[3::4] = [codes[d] for d in dtypes]
    return array.array("q", flat), grads


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, *, out: Optional[Sequence[torch.Tensor]] = None):
    """-> (clipped, norm): norm = the 2-norm over all elements of all tensors (a 0-dim float32 tensor, summed in 64 bits), clipped =
    every tensor times min(1, max_norm / (norm + 1e-6)), the factor in 32 bits, the product rounded to the tensor's type.

    grads: contiguous float32 / bfloat16 / float16 tensors of one device; out: contiguous tensors of the same types and numbers of
    elements that take the result -- a gradient itself, or memory that no other tensor of the call shares; None: new tensors.  A norm that
    is not finite is not hidden: infinite, it makes every finite gradient 0, NaN makes all of them NaN.  max_norm inf: the norm alone
    (nothing is scaled unless it is NaN).  No gradient passes through, and a forward-mode tangent is refused."""
    given, grads = grads, list(grads)
    if not max_norm >= 0.0:
        raise L.VQHipError(f"clip_grads: max_norm {max_norm}")
    if not grads:
        return [], torch.zeros((), dtype=torch.float32)
    L._no_tangent("clip_grads", grads)
    if out is None:
        table, grads = _table(grads, None)
        L._need_gpu(grads[0])
        out = [torch.empty_like(g) for g in grads]
        table[1::4] = array.array("q", [o.data_ptr() for o in out])
    else:
        out = grads if out is given else list(out)
        if len(out) != len(grads):
            raise L.VQHipError(f"clip_grads: {len(out)} results for {len(grads)} tensors")
        L._no_tangent("clip_grads", out)
        table, grads = _table(grads, out)
        L._need_gpu(grads[0])
    norm = _clip(grads[0], table, float(max_norm))
    L._written(out)
    return out, norm


def clip_grad_norm_(parameters: Iterable[torch.Tensor], max_norm: float, *, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of `parameters` in place to a global 2-norm of max_norm and returns the norm before (0-dim float32, on the
    device; nothing is read back unless error_if_nonfinite asks).  Parameters without a gradient are passed over; a gradient that is not
    contiguous is clipped through a contiguous copy."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = list(parameters)
    L._no_tangent("clip_grad_norm_", (p.grad for p in parameters))
    grads = list({id(p.grad): p.grad.detach() for p in parameters if p.grad is not None}.values())      # a shared one counts once
    work = [g if g.is_contiguous() else g.contiguous() for g in grads]
    if error_if_nonfinite and work:
        table, _ = _table(work, None)
        L._need_gpu(work[0])
        if not torch.isfinite(_clip(work[0], table, 0.0)).item():
            raise RuntimeError("clip_grad_norm_: the total norm of the gradients is not finite")
    _, norm = clip_grads(work, max_norm, out=work)
    for g, w in zip(grads, work):
        if w is not g:
            g.copy_(w)
    return norm
