"""Group norm with an activation on channels-last rows: the normalisation between a tokenizer's convolutions, in the layout that the
quantizers read -- a channels-last map goes through norm and quantizer without a transposing copy."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import nn

from . import _lib as L

NORM_MAX_C = 8192                                         # VQHIP_NORM_MAX_C
_ACTIVATIONS = {None: 0, "silu": 1}

_i64, _vp = ctypes.c_int64, ctypes.c_void_p


class _Norm(ctypes.Structure):                            # vqhip_group_norm_t
    _fields_ = [("x", _vp), ("dtype", _i64), ("B", _i64), ("N", _i64), ("C", _i64), ("stride_b", _i64), ("stride_n", _i64), ("groups", _i64),
                ("weight", _vp), ("bias", _vp), ("param_dtype", _i64), ("eps", ctypes.c_double), ("activation", _i64), ("lens", _vp), ("mask", _vp),
                ("mean", _vp), ("rstd", _vp), ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t)]


def _addr(t):
    return None if t is None else t.data_ptr()


def _struct(x, weight, bias, lens, mask, groups, eps, act, mean, ws, nws):
    b, n, c = x.shape
    sb, sn, _ = x.stride()
    param = weight if weight is not None else bias
    return _Norm(x.data_ptr(), L._ELEM_CODES[x.dtype], b, n, c, sb, sn, groups, _addr(weight), _addr(bias),
                 L.F32 if param is None else L._ELEM_CODES[param.dtype], eps, act, _addr(lens), _addr(mask), mean, mean + 4 * b * groups, ws, nws)


@L._on_device
def _forward(x, weight, bias, lens, mask, groups, eps, act, keep):
    """keep: mean and rstd in memory of their own, for a backward; otherwise behind the workspace"""
    b, n, c = x.shape
    lib, dev = L.lib(), x.device
    y = torch.empty((b, n, c), dtype=x.dtype, device=dev)
    nws = lib.vqhip_group_norm_workspace_bytes(b, n, c, groups)
    stats = torch.empty((2, b, groups), dtype=torch.float32, device=dev) if keep else None
    ws = torch.empty(nws + (0 if keep else 8 * b * groups), dtype=torch.uint8, device=dev)
    at = ws.data_ptr()
    s = _struct(x, weight, bias, lens, mask, groups, eps, act, stats.data_ptr() if keep else at + nws, at, nws)
    L._check(lib.vqhip_group_norm(ctypes.byref(s), y.data_ptr(), L._stream()), "vqhip_group_norm")
    return y, stats


@L._on_device
def _backward(grad, x, weight, bias, lens, mask, groups, eps, act, stats, want_x, want_w, want_b):
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
    dw = torch.empty_like(weight) if want_w else None
    db = torch.empty_like(bias) if want_b else None
    lib = L.lib()
    nws = lib.vqhip_group_norm_workspace_bytes(*x.shape, groups)
    ws = torch.empty(nws, dtype=torch.uint8, device=x.device)
    s = _struct(x, weight, bias, lens, mask, groups, eps, act, stats.data_ptr(), ws.data_ptr(), nws)
    L._check(lib.vqhip_group_norm_bwd(ctypes.byref(s), _addr(grad), _addr(dx), _addr(dw), _addr(db), L._stream()), "vqhip_group_norm_bwd")
    return dx, dw, db


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lens, mask, groups, eps, act):
        y, stats = _forward(x, weight, bias, lens, mask, groups, eps, act, True)
        ctx.save_for_backward(x, weight, bias, lens, mask, stats)
        ctx.args = groups, eps, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, bias, lens, mask, stats = ctx.saved_tensors
        L._no_tangent("group_norm's backward", (grad,))
        dx, dw, db = _backward(grad.resolve_neg().contiguous(), x, weight, bias, lens, mask, *ctx.args, stats, *ctx.needs_input_grad[:3])
        return dx, dw, db, None, None, None, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5, activation: Optional[str] = None, mask: Optional[torch.Tensor] = None,
               lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [b, ..., c] (float32 / bfloat16 / float16), channels last -> act(norm(x) * weight + bias), contiguous, x's shape and type.

    Mean and variance of each of the `num_groups` channel groups over all positions of a batch entry, in 32 bits or more, whatever x's
    type; activation None or 'silu'.  weight, bias [c]: both of one type, float32 or x's, either may be left out.  At most 2^22 entries and 8192
    channels.
    mask / lens: as in VectorQuantize.forward for x [b, n, c] -- bool [b, n], or the number of live rows [b] (integers; more than n counts as
    n, less than 1 as none).  Padding rows take no part in the statistics, may hold anything, and give zeros, gradients as well."""
    L._elem_code(x, "group_norm")
    if x.ndim < 2:
        raise L.VQHipError(f"group_norm: x {tuple(x.shape)}, expected [b, ..., c]")
    b, c = x.shape[0], x.shape[-1]
    if c < 1 or c > NORM_MAX_C or num_groups < 1 or c % num_groups:
        raise L.VQHipError(f"group_norm: {c} channels in {num_groups} groups: takes 1 to {NORM_MAX_C} channels in groups of one size")
    if activation not in _ACTIVATIONS:
        raise L.VQHipError(f"group_norm: activation {activation!r}, takes {tuple(_ACTIVATIONS)}")
    if not eps >= 0.0:
        raise L.VQHipError(f"group_norm: eps {eps}")
    for p in (weight, bias):
        if p is not None and (p.shape != (c,) or p.dtype not in (torch.float32, x.dtype)):
            raise L.VQHipError(f"group_norm: parameter {tuple(p.shape)} {p.dtype}, expected ({c},) float32 or {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise L.VQHipError(f"group_norm: weight of {weight.dtype}, bias of {bias.dtype}")
    if mask is not None and lens is not None:
        raise L.VQHipError("group_norm: mask and lens")
    if mask is not None and (x.ndim != 3 or mask.dtype != torch.bool or tuple(mask.shape) != tuple(x.shape[:2])):
        raise L.VQHipError(f"group_norm: mask {tuple(mask.shape)} {mask.dtype} for x {tuple(x.shape)}, expected bool [b, n] for [b, n, c]")
    if lens is not None and (x.ndim != 3 or lens.dtype not in (torch.int64, torch.int32) or tuple(lens.shape) != (b,)):
        raise L.VQHipError(f"group_norm: lens {tuple(lens.shape)} {lens.dtype} for x {tuple(x.shape)}, expected integers [b] for [b, n, c]")
    L._no_tangent("group_norm", (x, weight, bias))
    L._need_gpu(x, weight, bias, mask, lens)
    x = x.resolve_neg()                                     # (the library reads memory, where torch leaves a negation pending in a flag)
    rows = x if x.ndim == 3 else x.flatten(1, -2) if x.ndim > 3 else x[:, None]
    if rows.stride(-1) != 1 and c > 1:
        rows = rows.contiguous()
    if weight is not None:
        weight = weight.resolve_neg().contiguous()
    if bias is not None:
        bias = bias.resolve_neg().contiguous()
    mk = None if mask is None else mask.contiguous().view(torch.uint8)
    ln = None if lens is None else lens.to(torch.int64).contiguous()
    args = (rows, weight, bias, ln, mk, num_groups, float(eps), _ACTIVATIONS[activation])
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        y = _GroupNormFn.apply(*args)
    else:
        y, _ = _forward(*args, False)
    return y if x.ndim == 3 else y.view(x.shape)


class GroupNorm(nn.Module):
    """`group_norm` with its parameters (names and shapes of torch.nn.GroupNorm's).  Takes [b, ..., c], with channel_last=False [b, c, n] and
    with accept_image_fmap [b, c, h, w] -- VectorQuantize's conventions.  A map in torch's channels_last memory format is read in place
    and comes back in that format, which is the layout a quantizer with accept_image_fmap reads without a copy."""

    def __init__(self, num_groups: int, dim: int, eps: float = 1e-5, affine: bool = True, activation: Optional[str] = None,
                 channel_last: bool = True, accept_image_fmap: bool = False):
        super().__init__()
        if dim < 1 or num_groups < 1 or dim % num_groups:
            raise L.VQHipError(f"GroupNorm: {dim} channels in {num_groups} groups")
        if activation not in _ACTIVATIONS:
            raise L.VQHipError(f"GroupNorm: activation {activation!r}, takes {tuple(_ACTIVATIONS)}")
        self.num_groups, self.dim, self.eps, self.activation = num_groups, dim, eps, activation
        self.channel_last, self.accept_image_fmap = channel_last, accept_image_fmap
        self.weight = nn.Parameter(torch.ones(dim)) if affine else None
        self.bias = nn.Parameter(torch.zeros(dim)) if affine else None

    def extra_repr(self):
        return f"{self.num_groups}, {self.dim}, eps={self.eps}, activation={self.activation}"

    def forward(self, x, mask=None, lens=None):
        first = self.accept_image_fmap or not self.channel_last
        if first:
            if x.ndim != (4 if self.accept_image_fmap else 3):
                raise L.VQHipError(f"GroupNorm: x {tuple(x.shape)}, expected {'[b, c, h, w]' if self.accept_image_fmap else '[b, c, n]'}")
            x = x.movedim(1, -1)
        y = group_norm(x, self.num_groups, self.weight, self.bias, eps=self.eps, activation=self.activation, mask=mask, lens=lens)
        return y.movedim(-1, 1) if first else y
