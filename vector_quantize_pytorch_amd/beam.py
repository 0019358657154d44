"""Beam search over codes, or over any vocabulary: the selection over beams and continuations (`beam_select`) and the reordering of
the beams' states (`beam_reorder`), both differentiable.  `ResidualVQ.forward(beam_size=)` runs on them (reference: rvq.py:493-562).

    logits = model(tokens, caches)                                        # [b, beams, vocabulary]
    step = beam_select(logits, scores, beam_size, finished=finished, end_token=end)
    caches = beam_reorder(caches, step.parents)                           # every state [b, beams, ...] follows its beam
    scores, tokens = step.scores, step.tokens                             # [b, beam_size]
"""
from __future__ import annotations

import array
import ctypes
import math
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib as L

BEAM_MAX = 64            # VQHIP_BEAM_MAX: beams before and after a selection
_STATES = 32             # VQHIP_BEAM_STATES: states of one launch

_i64, _vp = ctypes.c_int64, ctypes.c_void_p


class BeamStep(NamedTuple):
    """the survivors of a selection, best first: accumulated scores (fp32), the beams they continue and the chosen continuations"""
    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor


class _Select(ctypes.Structure):                         # vqhip_beam_select_t
    _fields_ = [("logits", _vp), ("dtype", _i64), ("B", _i64), ("J", _i64), ("V", _i64), ("stride_b", _i64), ("stride_j", _i64),
                ("scores", _vp), ("mask", _vp), ("mask_stride_b", _i64), ("mask_stride_j", _i64), ("finished", _vp), ("end_token", _i64),
                ("normalize", _i64), ("K", _i64), ("out_scores", _vp), ("parents", _vp), ("tokens", _vp), ("lse", _vp),
                ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t)]


class _State(ctypes.Structure):                          # vqhip_beam_state_t
    _fields_ = [("src", _vp), ("dst", _vp), ("stride_b", _i64), ("stride_j", _i64), ("pieces", _i64), ("piece_stride", _i64),
                ("piece_bytes", _i64)]


def _addr(t):
    return None if t is None else t.data_ptr()


def _table(t: torch.Tensor, b: int, j: int, v: int) -> torch.Tensor:
    """t [..., j, v] as [b, j, v] with contiguous continuations, without a copy where the layout allows it"""
    if t.ndim != 3:
        t = t.reshape(b, j, v)
    if t.is_contiguous():
        return t
    return t if t.stride(-1) == 1 or v == 1 else t.contiguous()


@L._on_device
def _select(logits, scores, mask, finished, beam_size, end_token, normalize, want_lse):
    b, j, v = logits.shape
    dev = logits.device
    lib = L.lib()
    out = torch.empty((b, beam_size), dtype=torch.float32, device=dev)
    # (tensors of their own: views of one would share its version, and an edit of the tokens would stop the backward of a reordering)
    parents, tokens = torch.empty((b, beam_size), dtype=torch.int64, device=dev), torch.empty((b, beam_size), dtype=torch.int64, device=dev)
    lse = torch.empty((b, j), dtype=torch.float64, device=dev) if want_lse else None
    nws = lib.vqhip_beam_select_workspace_bytes(b, j, v, beam_size)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    s = _struct(logits, scores, mask, finished, end_token, normalize, out, parents, tokens, lse, ws, nws)
    L._check(lib.vqhip_beam_select(ctypes.byref(s), L._stream()), "vqhip_beam_select")
    return out, parents, tokens, lse


def _struct(logits, scores, mask, finished, end_token, normalize, out, parents, tokens, lse, ws=None, nws=0):
    b, j, v = logits.shape
    sb, sj, _ = logits.stride()
    mb, mj, _ = (0, 0, 0) if mask is None else mask.stride()
    return _Select(logits.data_ptr(), L._ELEM_CODES[logits.dtype], b, j, v, sb, sj, _addr(scores), _addr(mask), mb, mj, _addr(finished), end_token,
                   normalize, out.shape[1], out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), _addr(lse), _addr(ws), nws)


@L._on_device
def _select_bwd(grad, logits, mask, finished, end_token, normalize, out, parents, tokens, lse, want_logits, want_scores):
    b, j, v = logits.shape
    d_logits = torch.empty(b, j, v, dtype=logits.dtype, device=logits.device) if want_logits else None
    d_scores = torch.empty(b, j, dtype=torch.float32, device=logits.device) if want_scores else None
    s = _struct(logits, None, mask, finished, end_token, normalize, out, parents, tokens, lse)
    L._check(L.lib().vqhip_beam_select_bwd(ctypes.byref(s), _addr(grad), _addr(d_logits), _addr(d_scores), L._stream()), "vqhip_beam_select_bwd")
    return d_logits, d_scores


class _SelectFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, scores, mask, finished, beam_size, end_token, normalize):
        out, parents, tokens, lse = _select(logits, scores, mask, finished, beam_size, end_token, normalize, normalize)
        ctx.save_for_backward(logits, mask, finished, out, parents, tokens, lse)
        ctx.end_token, ctx.normalize = end_token, normalize
        ctx.mark_non_differentiable(parents, tokens)
        ctx.set_materialize_grads(False)
        return out, parents, tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _parents, _tokens):
        if grad is None:
            return (None,) * 7
        L._no_tangent("beam_select's backward", (grad,))
        logits, mask, finished, out, parents, tokens, lse = ctx.saved_tensors
        d_logits, d_scores = _select_bwd(grad.resolve_neg().contiguous(), logits, mask, finished, ctx.end_token, ctx.normalize, out, parents, tokens, lse,
                                         ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return d_logits, d_scores, None, None, None, None, None


def beam_select(logits: torch.Tensor, scores: Optional[torch.Tensor], beam_size: int, *, mask: Optional[torch.Tensor] = None,
                finished: Optional[torch.Tensor] = None, end_token: Optional[int] = None, normalize: bool = True) -> BeamStep:
    """The `beam_size` best of all continuations of all beams.

    logits [..., beams, vocabulary] (float32 / bfloat16 / float16), scores [..., beams] float32 (None: zeros): continuation v of beam j
    scores `scores[j] + log_softmax(logits[j])[v]`, or `scores[j] + logits[j, v]` with normalize=False (negative errors of codes, say).
    -> BeamStep(scores, parents, tokens), each [..., beam_size], best first; equal scores by ascending beam, then ascending token.

    mask      bool, broadcastable to logits: False leaves a continuation out -- of the softmax as well; its logits may hold anything (one that
              is broadcast over the vocabulary is copied to that size)
    finished  bool [..., beams]: such a beam is kept as it is, as its own only continuation `end_token`
    A score that is not a number counts as -inf: a beam whose logits hold NaN or +inf, or whose mask leaves nothing, has no
    continuation (normalize=True).  Where fewer than beam_size continuations are left, the last survivors have a score of -inf.
    Gradients reach logits and scores through the returned scores (backward mode); survivors of score -inf pass none on.  The backward reads the
    returned tensors: where one follows, edit copies of them."""
    L._elem_code(logits, "beam_select")
    if logits.ndim < 2:
        raise L.VQHipError(f"beam_select: logits {tuple(logits.shape)}, expected [..., beams, vocabulary]")
    *lead, j, v = logits.shape
    rows = logits.shape[:-1]
    if scores is not None and (scores.shape != rows or scores.dtype != torch.float32):
        raise L.VQHipError(f"beam_select: scores {tuple(scores.shape)} {scores.dtype}, expected {tuple(rows)} float32")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise L.VQHipError(f"beam_select: mask of {mask.dtype}, expected bool")
        try:
            mask = mask.expand(logits.shape)
        except RuntimeError:
            raise L.VQHipError(f"beam_select: mask {tuple(mask.shape)} does not broadcast to {tuple(logits.shape)}") from None
    if finished is not None:
        if finished.shape != rows or finished.dtype != torch.bool:
            raise L.VQHipError(f"beam_select: finished {tuple(finished.shape)} {finished.dtype}, expected {tuple(rows)} bool")
        if end_token is None or not 0 <= end_token < v:
            raise L.VQHipError(f"beam_select: finished beams need an end_token in [0, {v}), got {end_token}")
    if j < 1 or v < 1 or j > BEAM_MAX or not 1 <= beam_size <= min(BEAM_MAX, j * v):
        raise L.VQHipError(f"beam_select: {beam_size} survivors of {j} x {v} continuations: takes 1 to {BEAM_MAX} beams and survivors, "
                           "no more survivors than continuations")
    n = lead[0] if len(lead) == 1 else math.prod(lead)
    L._no_tangent("beam_select", (logits, scores))
    grad = torch.is_grad_enabled() and (logits.requires_grad or (scores is not None and scores.requires_grad))
    L._need_gpu(logits, scores, mask, finished)
    beam_size = int(beam_size)
    lg = _table(logits.resolve_neg(), n, j, v)              # (the library reads memory, where torch leaves a negation pending in a flag)
    sc = None if scores is None else scores.resolve_neg().contiguous()
    if sc is not None and len(lead) != 1:
        sc = sc.view(n, j)
    mk = None if mask is None else _table(mask, n, j, v).view(torch.uint8)
    fin = None if finished is None else finished.reshape(n, j).contiguous().view(torch.uint8)
    end = 0 if finished is None else int(end_token)
    if grad:
        out, parents, tokens = _SelectFn.apply(lg, sc, mk, fin, beam_size, end, bool(normalize))
    else:
        out, parents, tokens, _ = _select(lg, sc, mk, fin, beam_size, end, bool(normalize), False)
    if len(lead) != 1:
        out, parents, tokens = (t.view(*lead, beam_size) for t in (out, parents, tokens))
    return BeamStep(out, parents, tokens)


# ---- states ---------------------------------------------------------------------------------------------------------------------
def _collapse(sizes, strides):
    """(count, stride) of dims that lie behind each other like one, None where they do not"""
    n, st = 1, 0
    for d, s in zip(reversed(sizes), reversed(strides)):
        if d == 1:
            continue
        if n == 1:
            n, st = d, s
        elif s == n * st:
            n *= d
        else:
            return None
    return n, st


def _layout(t: torch.Tensor, nlead: int):
    """t [*lead, beams, ...] -> (t or its contiguous copy, batch stride, beam stride, pieces, piece stride, elements of a piece)"""
    if t.is_contiguous():
        run = math.prod(t.shape[nlead + 1:])
        return t, run * t.shape[nlead], run, 1, 0, run
    shape, strides = t.shape, t.stride()
    lead = _collapse(shape[:nlead], strides[:nlead])
    inner, inner_st = list(shape[nlead + 1:]), list(strides[nlead + 1:])
    run = 1
    while inner and (inner[-1] == 1 or inner_st[-1] == run):
        run *= inner.pop()
        inner_st.pop()
    pieces = _collapse(inner, inner_st)
    if lead is None or pieces is None:
        return _layout(t.contiguous(), nlead)
    return t, lead[1], strides[nlead], pieces[0], pieces[1], run


def _flagged(tensors):
    """whether a tensor's values are not what its memory holds: conj(), and the imaginary part of its result, only set a flag"""
    return any(map(torch.Tensor.is_conj, tensors)) or any(map(torch.Tensor.is_neg, tensors))


def _resolved(states):
    return [s.resolve_conj().resolve_neg() for s in states] if _flagged(states) else states


def _extent(t):
    """[first byte, behind the last byte) of a tensor's memory"""
    n, first = t.numel(), t.data_ptr()
    span = n if n == 0 or t.is_contiguous() else sum((d - 1) * s for d, s in zip(t.shape, t.stride())) + 1
    return first, first + span * t.element_size()


@L._on_device
def _reorder(parents, states, outs):
    nlead, k = parents.ndim - 1, parents.shape[-1]
    n, j = parents.numel() // k, states[0].shape[nlead]
    keep, flat, last = [], [], None                          # flat: vqhip_beam_state_t rows
    for s, o in zip(states, outs):
        if s.numel() == 0:
            continue
        key = s.shape, s.stride(), s.dtype
        if key == last:                                      # the caches of a model's layers: one layout for all
            t = s
        else:
            t, sb, sj, pieces, ps, run = _layout(s, nlead)
            es = t.element_size()
            form = sb * es, sj * es, pieces, ps * es, run * es
            last = key if t is s else None
            keep.append(t)
        flat += (t.data_ptr(), o.data_ptr(), *form)
    table = array.array("q", flat)
    for i in range(0, len(flat), 7 * _STATES):
        L._check(L.lib().vqhip_beam_reorder(table.buffer_info()[0] + 8 * i, min(_STATES, (len(flat) - i) // 7), _addr(parents), n, j, k, L._stream()),
                 "vqhip_beam_reorder")


@L._on_device
def _reorder_bwd(parents, j, grads):
    nlead, k = parents.ndim - 1, parents.shape[-1]
    n = parents.numel() // k
    lead = parents.shape[:-1]
    grads = [None if g is None else g.resolve_neg().contiguous() for g in grads]
    outs = [None if g is None else torch.empty(*lead, j, *g.shape[nlead + 1:], dtype=g.dtype, device=g.device) for g in grads]
    some = [(g, o) for g, o in zip(grads, outs) if g is not None and o.numel()]
    for i in range(0, len(some), _STATES):
        part = some[i:i + _STATES]
        arr = (_State * len(part))(*[(g.data_ptr(), o.data_ptr(), 0, 0, 1, 0, g.element_size() * (g.numel() // (n * k))) for g, o in part])
        dts = (_i64 * len(part))(*[L._ELEM_CODES[g.dtype] for g, _ in part])
        L._check(L.lib().vqhip_beam_reorder_bwd(arr, dts, len(part), _addr(parents), n, j, k, L._stream()), "vqhip_beam_reorder_bwd")
    return outs


def _results(parents, states):
    """new tensors for the reordered states"""
    outs, nlead, last, lead, device = [], parents.ndim - 1, None, tuple(parents.shape), parents.device
    for s in states:
        if s.shape != last:
            last = s.shape
            shape = lead + last[nlead + 1:]
        outs.append(torch.empty(shape, dtype=s.dtype, device=device))
    return outs


class _ReorderFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, parents, *states):
        nlead, k = parents.ndim - 1, parents.shape[-1]
        outs = tuple(_results(parents, states))
        _reorder(parents, states, outs)
        ctx.save_for_backward(parents)
        ctx.beams = states[0].shape[nlead]
        ctx.mark_non_differentiable(*[o for o, s in zip(outs, states) if not s.requires_grad])
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        parents, = ctx.saved_tensors
        L._no_tangent("beam_reorder's backward", grads)
        need = ctx.needs_input_grad[1:]
        return (None, *_reorder_bwd(parents, ctx.beams, [g if w else None for g, w in zip(grads, need)]))


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, *, out: Optional[Sequence[torch.Tensor]] = None) -> list:
    """states: tensors [..., beams, *] of any types and shapes behind the beams (caches, residuals, token histories); parents [..., k]
    int64 -> a list of [..., k, *]: row i of every result is row parents[i] of its state, all of them in one launch.  A parent outside
    [0, beams) gives a row of zeros.  States are read in place where their rows are evenly spaced runs (a cache cut to the positions in
    use, `cache[..., :length, :]`), otherwise from a contiguous copy.

    out: contiguous tensors that take the results (the other half of a double buffer); they may not share memory with a state or with
    each other, and neither a state nor a result may require a gradient.  Without it, gradients reach float32, bfloat16 and float16 states:
    beams continued by several rows get the sum, accumulated in 32 bits."""
    states = list(states)
    if parents.dtype != torch.int64 or parents.ndim < 1 or parents.shape[-1] < 1:
        raise L.VQHipError(f"beam_reorder: parents {tuple(parents.shape)} {parents.dtype}, expected int64 [..., k]")
    if not states:
        return []
    nlead = parents.ndim - 1
    j = states[0].shape[nlead] if states[0].ndim > nlead else 0
    device, fits = parents.get_device(), None                # fits: a shape that does
    for s in states:
        if s.get_device() != device:
            raise L.VQHipError(f"beam_reorder: tensors on different devices ({parents.device} and {s.device})")
        if s.shape != fits:
            if s.ndim <= nlead or s.shape[:nlead] != parents.shape[:-1] or s.shape[nlead] != j or j < 1:
                raise L.VQHipError(f"beam_reorder: state {tuple(s.shape)}, expected {tuple(parents.shape[:-1])} + ({j or 'beams'}, ...)")
            fits = s.shape
    L._no_tangent("beam_reorder", states)
    grad = torch.is_grad_enabled() and any(s.requires_grad for s in states)
    if out is None:
        if grad:
            for s in states:
                if s.requires_grad:
                    L._elem_code(s, "beam_reorder: state with a gradient")
        L._need_gpu(parents, *states)
        parents, states = parents.contiguous(), _resolved(states)
        if grad:
            return list(_ReorderFn.apply(parents, *states))
        out = _results(parents, states)
        if parents.numel():
            _reorder(parents, states, out)
    else:
        out = list(out)
        if grad:
            raise L.VQHipError("beam_reorder: out= with states that require a gradient")
        if torch.is_grad_enabled() and any(o.requires_grad for o in out):
            raise L.VQHipError("beam_reorder: a result that requires a gradient")
        if len(out) != len(states):
            raise L.VQHipError(f"beam_reorder: {len(out)} results for {len(states)} states")
        for s, o in zip(states, out):
            if o.shape != (*parents.shape, *s.shape[nlead + 1:]) or o.dtype != s.dtype or o.device != s.device or not o.is_contiguous():
                raise L.VQHipError(f"beam_reorder: out {tuple(o.shape)} {o.dtype}, expected contiguous "
                                   f"{(*parents.shape, *s.shape[nlead + 1:])} {s.dtype} on {s.device}")
        L._no_tangent("beam_reorder", out)
        if _flagged(out):
            raise L.VQHipError("beam_reorder: out with a pending conjugation or negation")
        taken = sorted([(*_extent(t), w) for w, ts in ((0, [*states, parents]), (1, out)) for t in ts if t.numel()])
        end = end_out = -1                                       # behind the last byte of any tensor, of any result so far
        for first, behind, is_out in taken:
            if first < (end if is_out else end_out):
                raise L.VQHipError("beam_reorder: out shares memory with a state, the parents or another result")
            end = max(end, behind)
            end_out = max(end_out, behind) if is_out else end_out
        L._need_gpu(parents, *states)
        parents, states = parents.contiguous(), _resolved(states)
        if parents.numel():
            _reorder(parents, states, out)
            L._written(out)
    return out
