"""What a decoder computes around its attention, on MI355X: the residual's
addition with the root-mean-square norm, and the log probabilities of tokens.

* ``add_rms_norm`` / ``add_rms_norm_q8``: ``x + branch`` and the norm of the
  sum in one pass (the reference adds and norms in ``Block.forward``,
  nsa_model.py:449-452), for training, and with rows in 8 bits for inference.
  ``NSATransformer(norm='rms', norm_impl='fused')`` runs its blocks on it.
* ``token_logprobs``: log probabilities of given tokens, the entropy and the
  best alternatives of every row of logits, with the gradient; the loss over
  the vocabulary (nsa_model.py:504-507) is their mean.
  ``NSATransformer(loss_impl='fused')`` and ``NSATransformer.score`` use it.

Tensors are float32 or bfloat16 on the GPU, at any alignment of their elements;
rows that are not dense are made contiguous.  Sums and statistics are float32.
Violations raise ``AssertionError``; a missing library raises ``RuntimeError``.
Every call launches on the current stream of its tensors' device, allocates
its outputs and workspace with torch, and never waits for the host: calls can
be captured into a graph.
"""

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

import _nsa_lib as L
import nsa_hip_ops as _ops

_FLOATS = (torch.float32, torch.bfloat16)
TOP_MAX = 64     # most alternatives of a row


def _check(t, what):
    assert t.is_cuda, f"{what}: a GPU tensor is needed"
    assert t.dtype in _FLOATS, f"{what}: dtype {t.dtype} is not supported (float32 or bfloat16)"


def _code(dtype):
    return {torch.float32: L.NSA_F32, torch.bfloat16: L.NSA_BF16, torch.float8_e4m3fn: L.NSA_E4M3}[dtype]


# ---------------------------------------------------------------------------
# residual addition with root-mean-square norm
# ---------------------------------------------------------------------------

def _norm_args(x, residual, weight, eps, what):
    _check(x, f"{what}: x")
    _check(weight, f"{what}: weight")
    assert x.dim() >= 1 and x.shape[-1] >= 1, f"{what}: x must be [..., D]"
    assert weight.shape == x.shape[-1:], f"{what}: weight must be [D]"
    assert weight.device == x.device, f"{what}: x and weight on different devices"
    if residual is not None:
        _check(residual, f"{what}: residual")
        assert residual.shape == x.shape and residual.device == x.device, f"{what}: residual must be like x"
    if eps is None:
        eps = torch.finfo(x.dtype if residual is None else residual.dtype).eps
    assert eps >= 0, f"{what}: eps must not be negative"
    return float(eps)


def _norm_fwd(x, residual, weight, eps, out_dtype, want_rstd):
    """-> (y, h, scale, rstd); h is x without a residual."""
    x, weight = x.contiguous(), weight.contiguous()
    D, rows = x.shape[-1], x.numel() // x.shape[-1]
    res = None if residual is None else residual.contiguous()
    h = x if res is None else torch.empty_like(res)
    y = torch.empty(x.shape, device=x.device, dtype=out_dtype)
    f32 = dict(device=x.device, dtype=torch.float32)
    scale = torch.empty(x.shape[:-1], **f32) if out_dtype == torch.float8_e4m3fn else None
    rstd = torch.empty(rows, **f32) if want_rstd else None
    with _ops.device_of(x):
        _ops._call("nsa_norm_fwd", _ops._lib().nsa_norm_fwd, L.ptr(x), L.ptr(res), L.ptr(weight),
                   L.ptr(None if res is None else h), L.ptr(y), L.ptr(scale), L.ptr(rstd), rows, D, eps,
                   _code(x.dtype), _code(h.dtype), _code(weight.dtype), _code(out_dtype), _ops._stream(x))
    return y, h, scale, rstd


class AddRmsNormHIP(torch.autograd.Function):
    """``(y, h)`` of ``add_rms_norm``; ``residual`` None gives y alone."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, out_dtype):
        ctx.set_materialize_grads(False)
        y, h, _, rstd = _norm_fwd(x, residual, weight, eps, out_dtype, any(ctx.needs_input_grad))
        ctx.save_for_backward(h, weight, rstd)
        ctx.meta = (x.dtype, residual is not None)
        return y if residual is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        x_dt, added = ctx.meta
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if dy is None:       # only the sum was used: its gradient passes through
            if dh is None:
                return None, None, None, None, None
            return (dh.to(x_dt) if need_x else None, dh if need_r else None,
                    torch.zeros_like(weight) if need_w else None, None, None)
        D, rows = h.shape[-1], h.numel() // h.shape[-1]
        h, weight, dy = h.contiguous(), weight.contiguous(), dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        dx = torch.empty(h.shape, device=h.device, dtype=x_dt)
        dres = torch.empty_like(h) if added and x_dt != h.dtype else None
        dw = torch.empty_like(weight) if need_w else None
        if rows == 0:
            return dx, dres if dres is not None else (dx if added else None), \
                torch.zeros_like(weight) if need_w else None, None, None
        with _ops.device_of(h):
            nbytes = int(_ops._lib().nsa_norm_bwd_workspace(rows, D, _ops._stream(h))) if need_w else 0
            ws = torch.empty(nbytes, device=h.device, dtype=torch.uint8) if need_w else None
            _ops._call("nsa_norm_bwd", _ops._lib().nsa_norm_bwd, L.ptr(dy), L.ptr(dh), L.ptr(h), L.ptr(weight),
                       L.ptr(rstd), L.ptr(dx), L.ptr(dres), L.ptr(dw), L.ptr(ws), nbytes, rows, D, _code(x_dt),
                       _code(h.dtype), _code(weight.dtype), _code(dy.dtype), _ops._stream(h))
        dr = None if not added else dx if dres is None else dres
        return dx, dr, dw, None, None


def add_rms_norm(x, residual, weight, eps=None, out_dtype=None):
    """``h = x + residual`` and ``y = h / sqrt(mean(h^2) + eps) * weight`` over
    the last dimension -> ``(y, h)``.

    ``x [..., D]`` is a branch's output and ``residual`` (same shape, or None:
    ``h`` is ``x`` itself) the stream it joins; each of x, residual and weight
    may be float32 or bfloat16 on its own.  The sum is formed in float32 and
    rounded once to the residual's dtype; the norm is taken of the rounded
    sum.  ``y`` is in ``out_dtype`` (default: h's dtype).  ``eps`` None is the
    machine epsilon of h's dtype, as in ``torch.nn.RMSNorm``.  Differentiable
    in x, residual and weight, from y and h; the weight's gradient has the
    same bits on every run."""
    eps = _norm_args(x, residual, weight, eps, "add_rms_norm")
    if out_dtype is None:
        out_dtype = x.dtype if residual is None else residual.dtype
    assert out_dtype in _FLOATS, "add_rms_norm: out_dtype must be float32 or bfloat16"
    if residual is None:
        return AddRmsNormHIP.apply(x, None, weight, eps, out_dtype), x
    return AddRmsNormHIP.apply(x, residual, weight, eps, out_dtype)


def add_rms_norm_q8(x, residual, weight, eps=None):
    """``add_rms_norm`` with the rows in 8 bits, for products in 8 bits:
    ``(q, scale, h)`` with ``q [..., D]`` float8_e4m3fn and ``scale [...]``
    float32, ``y ~ q * scale[..., None]``.

    A row's scale is its largest ``|y|`` (2^-100 at least) over 448; values are
    rounded once, to nearest even.  A row that holds NaN or an infinity has a
    NaN or infinite scale.  For inference: inputs that need a gradient are
    refused."""
    eps = _norm_args(x, residual, weight, eps, "add_rms_norm_q8")
    assert not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight))), \
        "add_rms_norm_q8 has no gradient: call it under torch.no_grad()"
    y, h, scale, _ = _norm_fwd(x, residual, weight, eps, torch.float8_e4m3fn, False)
    return y, scale, x if residual is None else h


# ---------------------------------------------------------------------------
# log probabilities of tokens
# ---------------------------------------------------------------------------

class TokenLogprobs(NamedTuple):
    """Per row of logits: ``logp`` (None without targets), ``entropy``, and with
    ``top`` > 0 the alternatives' ``top_logp`` and ``top_idx`` (else None)."""

    logp: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_idx: Optional[torch.Tensor]


class TokenLogprobsHIP(torch.autograd.Function):
    """``(logp, entropy, top_logp, top_idx)`` of dense ``z [rows, V]``."""

    @staticmethod
    def forward(ctx, z, targets, top):
        ctx.set_materialize_grads(False)
        z = z.contiguous()
        rows, V = z.shape
        f32 = dict(device=z.device, dtype=torch.float32)
        logp = None if targets is None else torch.empty(rows, **f32)
        ent, stat = torch.empty(rows, **f32), torch.empty(rows, 2, **f32)
        top_logp = torch.empty(rows, top, **f32)
        top_idx = torch.empty(rows, top, device=z.device, dtype=torch.int64)
        with _ops.device_of(z):
            nbytes = int(_ops._lib().nsa_logprob_workspace(rows, V, top, _ops._stream(z)))
            assert nbytes > 0, "token_logprobs: unsupported shape"
            ws = torch.empty(nbytes, device=z.device, dtype=torch.uint8)
            _ops._call("nsa_logprob_fwd", _ops._lib().nsa_logprob_fwd, L.ptr(z), L.ptr(targets), L.ptr(logp),
                       L.ptr(ent), L.ptr(stat), L.ptr(top_logp), L.ptr(top_idx), L.ptr(ws), nbytes, rows, V, top,
                       _code(z.dtype), _ops._stream(z))
        ctx.save_for_backward(z, targets, stat, ent)
        ctx.mark_non_differentiable(top_logp, top_idx)
        return logp, ent, top_logp, top_idx

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dent, _dtop, _didx):
        z, targets, stat, ent = ctx.saved_tensors
        if dlogp is None and dent is None:
            return None, None, None
        rows, V = z.shape
        dz = torch.empty_like(z)
        dlogp, dent = (None if d is None else d.float().contiguous() for d in (dlogp, dent))
        with _ops.device_of(z):
            _ops._call("nsa_logprob_bwd", _ops._lib().nsa_logprob_bwd, L.ptr(z), L.ptr(targets), L.ptr(stat),
                       L.ptr(ent), L.ptr(dlogp), L.ptr(dent), L.ptr(dz), rows, V, _code(z.dtype), _ops._stream(z))
        return dz, None, None


def token_logprobs(logits, targets=None, top=0):
    """Log probabilities under ``softmax(logits)`` over the last dimension of
    ``logits [..., V]`` -> ``TokenLogprobs``.

    ``targets [...]`` (an integer dtype): ``logp [...]`` is the log probability
    of each row's target; a target outside ``0 .. V-1`` (``-100`` included)
    leaves 0 and no gradient.  ``entropy [...]`` is ``-sum p ln p``.  ``top``
    (at most 64 and V) alternatives: ``top_logp [..., top]`` in descending
    order and their tokens ``top_idx`` (int64), equal logits by ascending
    token; NaN counts above every number.  All results are float32.

    A logit of -inf (a banned token) has probability 0 and adds nothing to
    the entropy; a row of nothing else has ``logp`` and ``top_logp`` -inf,
    entropy 0 and no gradient.  Rows that hold NaN or +inf give NaN.
    Differentiable in the logits, from ``logp`` and ``entropy``."""
    _check(logits, "token_logprobs: logits")
    assert logits.dim() >= 1 and logits.shape[-1] >= 1, "token_logprobs: logits must be [..., V]"
    V, lead = logits.shape[-1], logits.shape[:-1]
    assert isinstance(top, int) and 0 <= top <= min(TOP_MAX, V), "token_logprobs: top must be 0 .. min(64, V)"
    if targets is not None:
        assert targets.is_cuda and targets.device == logits.device, "token_logprobs: targets on the logits' device"
        assert targets.dtype in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8), \
            "token_logprobs: targets must be integers"
        assert targets.shape == lead, "token_logprobs: one target for each row"
        targets = targets.reshape(-1).long().contiguous()
    logp, ent, top_logp, top_idx = TokenLogprobsHIP.apply(logits.reshape(-1, V), targets, top)
    return TokenLogprobs(None if logp is None else logp.view(lead), ent.view(lead),
                         top_logp.view(*lead, top) if top else None, top_idx.view(*lead, top) if top else None)
