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
_CODE = {torch.float32: L.NSA_F32, torch.bfloat16: L.NSA_BF16, torch.float8_e4m3fn: L.NSA_E4M3}
TOP_MAX = 64     # most alternatives of a row


def _check(t, what):
    assert t.is_cuda, f"{what}: a GPU tensor is needed"
    assert t.dtype in _FLOATS, f"{what}: dtype {t.dtype} is not supported (float32 or bfloat16)"


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---------------------------------------------------------------------------
# residual addition with root-mean-square norm
# ---------------------------------------------------------------------------

def _norm_args(x, residual, weight, eps, what):
    _check(x, f"{what}: x")
    _check(weight, f"{what}: weight")
    D = x.shape[-1] if x.dim() else 0
    assert 1 <= D <= 1 << 24, f"{what}: x must be [..., D]"
    assert weight.shape == (D,), f"{what}: weight must be [D]"
    assert weight.device == x.device, f"{what}: x and weight on different devices"
    if residual is not None:
        _check(residual, f"{what}: residual")
        assert residual.shape == x.shape and residual.device == x.device, f"{what}: residual must be like x"
    if eps is None:
        eps = torch.finfo(x.dtype if residual is None else residual.dtype).eps
    assert eps >= 0, f"{what}: eps must not be negative"
    return eps


def _norm_fwd(x, residual, weight, eps, out_dtype, want_rstd):
    """-> (y, h, scale, rstd); h is x without a residual."""
    x, weight = x.contiguous(), weight.contiguous()
    D = x.shape[-1]
    rows = x.numel() // D
    if residual is None:
        h, r_at, h_at = x, None, None
    else:
        residual = residual.contiguous()
        h = torch.empty_like(residual)
        r_at, h_at = residual.data_ptr(), h.data_ptr()
    y = torch.empty_like(x, dtype=out_dtype)
    scale = rstd = None
    if out_dtype == torch.float8_e4m3fn:
        scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    if want_rstd:
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
    _ops.launch(x, "nsa_norm_fwd", x.data_ptr(), r_at, weight.data_ptr(), h_at, y.data_ptr(), L.addr(scale),
                L.addr(rstd), rows, D, eps, _CODE[x.dtype], _CODE[h.dtype], _CODE[weight.dtype], _CODE[out_dtype])
    return y, h, scale, rstd


def _norm_bwd(ctx, dy, dh=None):
    h, weight, rstd = ctx.saved_tensors
    x_dt, added = ctx.meta
    need_x, need_r, need_w = ctx.needs_input_grad[:3]
    if dy is None:       # only the sum was used: its gradient passes through
        if dh is None:
            return None, None, None, None, None
        return (dh.to(x_dt) if need_x else None, dh if need_r else None, torch.zeros_like(weight) if need_w else None,
                None, None)
    D = h.shape[-1]
    rows = h.numel() // D
    dy = dy.contiguous()
    dh = None if dh is None else dh.contiguous()
    dx = torch.empty_like(h, dtype=x_dt)
    dr = dx if added else None
    if added and x_dt != h.dtype:
        dr = torch.empty_like(h)
    if rows == 0:
        return dx, dr, torch.zeros_like(weight) if need_w else None, None, None
    dw = ws = None
    nbytes = 0
    if need_w:
        dw = torch.empty_like(weight)
        nbytes = _ops.workspace_bytes(h.get_device(), "nsa_norm_bwd_workspace", rows, D)
        ws = torch.empty(nbytes, device=h.device, dtype=torch.uint8)
    _ops.launch(h, "nsa_norm_bwd", dy.data_ptr(), L.addr(dh), h.data_ptr(), weight.data_ptr(), rstd.data_ptr(),
                dx.data_ptr(), None if dr is dx else L.addr(dr), L.addr(dw), L.addr(ws), nbytes, rows, D,
                _CODE[x_dt], _CODE[h.dtype], _CODE[weight.dtype], _CODE[dy.dtype])
    return dx, dr, dw, None, None


class AddRmsNormHIP(torch.autograd.Function):
    """``(y, h)`` of ``add_rms_norm``; ``residual`` None gives y alone."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, out_dtype):
        ctx.set_materialize_grads(False)
        weight = weight.contiguous()
        y, h, _, rstd = _norm_fwd(x, residual, weight, eps, out_dtype, True)
        ctx.save_for_backward(h, weight, rstd)
        ctx.meta = (x.dtype, residual is not None)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():      # (create_graph: a second derivative is refused when it is taken)
            return once_differentiable(_norm_bwd)(ctx, *grads)
        return _norm_bwd(ctx, *grads)


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
    if not _wants_grad(x, residual, weight):
        y, h, _, _ = _norm_fwd(x, residual, weight, eps, out_dtype, False)
        return y, x if residual is None else h
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
    assert not _wants_grad(x, residual, weight), "add_rms_norm_q8 has no gradient: call it under torch.no_grad()"
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


def _logprob_fwd(z, targets, top, want_stat):
    """-> (logp, entropy, top_logp, top_idx, stat) of dense ``z [rows, V]``."""
    rows, V = z.shape
    dev, f32 = z.device, torch.float32
    logp = None if targets is None else torch.empty(rows, device=dev, dtype=f32)
    ent = torch.empty(rows, device=dev, dtype=f32)
    stat = torch.empty(rows, 2, device=dev, dtype=f32) if want_stat else None
    top_logp = top_idx = None
    if top:
        top_logp = torch.empty(rows, top, device=dev, dtype=f32)
        top_idx = torch.empty(rows, top, device=dev, dtype=torch.int64)
    nbytes = _ops.workspace_bytes(z.get_device(), "nsa_logprob_workspace", rows, V, top)
    assert nbytes > 0, "token_logprobs: unsupported shape"
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes > 16 else None
    _ops.launch(z, "nsa_logprob_fwd", z.data_ptr(), L.addr(targets), L.addr(logp), ent.data_ptr(), L.addr(stat),
                L.addr(top_logp), L.addr(top_idx), L.addr(ws), nbytes, rows, V, top, _CODE[z.dtype])
    return logp, ent, top_logp, top_idx, stat


def _logprob_bwd(ctx, dlogp, dent, _dtop=None, _didx=None):
    z, targets, stat, ent = ctx.saved_tensors
    if dlogp is None and dent is None:
        return None, None, None
    rows, V = z.shape
    dz = torch.empty_like(z)
    dlogp = None if dlogp is None else dlogp.contiguous()
    dent = None if dent is None else dent.contiguous()
    _ops.launch(z, "nsa_logprob_bwd", z.data_ptr(), L.addr(targets), stat.data_ptr(), ent.data_ptr(), L.addr(dlogp),
                L.addr(dent), dz.data_ptr(), rows, V, _CODE[z.dtype])
    return dz, None, None


class TokenLogprobsHIP(torch.autograd.Function):
    """``(logp, entropy, top_logp, top_idx)`` of dense ``z [rows, V]``."""

    @staticmethod
    def forward(ctx, z, targets, top):
        ctx.set_materialize_grads(False)
        logp, ent, top_logp, top_idx, stat = _logprob_fwd(z, targets, top, True)
        ctx.save_for_backward(z, targets, stat, ent)
        if top:
            ctx.mark_non_differentiable(top_logp, top_idx)
        return logp, ent, top_logp, top_idx

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():      # (create_graph: a second derivative is refused when it is taken)
            return once_differentiable(_logprob_bwd)(ctx, *grads)
        return _logprob_bwd(ctx, *grads)


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
        if targets.dim() != 1 or targets.dtype != torch.int64 or not targets.is_contiguous():
            targets = targets.reshape(-1).long().contiguous()
    z = logits if logits.dim() == 2 and logits.is_contiguous() else logits.reshape(-1, V).contiguous()
    if _wants_grad(logits):
        logp, ent, top_logp, top_idx = TokenLogprobsHIP.apply(z, targets, top)
    else:
        logp, ent, top_logp, top_idx, _ = _logprob_fwd(z, targets, top, False)
    if len(lead) == 1:
        return TokenLogprobs(logp, ent, top_logp, top_idx)
    return TokenLogprobs(None if logp is None else logp.view(lead), ent.view(lead),
                         top_logp.view(*lead, top) if top else None, top_idx.view(*lead, top) if top else None)
