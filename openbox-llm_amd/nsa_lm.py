"""What a decoder computes around its attention, on MI355X: its embedding, the
residual's addition with the norm, and the log probabilities of tokens.

* ``add_rms_norm`` / ``add_rms_norm_q8``: ``x + branch`` and the norm of the
  sum in one pass (the reference adds and norms in ``Block.forward``,
  nsa_model.py:449-452), for training, and with rows in 8 bits for inference.
  ``NSATransformer(norm='rms', norm_impl='fused')`` runs its blocks on it.
* ``token_logprobs``: log probabilities of given tokens, the entropy and the
  best alternatives of every row of logits, with the gradient; the loss over
  the vocabulary (nsa_model.py:504-507) is their mean.
  ``NSATransformer(loss_impl='fused')`` and ``NSATransformer.score`` use it.

* ``add_layer_norm``: the same addition with the reference's own norm
  (nsa_model.py:449-452); ``NSATransformer(norm_impl='joined')``.
* ``embed``: rows of the token table with their positions' rows
  (nsa_model.py:455-511), and both tables' gradients by sorted tokens;
  ``NSATransformer(embed_impl='fused')``.
* ``linear_logprobs``: log probabilities of given tokens from the rows behind the
  last norm, without the logits, with the gradients;
  ``NSATransformer(loss_impl='pieces')``.

Tensors are float32 or bfloat16 on the GPU, at any alignment of their elements;
rows that are not dense are made contiguous.  Sums and statistics are float32.
Violations raise ``AssertionError``; a missing library raises ``RuntimeError``.
Every call launches on the current stream of its tensors' device, allocates
its outputs and workspace with torch, and never waits for the host: calls can
be captured into a graph (a backward, as any torch function's, with no eager
graph of the same leaves alive).  First derivatives only, in reverse mode: dual
tensors are refused.  The checks, allocations and autograd nodes are C++
(csrc/nsa_torch.cpp).
"""

from typing import NamedTuple, Optional

import torch

import _nsa_lib as L
import nsa_hip_ops as _ops


# ---------------------------------------------------------------------------
# residual addition with root-mean-square norm
# ---------------------------------------------------------------------------

def add_rms_norm(x, residual, weight, eps=None, out_dtype=None):
    """``h = x + residual`` and ``y = h / sqrt(mean(h^2) + eps) * weight`` over
    the last dimension -> ``(y, h)``.

    ``x [..., D]`` is a branch's output and ``residual`` (same shape, or None:
    ``h`` is ``x`` itself) the stream it joins; each of x, residual and weight
    may be float32 or bfloat16 on its own.  The sum is formed in float32 and
    rounded once to the residual's dtype; the norm is taken of the rounded
    sum.  ``y`` is in ``out_dtype`` (default: h's dtype).  ``eps`` None is
    float32's machine epsilon 2^-23 whatever the dtypes, what
    ``torch.nn.RMSNorm`` adds in float32 and in bfloat16; with 0 a row of zeros
    is NaN.  Differentiable in x, residual and weight, from y and h; the
    weight's gradient has the same bits on every run."""
    f = L.torch_side().add_rms_norm
    if _ops._TIMER is None:
        return f(x, residual, weight, eps, out_dtype)
    with _ops._span("nsa_norm_fwd"):
        return f(x, residual, weight, eps, out_dtype)


def add_rms_norm_q8(x, residual, weight, eps=None):
    """``add_rms_norm`` with the rows in 8 bits, for products in 8 bits:
    ``(q, scale, h)`` with ``q [..., D]`` float8_e4m3fn and ``scale [...]``
    float32, ``y ~ q * scale[..., None]``.

    A row's scale is its largest ``|y|`` (2^-100 at least) over 448; values are
    rounded once, to nearest even.  A row that holds NaN or an infinity has a
    NaN or infinite scale.  For inference: inputs that need a gradient are
    refused."""
    f = L.torch_side().add_rms_norm_q8
    if _ops._TIMER is None:
        return f(x, residual, weight, eps)
    with _ops._span("nsa_norm_fwd"):
        return f(x, residual, weight, eps)


def add_layer_norm(x, residual, weight, bias=None, eps=1e-5, out_dtype=None):
    """``h = x + residual`` and ``y = (h - mean(h)) / sqrt(var(h) + eps) * weight +
    bias`` over the last dimension -> ``(y, h)``; ``var`` is the mean square about
    the mean, as in ``torch.nn.LayerNorm``.

    Shapes, dtypes, rounding and derivatives as in ``add_rms_norm``; ``bias [D]``
    (or None) in the weight's dtype.  The gradients of weight and bias have the
    same bits on every run.  ``eps`` 0 makes a row of equal elements NaN."""
    f = L.torch_side().add_layer_norm
    if _ops._TIMER is None:
        return f(x, residual, weight, bias, eps, out_dtype)
    with _ops._span("nsa_lnorm_fwd"):
        return f(x, residual, weight, bias, eps, out_dtype)


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------

def embed(tokens, weight, scale=1.0, pos_weight=None, positions=None, out_dtype=None):
    """``scale * weight[tokens] + pos_weight[positions]`` -> ``[..., D]`` in
    ``out_dtype`` (default: the weight's), formed in float32 and rounded once.

    ``tokens [..., T]`` and ``positions`` (the same shape) are integers; without
    ``positions`` the token at index t of the last dimension takes row t of
    ``pos_weight [P, D]``, and without ``pos_weight`` there is no position.  A
    token outside ``0 .. V-1`` (padding) adds nothing and has no gradient, nor has
    a position outside ``0 .. P-1``.  Differentiable in both tables: dense
    gradients, summed in float32, with the same bits on every run."""
    f = L.torch_side().embed
    if _ops._TIMER is None:
        return f(tokens, weight, scale, pos_weight, positions, out_dtype)
    with _ops._span("nsa_embed_fwd"):
        return f(tokens, weight, scale, pos_weight, positions, out_dtype)


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
    assert isinstance(top, int), "token_logprobs: top must be 0 .. min(64, V)"
    f = L.torch_side().token_logprobs
    if _ops._TIMER is None:
        return TokenLogprobs(*f(logits, targets, top))
    with _ops._span("nsa_logprob_fwd"):
        return TokenLogprobs(*f(logits, targets, top))


class LinearLogprobs(NamedTuple):
    """Per row: ``logp`` (None without targets) and ``lse``."""

    logp: Optional[torch.Tensor]
    lse: torch.Tensor


def linear_logprobs(x, weight, targets=None):
    """Log probabilities under ``softmax(x @ weight.T)`` without forming the logits:
    ``x [..., D]``, ``weight [V, D]`` -> ``LinearLogprobs`` of float32 ``[...]``.

    ``lse`` is the logits' log-sum-exp and ``logp`` (with integer ``targets [...]``)
    the target's log probability; a target outside ``0 .. V-1`` (``-100`` included)
    leaves 0 and no gradient.  Differentiable in x and weight, from both outputs;
    the backward forms the logits a second time, in pieces of 1 GB at most (or 256
    of the vocabulary), and has the same bits on every run.

    float32 rows are computed in float32's precision.  bfloat16 rows are products of
    bfloat16 with float32 sums, and the logits' gradient is rounded once to bfloat16
    on its way into the products with x and weight, but for the targets' own elements,
    which keep float32's digits in both; float32 weights beside bfloat16 rows are
    rounded to bfloat16 first (as under autocast) and have a float32 gradient.  At most
    2^22 rows.

    Every finite logit counts, whatever its size.  A row with NaN or plus infinity among
    its logits, or with minus infinity alone, is NaN, and so is its gradient where it has
    one (an ignored row's is 0; ``weight``'s sums that 0 times the row of x).  The backward's
    probabilities are formed from ``lse`` as float32 holds it: within ``|lse| 2^-23`` of
    their size."""
    f = L.torch_side().linear_logprobs
    if _ops._TIMER is None:
        return LinearLogprobs(*f(x, weight, targets))
    with _ops._span("nsa_head_fwd"):
        return LinearLogprobs(*f(x, weight, targets))
