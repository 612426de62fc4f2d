"""The compositions of rg's primitive ops that the GPT workload and its sampler use: softmax and
log-softmax over the last axis, cross-entropy, the tanh GELU, and the top-k / nucleus logit
filters. Each is written as the same sequence of primitive ops as rg's python/rg/nn.py
(softmax nn.py:40-42, log-softmax and logsumexp nn.py:29-37, cross-entropy nn.py:78-84, GELU
nn.py:25-27, filters nn.py:60-72), so the device receives the plan rg would build; the row
statistics go through `stop_gradient`, as in rg, so autodiff emits rg's backward chains.

Below them, the objectives that rg has no counterpart for: the log-probability of given tokens, the
clipped policy loss with a KL term, the preference loss over pairs of sequences and the distillation
from a teacher's top logits. Each is one operation of the engine. They take logits (..., V), int32 labels
of the leading shape (clamped to [0, V), as indices are everywhere) and operands of the leading shape in
the logits' dtype. Gradients flow to the logits only; the other operands are data. Only the first result
of a loss is differentiable, the others are for reporting (differentiating them is an error). Positions
with weight 0 count nothing, whatever they hold. A loss computes its gradient in the same pass over the
logits, so it is an output of the forward step; a loss that is only evaluated does not compute it. A loss with
a factor multiplies that gradient afterwards, one more pass over it: the weights take a factor for nothing.
"""
import math

from .tracing import argsort, cumsum, exp, objective, stop_gradient, take_along_axis, tanh, top_k, where

_GELU_C = math.sqrt(2.0 / math.pi)


def gelu(x):
    return 0.5 * x * (1.0 + tanh(_GELU_C * (x + 0.044715 * x * x * x)))


def _row_max(x, axis):
    return stop_gradient(x.max(axis=axis, keepdims=True))


def softmax(x, axis=-1):
    e = exp(x - _row_max(x, axis))
    return e / e.sum(axis=axis, keepdims=True)


def logsumexp(x, axis=-1, keepdims=False):
    m = _row_max(x, axis)
    out = exp(x - m).sum(axis=axis, keepdims=True).log() + m
    return out if keepdims else out.squeeze(axis)


def log_softmax(x, axis=-1):
    return x - logsumexp(x, axis=axis, keepdims=True)


def cross_entropy(logits, labels, axis=-1):
    """Mean negative log-likelihood of int32 class labels."""
    picked = take_along_axis(log_softmax(logits, axis), labels.reshape(tuple(labels.shape) + (1,)))
    return -picked.mean()


def top_k_logits(logits, k):
    """Logits outside the k largest of the last axis drop to -1e9."""
    values, _ = top_k(logits, k)
    return where(logits >= values[..., -1:], logits, -1e9)


def top_p_logits(logits, p):
    """Nucleus filter: a token stays while the probability mass ranked above it is below p."""
    order = argsort(logits, descending=True)
    probs = softmax(take_along_axis(logits, order))
    kept = (cumsum(probs) - probs) < p
    return where(take_along_axis(kept, argsort(order.cast(logits.dtype))), logits, -1e9)


def token_log_prob(logits, labels):
    """log_softmax(logits) at `labels`, without the full log_softmax: -token_log_prob(logits, labels).mean()
    is the cross-entropy. The gradient may weight each position differently."""
    return objective("token_log_prob", logits, labels)[0]


def policy_loss(logits, labels, old_logp, advantages, weights, ref_logp=None, clip_low=0.2, clip_high=0.2, kl=0.0):
    """`(loss, terms, logp)` of the clipped policy loss: with r = exp(logp - old_logp) and d = ref_logp - logp,
    terms = weights * (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl (exp(d) - d - 1)) and loss their
    sum. The weights carry the mask and the averaging; `ref_logp` goes with a kl != 0."""
    if (kl != 0) != (ref_logp is not None):
        raise ValueError("ref_logp goes with a kl coefficient that is not 0")
    data = (labels, old_logp, advantages, weights) + (() if ref_logp is None else (ref_logp,))
    return objective("policy_loss", logits, *data, clip_low=float(clip_low), clip_high=float(clip_high), kl=float(kl))[:3]


def preference_loss(logits, labels, weights, ref_logp, beta=0.1, smoothing=0.0):
    """`(loss, margins, logp)` of the paired preference loss over 2 n sequences, logits (2 n, T, V), chosen
    ones first: logp = S = (weights * token log-probability).sum over T (2 n), margins = h =
    beta ((S - ref_logp) of the chosen - of the rejected one) (n), loss the mean over pairs of
    -(1 - smoothing) log sigma(h) - smoothing log sigma(-h). `ref_logp` (2 n) is the reference's S."""
    return objective("preference_loss", logits, labels, weights, ref_logp, beta=float(beta), smoothing=float(smoothing))[:3]


def distillation_loss(logits, index, teacher, weights, temperature=1.0):
    """`(loss, terms)` of the distillation from a teacher's k top logits, `teacher` (..., k) at vocabulary
    positions `index` (..., k): with q = softmax(teacher / T) and p = softmax(logits / T), terms =
    weights * T^2 * sum q (log q - log p) and loss their sum. Teacher entries of -inf are absent, an index
    given twice counts twice, k is at most 1024. T is between 2^-60 and 2^60."""
    return objective("distillation_loss", logits, index, teacher, weights, temperature=float(temperature))[:2]
