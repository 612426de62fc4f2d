"""Objectives over logits that are already on the GPU, as torch tensors: the calls of include/rgc.h
(rgc_token_log_prob .. rgc_distillation_loss) with outputs allocated by torch, on torch's current stream of
the logits' device. Compiled programs have the same objectives in `frontend.nn`.

Every function takes logits of shape (..., V), float32 or float64, whose last axis is contiguous and whose
leading axes fold into at most two strides (a model's output, or a slice of its positions such as
`logits[:, :-1]`). Labels and indices are int32 of the leading shape and are clamped to [0, V); all other
operands have the logits' dtype and the leading shape. Positions with weight 0 are not read: they count
nothing, whatever they hold (padding may be NaN, with labels of -100), and their gradient is 0.

`grad=False` computes the loss alone. `out` receives the gradient: a tensor of the logits' shape and dtype,
which may be the logits themselves (they are then overwritten). A refused argument raises ValueError or
TypeError before anything is launched. Nothing synchronises, so the calls can be captured into CUDA graphs.
"""
from typing import NamedTuple, Optional

import torch

from . import load_native

_DTYPES = {torch.float32: 0, torch.float64: 1}
_rg = None


def _native():
    global _rg
    if _rg is None:
        _rg = load_native()
    return _rg


# The current stream's handle without building a Stream object, where torch has the call.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _rows(x, out=None):
    """The leading axes of `x` as (outer, inner, outer stride, inner stride), and the same strides of `out`:
    axes that chain in both are one."""
    if x.dim() < 1:
        raise ValueError("logits need a last axis")
    shape = x.shape
    strides = [x.stride()] if out is None else [x.stride(), out.stride()]
    for s in strides:
        if s[-1] != 1 and shape[-1] != 1:
            raise ValueError("the last axis of the logits and of out must be contiguous")
    groups = []  # (extent, stride of each), slowest first
    for axis, n in enumerate(shape[:-1]):
        if n == 1:
            continue
        at = [s[axis] for s in strides]
        if groups and all(before == n * s for before, s in zip(groups[-1][1], at)):
            groups[-1] = (groups[-1][0] * n, at)
        else:
            groups.append((n, at))
    if len(groups) > 2:
        raise ValueError("the leading axes of the logits (and of out) have more than two independent strides; make them contiguous")
    none = (1, [0] * len(strides))
    (outer, so), (inner, si) = groups + [none] * (2 - len(groups))
    return outer, inner, so, si


class _Call:
    """The logits of a call, where their gradient goes, and the stream it runs on. `sequences`: the leading
    axes are (sequences, positions) as they are."""

    __slots__ = ("logits", "index", "dtype", "lead", "grad", "args", "grad_args", "out")

    def __init__(self, logits, grad=False, out=None, sequences=False):
        if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
            raise TypeError("logits must be a CUDA tensor")
        self.dtype = logits.dtype
        dtype = _DTYPES.get(self.dtype)
        if dtype is None:
            raise TypeError(f"logits must be float32 or float64, not {logits.dtype}")
        shape = logits.shape
        if sequences and len(shape) != 3:
            raise ValueError("logits must be (sequences, positions, vocabulary)")
        self.logits, self.index, self.lead, self.out = logits, logits.get_device(), shape[:-1], out
        if out is not None:
            if not grad:
                raise ValueError("out is given but no gradient is asked for")
            if not isinstance(out, torch.Tensor) or out.get_device() != self.index or out.dtype != self.dtype or out.shape != shape:
                raise ValueError("out must have the logits' shape, dtype and device")
        elif len(shape) and logits.is_contiguous() and shape[-1]:
            # The usual case, in as few steps as there are.
            v = shape[-1]
            outer, inner = (shape[0], shape[1]) if sequences else (logits.numel() // v, 1)
            self.grad = torch.empty_like(logits, memory_format=torch.contiguous_format) if grad else None
            self.args = (logits.data_ptr(), outer, inner, v, inner * v, v, dtype)
            self.grad_args = (self.grad.data_ptr(), inner * v, v) if grad else (0, 0, 0)
            return
        self.grad = out if out is not None else logits.new_empty(shape) if grad else None
        if sequences:
            strides = [logits.stride()] if self.grad is None else [logits.stride(), self.grad.stride()]
            if any(s[2] != 1 for s in strides) and shape[2] != 1:
                raise ValueError("the last axis of the logits and of out must be contiguous")
            outer, inner = shape[:2]
            so, si = [s[0] for s in strides], [s[1] for s in strides]
        else:
            outer, inner, so, si = _rows(logits, self.grad)
        self.args = (logits.data_ptr(), outer, inner, shape[-1], so[0], si[0], dtype)
        self.grad_args = (0, 0, 0) if self.grad is None else (self.grad.data_ptr(), so[1], si[1])

    def per_row(self, t, what, shape=None, dtype=None):
        """A contiguous operand on the logits' device."""
        if not isinstance(t, torch.Tensor) or t.get_device() != self.index:
            raise TypeError(f"{what} must be a tensor on the logits' device")
        if t.dtype != (dtype or self.dtype):
            raise TypeError(f"{what} must be {dtype or self.dtype}, not {t.dtype}")
        if t.shape != (self.lead if shape is None else shape):
            raise ValueError(f"{what} has shape {tuple(t.shape)}, not {tuple(self.lead if shape is None else shape)}")
        return t if t.is_contiguous() else t.contiguous()

    def run(self, call, *args):
        if self.index == torch.cuda.current_device():
            call(self.args, *args, _stream(self.index))
        else:
            with torch.cuda.device(self.index):
                call(self.args, *args, _stream(self.index))
        if self.out is not None:  # autograd refuses what it has saved of the tensor's former contents
            torch.autograd.graph.increment_version(self.out)


def token_log_prob(logits, labels, *, stats=False):
    """log softmax(logits) at `labels`; with `stats=True` also the row statistics (..., 2) = (maximum, sum of
    exp(logits - maximum)) that `token_log_prob_grad` takes."""
    c = _Call(logits)
    labels = c.per_row(labels, "labels", dtype=torch.int32)
    logp = logits.new_empty(c.lead)
    st = logits.new_empty((*c.lead, 2)) if stats else None
    c.run(_native().token_log_prob, labels.data_ptr(), logp.data_ptr(), st.data_ptr() if stats else 0)
    return (logp, st) if stats else logp


def token_log_prob_grad(logits, labels, stats, dlogp, *, out=None):
    """The gradient with respect to `logits` of token_log_prob for the cotangent `dlogp`."""
    c = _Call(logits, True, out)
    labels = c.per_row(labels, "labels", dtype=torch.int32)
    stats = c.per_row(stats, "stats", shape=(*c.lead, 2))
    dlogp = c.per_row(dlogp, "dlogp")
    c.run(_native().token_log_prob_grad, labels.data_ptr(), stats.data_ptr(), dlogp.data_ptr(), c.grad_args)
    return c.grad


class PolicyLoss(NamedTuple):
    loss: torch.Tensor            # scalar: the sum of the terms
    terms: torch.Tensor           # per position, weighted
    logp: torch.Tensor            # log-probabilities of the labels (0 where the weight is 0)
    grad: Optional[torch.Tensor]  # of the loss with respect to the logits


def policy_loss(logits, labels, old_logp, advantages, weights, *, ref_logp=None, clip_low=0.2, clip_high=0.2, kl=0.0, grad=True, out=None):
    """The clipped policy loss: with r = exp(logp - old_logp) and d = ref_logp - logp, the sum over positions
    of weights * (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl (exp(d) - d - 1)). The weights carry the
    mask and the averaging (mask / mask.sum() for a mean over tokens). `ref_logp` goes with a kl != 0."""
    if (kl != 0) != (ref_logp is not None):
        raise ValueError("ref_logp goes with a kl coefficient that is not 0")
    c = _Call(logits, grad, out)
    labels = c.per_row(labels, "labels", dtype=torch.int32)
    old = c.per_row(old_logp, "old_logp")
    adv = c.per_row(advantages, "advantages")
    w = c.per_row(weights, "weights")
    ref = c.per_row(ref_logp, "ref_logp") if ref_logp is not None else None
    loss, terms, logp = logits.new_empty(()), torch.empty_like(w), torch.empty_like(w)
    c.run(_native().policy_loss, labels.data_ptr(), old.data_ptr(), adv.data_ptr(), w.data_ptr(), 0 if ref is None else ref.data_ptr(),
          clip_low, clip_high, kl, loss.data_ptr(), terms.data_ptr(), logp.data_ptr(), c.grad_args)
    return PolicyLoss(loss, terms, logp, c.grad)


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor            # scalar: the mean over pairs
    margins: torch.Tensor         # (n,) beta times the difference of the log ratios
    logp: torch.Tensor            # (2 n,) weighted log-probability of each sequence
    grad: Optional[torch.Tensor]  # of the loss with respect to the logits


def preference_loss(logits, labels, weights, ref_logp, *, beta=0.1, smoothing=0.0, grad=True, out=None):
    """The paired preference loss over 2 n sequences, logits (2 n, T, V), the n chosen ones before the n rejected
    ones: S = sum over positions of weights * logp, h = beta ((S - ref_logp)[chosen] - (S - ref_logp)[rejected]),
    and the mean over pairs of -(1 - smoothing) log sigma(h) - smoothing log sigma(-h). `ref_logp` (2 n,) holds the
    reference's S; weights are the mask of the answers' tokens (divided by their number for a mean per token)."""
    c = _Call(logits, grad, out, sequences=True)
    n, t = c.lead
    if n < 2 or n % 2:
        raise ValueError("logits must hold pairs of sequences: an even number of at least 2")
    labels = c.per_row(labels, "labels", dtype=torch.int32)
    w = c.per_row(weights, "weights")
    ref = c.per_row(ref_logp, "ref_logp", shape=(n,))
    nbytes = _native().preference_workspace(n, t, _DTYPES[c.dtype])
    workspace = logits.new_empty((nbytes,), dtype=torch.uint8)
    loss, margins, logp = logits.new_empty(()), logits.new_empty((n // 2,)), torch.empty_like(ref)
    c.run(_native().preference_loss, labels.data_ptr(), w.data_ptr(), ref.data_ptr(), beta, smoothing, loss.data_ptr(), margins.data_ptr(),
          logp.data_ptr(), c.grad_args, workspace.data_ptr(), nbytes)
    return PreferenceLoss(loss, margins, logp, c.grad)


class DistillationLoss(NamedTuple):
    loss: torch.Tensor            # scalar: the sum of the terms
    terms: torch.Tensor           # per position, weighted
    grad: Optional[torch.Tensor]  # of the loss with respect to the logits


def distillation_loss(logits, index, teacher, weights, *, temperature=1.0, grad=True, out=None):
    """Distillation from a teacher's top logits: `teacher` (..., k) at the vocabulary positions `index` (..., k).
    With q = softmax(teacher / T) and p = softmax(logits / T), the sum over positions of
    weights * T^2 * sum_k q (log q - log p). Entries of -inf are absent (rows may hold fewer than k), an
    index given twice counts twice, and k is at most 1024. T is between 2^-60 and 2^60."""
    c = _Call(logits, grad, out)
    if not isinstance(index, torch.Tensor) or index.dim() < 1:
        raise TypeError("index must be a tensor with a last axis of teacher entries")
    k = index.shape[-1]
    index = c.per_row(index, "index", shape=(*c.lead, k), dtype=torch.int32)
    teacher = c.per_row(teacher, "teacher", shape=(*c.lead, k))
    w = c.per_row(weights, "weights")
    loss, terms = logits.new_empty(()), torch.empty_like(w)
    c.run(_native().distillation_loss, index.data_ptr(), teacher.data_ptr(), w.data_ptr(), k, temperature, loss.data_ptr(), terms.data_ptr(), c.grad_args)
    return DistillationLoss(loss, terms, c.grad)
