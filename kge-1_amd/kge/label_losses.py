"""Losses on the log-probability of ONE label per score row: what tunes a trained model on sampled
answers (a policy) or on preferences between answers.  The kernels are csrc/label_loss.hip; there is no
counterpart in the reference.

``scores`` is a [n, m] block in fp32, bf16 or fp16 with unit column stride and any row stride (an
all-entities block of ``KgeModel.score_sp``, a padded buffer, a slice); ``labels`` holds one column
per row, or -1 for a row that carries nothing (padding of a batch): it is not read and gets a zero
gradient.  Scores of -inf (masked candidates) have probability 0.

* ``label_logprobs``        -- log softmax(scores / temperature)[label] per row, differentiable
* ``policy_loss``           -- clipped policy loss with a KL term, differentiable
* ``preference_loss``       -- paired log ratios of label sequences, differentiable
* ``policy_loss_grad``, ``preference_loss_grad`` -- loss AND gradient in one call, for callers that
  feed the gradient on themselves (``scores.backward(grad)``); ``out=scores`` writes it in place

The differentiable forms keep the scores and two numbers per row; their backward pass reads the
scores again.  Gradients flow into ``scores`` only.
"""
from __future__ import annotations

import contextlib
import math
from typing import Optional, Tuple, Union

import torch

from . import _lib as L

_cur_device = getattr(torch._C, "_cuda_getDevice", None)


def _capturing() -> bool:
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


def is_on_current_device(t: torch.Tensor) -> bool:
    return _cur_device is not None and _cur_device() == t.get_device()


def on_device_of(t: torch.Tensor):
    """A context in which t's device is the current one (launches go to ITS current stream)."""
    return contextlib.nullcontext() if is_on_current_device(t) else torch.cuda.device(t.get_device())


def _score_rows(scores: torch.Tensor) -> torch.Tensor:
    """The score block with unit column stride and rows that do not overlap."""
    if scores.dtype not in L.DTYPES:
        raise ValueError(f"scores: expected float32, bfloat16 or float16, got {scores.dtype}")
    shape = scores.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"scores: expected [n, m] with m >= 1, got {list(shape)}")
    n, m = shape
    if (m > 1 and scores.stride(1) != 1) or (n > 1 and scores.stride(0) < m):
        scores = scores.contiguous()
    return scores


def _ld(x: torch.Tensor) -> int:
    n, m = x.shape
    return x.stride(0) if n > 1 else m


def _labels(labels: torch.Tensor, scores: torch.Tensor) -> torch.Tensor:
    n, m = scores.shape
    if labels.dtype is torch.int64 and labels.shape == (n,) and labels.is_contiguous() and not L.CHECK_INDEX:
        _same_device(labels, scores, "labels")
        return labels
    if labels.dim() != 1 or labels.numel() != n:
        raise ValueError(f"labels: expected [{n}], got {list(labels.shape)}")
    if labels.is_floating_point() or labels.dtype == torch.bool:
        raise ValueError(f"labels: expected integers, got {labels.dtype}")
    _same_device(labels, scores, "labels")
    labels = L.idx64(labels)
    if L.CHECK_INDEX and n > 0 and not _capturing():
        lo, hi = int(labels.min()), int(labels.max())
        if lo < -1 or hi >= m:
            raise IndexError(f"label: index out of range [{lo}, {hi}] for {m} columns (-1: no label)")
    return labels


def _same_device(t: torch.Tensor, scores: torch.Tensor, what: str):
    if t.get_device() != scores.get_device():  # (-1: CPU)
        raise ValueError(f"{what}: on {t.device}, the scores are on {scores.device}")


def _vector(t: Optional[torch.Tensor], n: int, scores: torch.Tensor, what: str) -> Optional[torch.Tensor]:
    """A constant of n numbers as contiguous fp32 on the scores' device."""
    if t is None:
        return None
    if (t.dtype is torch.float32 and t.shape == (n,) and t.is_contiguous() and not t.requires_grad
            and t.get_device() == scores.get_device()):
        return t
    if t.dim() != 1 or t.numel() != n:
        raise ValueError(f"{what}: expected [{n}], got {list(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: no gradient flows into it, pass it detached")
    if not t.is_floating_point():
        raise ValueError(f"{what}: expected floating point numbers, got {t.dtype}")
    _same_device(t, scores, what)
    return t.detach().to(torch.float32).contiguous()


def _temperature(temperature: float) -> float:
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:  # log2(e) / temperature is a 32-bit factor, neither 0 nor infinite
        raise ValueError(f"temperature={temperature}: expected a number in [1e-30, 1e30]")
    return temperature


def _finite(value: float, what: str, low: float = -math.inf, high: float = math.inf) -> float:
    value = float(value)
    if not (math.isfinite(value) and low <= value <= high):
        raise ValueError(f"{what}={value}: expected a number in [{low}, {high}]")
    return value


def _workspace(scores: torch.Tensor, pairs: int = 0):
    size = L.lib().kge_label_ws_size(scores.shape[0], scores.shape[1], L.DTYPES[scores.dtype], pairs)
    return torch.empty(size, device=scores.device, dtype=torch.uint8), size


def _grad_ld(ld: int, m: int, scores: torch.Tensor) -> int:
    if ld <= m + 64:
        return ld
    per = 16 // scores.element_size()
    return (m + per - 1) // per * per


def _grad_buffer(scores: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    """Where the gradient goes: ``out``, or new rows with the scores' stride (the kernels store 16
    bytes at a time where a row and its gradient are aligned alike), padded if that is far wider."""
    n, m = scores.shape
    if out is None:
        return scores.new_empty_strided((n, m), (_grad_ld(_ld(scores), m, scores), 1))
    if out.shape != scores.shape or out.dtype != scores.dtype or out.device != scores.device:
        raise ValueError("out: expected the scores' shape, type and device")
    if (m > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < m):
        raise ValueError("out: expected unit column stride and rows that do not overlap")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out: part of an autograd graph, pass a detached tensor")
    if (n > 0 and out.untyped_storage().data_ptr() == scores.untyped_storage().data_ptr()
            and not (out.data_ptr() == scores.data_ptr() and _ld(out) == _ld(scores))):
        es, a, b = out.element_size(), out.data_ptr(), scores.data_ptr()
        if a < b + ((n - 1) * _ld(scores) + m) * es and b < a + ((n - 1) * _ld(out) + m) * es:
            raise ValueError("out: overlaps the scores without being the same rows")
    if not out.is_inference():  # a graph that has saved the scores sees that they are gone
        torch.autograd.graph.increment_version(out)
    return out


def _launch_logprobs(scores, labels, temperature, want_stats):
    n, m = scores.shape
    logp = torch.empty(n, device=scores.device, dtype=torch.float32)
    stats = torch.empty(n, 2, device=scores.device, dtype=torch.float32) if want_stats else None
    ws, size = _workspace(scores)
    L._check(L.lib().kge_label_logprobs(L.ptr(scores), L.DTYPES[scores.dtype], _ld(scores), n, m, L.ptr(labels),
                                        temperature, L.ptr(logp), L.ptr(stats), L.ptr(ws), size, L.stream()),
             "kge_label_logprobs")
    return logp, stats


def _launch_grad(scores, labels, temperature, stats, coef, gscale):
    """(lean: it runs on autograd's device thread, where Python is slow and every launch-bound step waits for it)"""
    if not is_on_current_device(scores):
        with torch.cuda.device(scores.get_device()):
            return _launch_grad(scores, labels, temperature, stats, coef, gscale)
    n, m = scores.shape
    ld = scores.stride(0) if n > 1 else m
    ldg = _grad_ld(ld, m, scores)
    grad = scores.new_empty_strided((n, m), (ldg, 1))
    status = L.lib().kge_label_grad(scores.data_ptr(), L.DTYPES[scores.dtype], ld, n, m, labels.data_ptr(), temperature,
                                    stats.data_ptr(), coef.data_ptr(), None if gscale is None else gscale.data_ptr(),
                                    grad.data_ptr(), ldg, L.stream())
    if status:
        L._check(status, "kge_label_grad")
    return grad


def first_order(gradient):
    """The ``backward`` of a Function whose ``gradient(ctx, *grads)`` is no graph itself: once_differentiable, whose
    wrapping only a pass that builds a graph (create_graph) pays for."""
    once = torch.autograd.function.once_differentiable(gradient)

    def backward(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else gradient(ctx, *grads)

    return staticmethod(backward)


class _LabelLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, labels, temperature):
        logp, stats = _launch_logprobs(scores, labels, temperature, True)
        ctx.temperature = temperature
        ctx.save_for_backward(scores, labels, stats)
        return logp

    @first_order
    def backward(ctx, g):
        scores, labels, stats = ctx.saved_tensors
        return _launch_grad(scores, labels, ctx.temperature, stats, g.contiguous(), None), None, None


def label_logprobs(scores: torch.Tensor, labels: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """[n] fp32: log softmax(scores[i] / temperature)[labels[i]], 0 where the label is -1.  What
    ``old_logp`` and ``ref_logp`` of the losses below are made of (under ``torch.no_grad()``)."""
    temperature = _temperature(temperature)
    scores = _score_rows(scores)
    labels = _labels(labels, scores)
    L.require_device(scores)
    with on_device_of(scores):
        if scores.requires_grad and torch.is_grad_enabled():
            return _LabelLogprobs.apply(scores, labels, temperature)
        return _launch_logprobs(scores, labels, temperature, False)[0]


class _Policy:
    """The checked arguments of a policy loss."""

    def __init__(self, scores, labels, advantages, old_logp, ref_logp, clip, kl, temperature, weights, scale):
        self.temperature = _temperature(temperature)
        low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
        self.low, self.high = _finite(low, "clip", 0.0), _finite(high, "clip", 0.0)
        self.kl, self.scale = _finite(kl, "kl", 0.0), _finite(scale, "scale")
        if self.kl > 0.0 and ref_logp is None:
            raise ValueError("kl > 0 needs ref_logp")
        self.scores = _score_rows(scores)
        n = self.scores.shape[0]
        self.labels = _labels(labels, self.scores)
        self.advantages = _vector(advantages, n, self.scores, "advantages")
        self.old = _vector(old_logp, n, self.scores, "old_logp")
        self.ref = _vector(ref_logp, n, self.scores, "ref_logp")
        if self.kl == 0.0:
            self.ref = None  # a term of weight 0: whatever the reference says
        self.weights = _vector(weights, n, self.scores, "weights")

    def launch(self, stats=None, coef=None, grad=None):
        s = self.scores
        n, m = s.shape
        loss = torch.empty((), device=s.device, dtype=torch.float32)
        logp = torch.empty(n, device=s.device, dtype=torch.float32)
        ws, size = _workspace(s)
        L._check(L.lib().kge_policy_loss(
            L.ptr(s), L.DTYPES[s.dtype], _ld(s), n, m, L.ptr(self.labels), L.ptr(self.advantages), L.ptr(self.old),
            L.ptr(self.ref), L.ptr(self.weights), self.low, self.high, self.kl, self.temperature, self.scale,
            L.ptr(loss), L.ptr(logp), L.ptr(stats), L.ptr(coef), L.ptr(grad), _ld(grad) if grad is not None else 0,
            L.ptr(ws), size, L.stream()), "kge_policy_loss")
        return loss, logp


class _LabelLoss(torch.autograd.Function):
    """A loss of the rows' label log-probabilities; args.launch leaves each row's coefficient."""

    @staticmethod
    def forward(ctx, scores, args):
        n = scores.shape[0]
        stats = torch.empty(n, 2, device=scores.device, dtype=torch.float32)
        coef = torch.empty(n, device=scores.device, dtype=torch.float32)
        loss, seen = args.launch(stats, coef)
        ctx.temperature = args.temperature
        ctx.save_for_backward(scores, args.labels, stats, coef)
        ctx.mark_non_differentiable(seen)
        ctx.set_materialize_grads(False)
        return loss, seen

    @first_order
    def backward(ctx, g, _g_seen):
        if g is None:
            return None, None
        scores, labels, stats, coef = ctx.saved_tensors
        return _launch_grad(scores, labels, ctx.temperature, stats, coef, g.float()), None


def policy_loss(scores: torch.Tensor, labels: torch.Tensor, advantages: torch.Tensor, old_logp: torch.Tensor,
                ref_logp: Optional[torch.Tensor] = None, *, clip: Union[float, Tuple[float, float]] = 0.2,
                kl: float = 0.0, temperature: float = 1.0, weights: Optional[torch.Tensor] = None,
                scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, logp): with l = log softmax(scores[i] / temperature)[labels[i]], r = exp(l - old_logp[i]),
    d = ref_logp[i] - l and A = advantages[i], the 0-dim
        loss = scale * sum_i weights[i] * (-min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(d) - d - 1))
    (clip = (low, high) or one number for both) and the detached l of every row.  A row beyond its
    border of the clip range keeps only the KL term's gradient; on the border the gradient flows."""
    args = _Policy(scores, labels, advantages, old_logp, ref_logp, clip, kl, temperature, weights, scale)
    L.require_device(args.scores)
    with on_device_of(args.scores):
        if args.scores.requires_grad and torch.is_grad_enabled():
            return _LabelLoss.apply(args.scores, args)
        return args.launch()


def policy_loss_grad(scores: torch.Tensor, labels: torch.Tensor, advantages: torch.Tensor, old_logp: torch.Tensor,
                     ref_logp: Optional[torch.Tensor] = None, *, clip: Union[float, Tuple[float, float]] = 0.2,
                     kl: float = 0.0, temperature: float = 1.0, weights: Optional[torch.Tensor] = None,
                     scale: float = 1.0, out: Optional[torch.Tensor] = None):
    """(loss, logp, grad): ``policy_loss`` and its gradient with respect to the scores in one call,
    outside autograd.  out: where the gradient goes (the scores themselves: in place)."""
    args = _Policy(scores.detach(), labels, advantages, old_logp, ref_logp, clip, kl, temperature, weights, scale)
    L.require_device(args.scores)
    with on_device_of(args.scores):
        grad = _grad_buffer(args.scores, out)
        return (*args.launch(grad=grad), grad)


class _Preference:
    """The checked arguments of a preference loss."""

    def __init__(self, scores, labels, seq_ptr, ref_logp, beta, smoothing, average, temperature, scale):
        self.temperature = _temperature(temperature)
        self.beta, self.scale = _finite(beta, "beta", 0.0), _finite(scale, "scale")
        self.smoothing, self.average = _finite(smoothing, "smoothing", 0.0, 1.0), bool(average)
        self.scores = _score_rows(scores)
        self.labels = _labels(labels, self.scores)
        if seq_ptr.dim() != 1 or seq_ptr.numel() % 2 != 1 or seq_ptr.is_floating_point() or seq_ptr.dtype == torch.bool:
            raise ValueError("seq_ptr: expected 2 pairs + 1 ascending row numbers (two sequences per pair), got "
                             f"{list(seq_ptr.shape)} {seq_ptr.dtype}")
        _same_device(seq_ptr, self.scores, "seq_ptr")
        self.ptr = L.idx64(seq_ptr)
        self.pairs = self.ptr.numel() // 2
        if L.CHECK_INDEX and not _capturing():
            v = self.ptr.tolist()
            if v[0] < 0 or v[-1] > self.scores.shape[0] or any(a > b for a, b in zip(v, v[1:])):
                raise IndexError(f"seq_ptr: expected ascending rows in [0, {self.scores.shape[0]}]")
        self.ref = _vector(ref_logp, 2 * self.pairs, self.scores, "ref_logp")

    def launch(self, stats=None, coef=None, grad=None):
        s = self.scores
        n, m = s.shape
        loss = torch.empty((), device=s.device, dtype=torch.float32)
        seq_logp = torch.empty(2 * self.pairs, device=s.device, dtype=torch.float32)
        logp = torch.empty(n, device=s.device, dtype=torch.float32)
        ws, size = _workspace(s, self.pairs)
        L._check(L.lib().kge_preference_loss(
            L.ptr(s), L.DTYPES[s.dtype], _ld(s), n, m, L.ptr(self.labels), L.ptr(self.ptr), self.pairs, L.ptr(self.ref),
            self.beta, self.smoothing, int(self.average), self.temperature, self.scale, L.ptr(loss), L.ptr(seq_logp),
            L.ptr(logp), L.ptr(stats), L.ptr(coef), L.ptr(grad), _ld(grad) if grad is not None else 0, L.ptr(ws), size,
            L.stream()), "kge_preference_loss")
        return loss, seq_logp


def preference_loss(scores: torch.Tensor, labels: torch.Tensor, seq_ptr: torch.Tensor,
                    ref_logp: Optional[torch.Tensor] = None, *, beta: float = 0.1, smoothing: float = 0.0,
                    average: bool = False, temperature: float = 1.0,
                    scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, seq_logp).  Sequence q is the rows seq_ptr[q] .. seq_ptr[q + 1] - 1 (an answer of one or
    more labels); pair k prefers sequence 2 k to sequence 2 k + 1.  seq_logp[q] is the sum (average:
    the mean) of the log-probabilities of the sequence's labels, detached;
        z_k  = beta ((seq_logp[2k] - ref_logp[2k]) - (seq_logp[2k+1] - ref_logp[2k+1]))
        loss = -scale * sum_k (1 - smoothing) log sigma(z_k) + smoothing log sigma(-z_k)
    ref_logp: [2 pairs], the same sums under the reference model (None: 0).  Rows of no sequence get
    a zero gradient."""
    args = _Preference(scores, labels, seq_ptr, ref_logp, beta, smoothing, average, temperature, scale)
    L.require_device(args.scores)
    with on_device_of(args.scores):
        if args.scores.requires_grad and torch.is_grad_enabled():
            return _LabelLoss.apply(args.scores, args)
        return args.launch()


def preference_loss_grad(scores: torch.Tensor, labels: torch.Tensor, seq_ptr: torch.Tensor,
                         ref_logp: Optional[torch.Tensor] = None, *, beta: float = 0.1, smoothing: float = 0.0,
                         average: bool = False, temperature: float = 1.0, scale: float = 1.0,
                         out: Optional[torch.Tensor] = None):
    """(loss, seq_logp, grad): ``preference_loss`` and its gradient with respect to the scores in one
    call, outside autograd.  out: where the gradient goes (the scores themselves: in place)."""
    args = _Preference(scores.detach(), labels, seq_ptr, ref_logp, beta, smoothing, average, temperature, scale)
    L.require_device(args.scores)
    with on_device_of(args.scores):
        grad = _grad_buffer(args.scores, out)
        return (*args.launch(grad=grad), grad)
