"""Row operators on logits: what a model's user does with them besides sampling.

* ``token_logprobs``: the log-probability of one token per row, and the row's
  entropy (the log-probabilities of sampled tokens, and the loss of training
  on them);
* ``top_logits``: the k largest logits of each row with the log-sum of the
  rest (the top log-probabilities a server reports, and what a teacher leaves
  for distillation);
* ``policy_loss``: the clipped policy-ratio loss with a KL and an entropy term;
* ``distill_loss``: KL(teacher || student) against a ``top_logits`` record.

They take the logits, packed masks and statuses of ``exactsample_b200.verify``
and share its rules: every tensor is on the logits' device, bad values inside
device tensors do not raise but show up as that row's status, and a row's
results are the same bits in any batch. Temperatures are one number, or one
float64 per row, where ``verify`` has one per request, and are positive: there
is no greedy 0, whose rows would be INVALID_INPUT. ``include/exactsample_b200.h`` states
each operator's formulas and what its statuses mean.

A call launches one kernel on the current stream. It allocates its per-row
outputs, reads nothing from the host and needs no workspace, so calls may
overlap on any streams and be captured in CUDA graphs. A row is read once: a
loss that is given ``grad`` writes its gradient from the same read.

Gradients come in two ways. With ``grad=`` a tensor of the logits' type and
shape (the logits themselves too, which it then replaces), the call fills it
with the gradient of the sum of the row losses: nothing is recorded for
autograd. Without it, on logits that require a gradient, the result is
differentiable by the logits, once and in reverse mode (forward-mode
derivatives are refused), and the backward pass reads them a second time.
To capture a whole training step in a CUDA graph, ``grad=`` is the way that
does not depend on what autograd's accumulation nodes were made on. The calls
can be traced (torch.compile, tensors without memory) once the library is
loaded, which ``exactsample_b200.cuda.load_library`` or any call of one does.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from .cuda import load_library


@dataclass(slots=True)
class TokenLogprobs:
    logprobs: Any  # float32 [rows]
    entropy: Any   # float32 [rows]
    status: Any    # int32 [rows]


@dataclass(slots=True)
class TopLogits:
    values: Any         # float32 [rows, k]: logits, in descending order
    ids: Any            # int64 [rows, k], -1 past the row's allowed tokens
    rest: Any           # float32 [rows]: log of the other tokens' sum of exp(logit / temperature)
    status: Any = None  # int32 [rows]


@dataclass(slots=True)
class PolicyLoss:
    loss: Any      # float32 [rows]
    logprobs: Any  # float32 [rows]
    kl: Any        # float32 [rows]
    entropy: Any   # float32 [rows]
    status: Any    # int32 [rows]


@dataclass(slots=True)
class DistillLoss:
    loss: Any    # float32 [rows]
    status: Any  # int32 [rows]


class _Operators:
    """The torch ops, loaded when one is first asked for."""

    def __getattr__(self, name):
        load_library()
        op = getattr(torch.ops.exactsample, name).default
        setattr(self, name, op)
        return op


_ops = _Operators()


def _temperature(value):
    """(tensor or None, the number that holds when there is none)."""
    if isinstance(value, torch.Tensor):
        return value, 1.0
    return None, float(value)


def _tracked(logits, grad, *others) -> bool:
    """Whether the call is recorded for autograd; refuses what has no gradient."""
    if not torch.is_grad_enabled():
        return False
    for t in others:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            raise ValueError("row operators are differentiable by the logits only; detach the other inputs")
    if not logits.requires_grad:
        return False
    if grad is not None:
        raise ValueError("grad= takes the gradient in the call itself: pass detached logits, or leave grad out")
    return True


def token_logprobs(logits, tokens, *, temperature=1.0, mask=None, grad=None, grad_logprobs=None,
                   grad_entropy=None) -> TokenLogprobs:
    """log p[token] and the entropy of each row of ``logits`` [rows, vocab] (float16, bfloat16 or float32).

    ``tokens`` is int64 [rows]; a negative token marks a row without one,
    whose results are 0. ``temperature`` divides the logits: a number, or
    float64 [rows]. ``mask`` is the packed int32 mask of ``verify``. Logprobs
    and entropy are differentiable by the logits; ``grad=`` instead receives
    the gradient of ``sum(grad_logprobs * logprobs + grad_entropy * entropy)``
    (float32 [rows] each; one left out counts as zeros).
    """
    per_row, everywhere = _temperature(temperature)
    if _tracked(logits, grad, per_row, grad_logprobs, grad_entropy):
        if grad_logprobs is not None or grad_entropy is not None:
            raise ValueError("grad_logprobs and grad_entropy need grad")
        return TokenLogprobs(*_ops.token_logprobs_tracked(logits, tokens, per_row, everywhere, mask))
    return TokenLogprobs(*_ops.token_logprobs(logits, tokens, per_row, everywhere, mask, grad, grad_logprobs,
                                                      grad_entropy))


def top_logits(logits, k: int, *, temperature=1.0, mask=None) -> TopLogits:
    """The ``k`` (1 to 256) largest logits of each row, the lowest id first among equal ones, and the rest's log-sum.

    ``values`` are the logits as they are; ``temperature`` is what ``rest`` is
    taken at. Log-probabilities follow as ``values / temperature - total`` with
    ``total = logaddexp(logsumexp(values / temperature), rest)``. Not recorded
    for autograd: it is a teacher's or a server's pass. Rows that a mask, or
    logits of -inf, leave without tokens over a long range of ids take a path
    of milliseconds, as do rows of equal logits in numbers.
    """
    per_row, everywhere = _temperature(temperature)
    return TopLogits(*_ops.top_logits(logits, k, per_row, everywhere, mask))


def policy_loss(logits, tokens, old_logprobs, advantages, *, ref_logprobs=None, weights=None, temperature=1.0,
                mask=None, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                entropy_coef: float = 0.0, grad=None) -> PolicyLoss:
    """The clipped policy-ratio loss of each row's token, times the row's weight.

    ``tokens``, ``temperature`` and ``mask`` are ``token_logprobs``'s: with
    the temperature and masks the tokens were sampled under, the ratio is that
    of the distributions they came from, if those were not truncated by top-k,
    top-p or min-p (probabilities here are over all allowed tokens).
    ``old_logprobs``, ``advantages``,
    ``ref_logprobs`` and ``weights`` are float32 [rows]. The clip range of the
    ratio is [1 - clip_low, 1 + clip_high]. ``loss`` is differentiable by the
    logits; the other outputs are for monitoring.
    """
    per_row, everywhere = _temperature(temperature)
    coefficients = (float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef))
    if _tracked(logits, grad, old_logprobs, advantages, ref_logprobs, weights, per_row):
        return PolicyLoss(*_ops.policy_loss_tracked(logits, tokens, old_logprobs, advantages, ref_logprobs, weights,
                                                    per_row, everywhere, mask, *coefficients))
    return PolicyLoss(*_ops.policy_loss(logits, tokens, old_logprobs, advantages, ref_logprobs, weights,
                                                per_row, everywhere, mask, *coefficients, grad))


def distill_loss(logits, teacher: TopLogits, *, weights=None, temperature=1.0, mask=None, tail: bool = True,
                 grad=None) -> DistillLoss:
    """KL(teacher || student) of each row, times the row's weight.

    ``teacher`` is a ``top_logits`` record of the teacher's rows, made at the
    same ``temperature``. With ``tail`` the teacher's remaining probability is
    held against the student's as one bucket; without it the teacher is
    renormalised over the tokens it kept. Entries with a negative id are
    unused, and a row without used entries is padding, unless the record's
    ``status`` says that the teacher's row failed: then it has that status (its
    loss is 0 and its gradient zeros as well). ``mask`` limits the student. The loss is that of probabilities at ``temperature``: multiply it
    (or ``weights``) by the temperature squared for gradients that keep their
    scale across temperatures.
    """
    per_row, everywhere = _temperature(temperature)
    if tail and teacher.rest is None:
        raise ValueError("tail=True needs the teacher's rest")
    rest = teacher.rest if tail else None
    if _tracked(logits, grad, teacher.values, rest, weights, per_row):
        return DistillLoss(*_ops.distill_loss_tracked(logits, teacher.values, teacher.ids, rest, weights, per_row,
                                                      everywhere, mask, teacher.status))
    return DistillLoss(*_ops.distill_loss(logits, teacher.values, teacher.ids, rest, weights, per_row,
                                          everywhere, mask, grad, teacher.status))
