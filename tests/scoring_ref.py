"""The row operators' formulas in 64 bits on the CPU, one row at a time, and
how far a kernel with 32-bit arithmetic may be from them.

Gradients are torch's own differentiation of the forward formulas; the CPU
tests hold those against finite differences.
"""
from __future__ import annotations

import math

import torch

from exactsample_b200 import Status

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
SMALLEST = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}


def unpack_mask(words, vocab):
    """bool [rows, vocab] of packed int32 words."""
    bits = torch.arange(vocab)
    return ((words.cpu()[:, bits // 32].to(torch.int64) >> (bits % 32)) & 1).bool()


def pack_mask(allowed):
    """Packed int32 words of bool [rows, vocab]."""
    rows, vocab = allowed.shape
    words = (vocab + 31) // 32
    padded = torch.zeros(rows, words * 32, dtype=torch.int64)
    padded[:, :vocab] = allowed
    sums = (padded.view(rows, words, 32) << torch.arange(32)).sum(2)
    return torch.where(sums >= 2**31, sums - 2**32, sums).to(torch.int32)


def row_status(z, allowed, temperature):
    """ES_INVALID_INPUT / ES_NO_VALID_TOKEN / OK of the logits alone."""
    if torch.isnan(z).any() or (z == math.inf).any() or not (math.isfinite(temperature) and temperature > 0):
        return Status.INVALID_INPUT
    if not (allowed & (z > -math.inf)).any():
        return Status.NO_VALID_TOKEN
    return Status.OK


def logp_of(z, allowed, temperature):
    return torch.log_softmax((z / temperature).masked_fill(~allowed, -math.inf), 0)


def entropy_of(logp):
    live = logp > -math.inf
    return -(logp[live].exp() * logp[live]).sum()


def policy_of(lp, entropy, old, adv, ref, weight, low, high, kl_coef, entropy_coef):
    ratio = (lp - old).exp()
    clipped = ratio.clamp(1 - low, 1 + high)
    value = -(ratio * adv if ratio * adv <= clipped * adv else clipped.detach() * adv)
    kl = torch.zeros((), dtype=torch.float64) if ref is None else (ref - lp).exp() - (ref - lp) - 1
    return weight * (value + kl_coef * kl - entropy_coef * entropy), kl


def distill_of(logp, values, ids, rest, temperature):
    """(loss, whether the student has no mass where the teacher has some)."""
    used = ids >= 0
    t = values[used] / temperature
    q = logp[ids[used]]
    kept = torch.zeros(logp.numel(), dtype=torch.bool)
    kept[ids[used]] = True
    if rest is not None:
        t = torch.cat([t, rest[None]])
        others = logp[~kept & (logp > -math.inf)]
        q = torch.cat([q, (torch.logsumexp(others, 0) if others.numel() else torch.tensor(-math.inf).double())[None]])
    t = torch.log_softmax(t, 0)
    on = t.exp() > 0
    lost = bool((q[on] == -math.inf).any())
    return (t[on].exp() * (t[on] - q[on])).sum(), lost


def top_of(z, allowed, temperature, k):
    """(values, ids, rest) by a stable sort."""
    z = z.masked_fill(~allowed, -math.inf)
    order = torch.sort(z, descending=True, stable=True)
    count = min(k, int((z > -math.inf).sum()))
    values = torch.full((k,), -math.inf, dtype=torch.float64)
    ids = torch.full((k,), -1, dtype=torch.int64)
    values[:count], ids[:count] = order.values[:count], order.indices[:count]
    others = order.values[count:] / temperature
    rest = float(torch.logsumexp(others, 0)) if others.numel() else -math.inf
    return values, ids, rest


class RowBounds:
    """How far 32-bit results of one row may be from the exact ones.

    With d = x - max(x) per token, in natural units:
    * an exponential exp(d) is off by 2^-22 (the hardware's exp2 to 2 units in
      the last place) and by its argument: the difference, the product and
      the scale are each rounded once, 3 * 2^-24 |d| together;
    * a partial sum adds at most `terms` exponentials, then about 24 joins
      (two halves, 5 + 3 shuffles each a product and a sum, 16 ranks):
      2^-24 each.
    """

    def __init__(self, logp, vocab):
        live = logp > -math.inf
        p, d = logp[live].exp(), (logp[live] - logp[live].max())
        self.m1 = float((p * d.abs()).sum())
        self.m2 = float((p * d * d).sum())
        # The reference that exponents are taken against is one of the row's
        # tokens, at most 2^60 below the maximum.
        self.gap = min(float(d.abs().max()), 60 * math.log(2.0))
        terms = vocab / 256 / 2 + 8
        self.sum = 2.0**-22 + (terms + 24) * 2.0**-24 + 3 * 2.0**-24 * self.m1

    def logprob(self, lp):
        return self.sum + 2.0**-24 * abs(float(lp))

    def entropy(self, h):
        # log(sum) and the ratio of sums: each term of the second carries |d|.
        # Against a reference `gap` away, a term's product, the ratio and the
        # difference are rounded once each in numbers larger by gap.
        return self.sum * (2 + 2 * self.m1) + 3 * 2.0**-24 * (self.m2 + self.gap) + 2.0**-23 * abs(float(h))

    def probability(self, logp):
        """Relative, of each token's probability times the row's coefficient.

        The coefficient's way in 32 bits: 1 / temperature, its product with
        the slope, the entropy's part (a product, a difference), 1 / sum, the
        product with it, the correction of the exponent's reference (three),
        and the last product: ten roundings."""
        d = (logp - logp.max()).clamp(min=-200).abs()
        return 2.0**-22 + 3 * 2.0**-24 * d + self.sum + 10 * 2.0**-24


def token_grad_bound(bounds, logp, grad, token, on_lp, on_h, h, temperature, dtype):
    """Per token, for the gradient of on_lp * lp + on_h * H at `token`."""
    p = logp.exp()
    # The kernel's sum has h, log(sum) and d in it, and log(sum) = d - log p.
    d = (logp - logp.max()).clamp(min=-1e4).abs()
    size = abs(on_lp) + abs(on_h) * (logp.clamp(min=-1e4).abs() + abs(h) + 2 * d)
    absolute = p * (size * bounds.probability(logp) + abs(on_h) * bounds.entropy(h)) / temperature
    # The token's own entry, (1 - p) on_lp / temperature and the entropy's
    # part, moves with p by as much, and is a product of its own: 1 /
    # temperature and two products are rounded once each (2^-24), and expm1
    # is within one unit in the last place (2^-23).
    absolute[token] += 5 * 2.0**-24 * (abs(on_lp) * float(-torch.expm1(logp[token])) +
                                       abs(on_h) * float(p[token]) * (abs(float(logp[token])) + abs(h))) / temperature
    # An exponential below 2^-126 (of the maximum's, at most the sum) is
    # flushed to zero: p is then off by at most 2^-126, and the gradient by
    # that times size / temperature, which exceeds the type's smallest number
    # for large |d| and small temperatures.
    absolute = absolute + 2.0**-126 * size / temperature
    return absolute + grad.abs() * HALF_STEP[dtype] * 1.01 + SMALLEST[dtype]


def test_rows(generator, rows, vocab, dtype, scale=3.0):
    """Logits of N(0, scale^2) with a few peaks, on the CPU."""
    x = torch.randn(rows, vocab, generator=generator, dtype=torch.float64) * scale
    for r in range(rows):
        at = torch.randint(vocab, (min(vocab, 16),), generator=generator)
        x[r, at] += 10 * torch.rand(at.numel(), generator=generator, dtype=torch.float64)
    return x.to(dtype)


test_rows.__test__ = False
