"""The row operators on logits (exactsample_b200.scoring), as cases to measure:

* token_logprobs: log-probability of one token per row and the row's entropy,
  forward, and with its gradient;
* top_logits: the k largest logits of each row, their ids, and the log-sum of
  the rest (the record a teacher leaves for distillation, and the top
  log-probabilities a server reports);
* distill_loss: KL(teacher || student) against such a record, with its gradient;
* policy_loss: the clipped policy-ratio loss with a KL and an entropy term,
  with its gradient.

``own`` false: the same results from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

VOCAB = 151_936  # the benchmark configurations' vocabulary
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def listed():
    return [
        # One sequence decoding: the log-probability of the token just sampled.
        dict(name="logprobs one row", op="logprobs", how="loss", rows=1, vocab=VOCAB, dtype="bf16", temperature=1.0,
             mask=False, ignored=0),
        # A serving batch (the headline's 128 requests, fp32 logits) with grammar masks, sampled at 0.6.
        dict(name="logprobs batch masked", op="logprobs", how="loss", rows=128, vocab=VOCAB, dtype="f32",
             temperature=0.6, mask=True, ignored=0),
        # Training on log-probabilities through autograd: 2,048 tokens, a third of a padded batch without a token.
        dict(name="logprobs autograd padded", op="logprobs", how="autograd", rows=2048, vocab=VOCAB, dtype="bf16",
             temperature=1.0, mask=False, ignored=683),
        # The top log-probabilities a server reports for eight requests.
        dict(name="top 20 of 8 rows", op="top", how="loss", rows=8, vocab=VOCAB, dtype="bf16", temperature=1.0,
             mask=False, ignored=0, k=20),
        # A teacher's pass over 2,048 tokens, 64 logits kept of each.
        dict(name="top 64 of 2048 rows", op="top", how="loss", rows=2048, vocab=VOCAB, dtype="bf16", temperature=1.0,
             mask=False, ignored=0, k=64),
        # An odd vocabulary in fp32 whose rows start at every alignment, at a distillation temperature.
        dict(name="top 128 odd vocabulary", op="top", how="loss", rows=777, vocab=50_257, dtype="f32",
             temperature=2.0, mask=False, ignored=0, k=128),
        # A drafter's small distillation step on a small vocabulary.
        dict(name="distill 64 rows small", op="distill", how="step", rows=64, vocab=32_000, dtype="f16",
             temperature=1.0, mask=False, ignored=0, k=16, tail=True),
        # A distillation step on a full batch: loss and gradient in one call.
        dict(name="distill step 4096 rows", op="distill", how="step", rows=4096, vocab=VOCAB, dtype="bf16",
             temperature=1.0, mask=False, ignored=0, k=64, tail=True),
        # fp32 logits of an odd vocabulary through autograd, the teacher renormalised over what it kept.
        dict(name="distill autograd odd", op="distill", how="autograd", rows=1001, vocab=50_257, dtype="f32",
             temperature=2.0, mask=False, ignored=0, k=128, tail=False),
        # The smallest policy step: 16 tokens, fp32 logits.
        dict(name="policy step 16 rows", op="policy", how="step", rows=16, vocab=VOCAB, dtype="f32", temperature=1.0,
             mask=False, ignored=0, kl=0.02, entropy=0.0),
        # A full policy step with the KL and the entropy term, tail rows padded.
        dict(name="policy step 4096 rows", op="policy", how="step", rows=4096, vocab=VOCAB, dtype="bf16",
             temperature=1.0, mask=False, ignored=200, kl=0.02, entropy=0.003),
        # Tokens sampled under grammar masks at 0.6, loss and gradient through autograd.
        dict(name="policy autograd masked", op="policy", how="autograd", rows=500, vocab=VOCAB, dtype="f16",
             temperature=0.6, mask=True, ignored=0, kl=0.0, entropy=0.01),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logprobs", "top", "distill", "policy"])
    vocab = rng.choice([VOCAB, log_int(500, 200_000), log_int(500, 200_000)])
    rows = log_int(1, max(1, min(8192, 300_000_000 // vocab)))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                temperature=rng.choice([1.0, 1.0, 0.6, round(rng.uniform(0.5, 2.0), 3)]),
                mask=rng.random() < 0.25, ignored=rng.choice([0, 0, rows // 3]))
    case["how"] = "loss" if op == "top" else rng.choice(["loss", "step", "autograd"])
    if op == "top":
        case["ignored"] = 0
    if op in ("top", "distill"):
        case["k"] = log_int(1, 256 if vocab > 1000 else 64)
    if op == "distill":
        case["tail"] = rng.random() < 0.7
    if op == "policy":
        case["kl"] = rng.choice([0.0, round(rng.uniform(0.001, 0.1), 4)])
        case["entropy"] = rng.choice([0.0, round(rng.uniform(0.001, 0.02), 4)])
    return case


# ---------------------------------------------------------------- inputs
def _logits(g, rows, vocab, dtype):
    """N(0, 2^2) noise plus U(8, 16) on 64 token ids per row, as the benchmark's synthetic rows (the ids one to
    each 64th of the row, so that they are distinct)."""
    x = torch.randn((rows, vocab), device="cuda", generator=g).mul_(2.0)
    span = vocab // 64
    ids = torch.randint(span, (rows, 64), device="cuda", generator=g) + span * torch.arange(64, device="cuda")
    x.scatter_(1, ids, torch.rand((rows, 64), device="cuda", generator=g) * 8 + 8)
    return x.to(dtype)


def _mask_words(g, rows, vocab):
    """Packed masks that allow about half of the tokens (bit t % 32 of word t // 32)."""
    words = torch.randint(0, 2**32, (rows, (vocab + 31) // 32), device="cuda", generator=g, dtype=torch.int64)
    words[:, 0] |= 1  # never empty
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)


def _allowed(words, vocab):
    bits = torch.arange(vocab, device=words.device)
    return (words[:, bits // 32] >> (bits % 32)) & 1 != 0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    s = dict(case=case, logits=_logits(g, rows, vocab, DTYPES[case["dtype"]]),
             mask=_mask_words(g, rows, vocab) if case["mask"] else None,
             temperature=case["temperature"])
    used = rows - case["ignored"]
    if case["op"] == "top":
        return s
    # A mean over the rows; fp16 gradients are scaled into their range, as fp16 training does.
    scale = 64.0 if case["dtype"] == "f16" else 1.0 / rows
    if case["op"] in ("distill", "policy"):
        s["weights"] = (0.5 + torch.rand((rows,), device="cuda", generator=g)) * scale
        scale = 1.0
    if case["how"] == "autograd":
        s["grad_out"] = (0.5 + torch.rand((rows,), device="cuda", generator=g)) * scale
        s["grad_entropy"] = -0.01 * torch.rand((rows,), device="cuda", generator=g) * scale
    elif case["how"] == "step":
        s["grad_out"] = -(0.5 + torch.rand((rows,), device="cuda", generator=g)) * scale
        s["grad_entropy"] = None
    x = s["logits"].float() / case["temperature"]
    if case["mask"]:
        x.masked_fill_(~_allowed(s["mask"], vocab), -math.inf)
    if case["op"] == "distill":
        # The teacher: near the student, its k largest logits and the log-sum of its others.
        t = torch.randn((rows, vocab), device="cuda", generator=g).mul_(0.7).add_(s["logits"])
        t.masked_fill_(x == -math.inf, -math.inf)
        k = min(case["k"], vocab)
        values, ids = t.topk(k, dim=1)
        t = t.scatter_(1, ids, -math.inf).div_(case["temperature"])
        ids[used:] = -1
        s.update(values=values, ids=ids, rest=t.logsumexp(1) if case["tail"] else None)
    else:
        # Tokens drawn from the rows' own distributions.
        noise = torch.rand((rows, vocab), device="cuda", generator=g).clamp_(min=1e-20).log_().neg_().log_()
        tokens = (x - noise).argmax(1)
        del noise
        if case["op"] == "policy":
            m = x.amax(1, keepdim=True)
            logprobs = (x.gather(1, tokens[:, None]) - m)[:, 0] - (x - m).exp_().sum(1).log()
            # The ratio's logarithm, kept clear of the two clip borders.
            ratio = 0.25 * torch.randn((rows,), device="cuda", generator=g)
            for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
                ratio = torch.where((ratio - border).abs() < 1e-3, ratio + 3e-3, ratio)
            s["old_logprobs"] = logprobs - ratio
            s["ref_logprobs"] = logprobs + 0.4 * torch.randn((rows,), device="cuda", generator=g) if case["kl"] else None
            s["advantages"] = torch.randn((rows,), device="cuda", generator=g)
        tokens[used:] = -1
        s["tokens"] = tokens
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"logprobs": _plain_logprobs, "top": _plain_top, "distill": _plain_distill,
            "policy": _plain_policy}[state["case"]["op"]](state)


def _run_own(s):
    from exactsample_b200 import scoring

    case, logits = s["case"], s["logits"]
    common = dict(temperature=s["temperature"], mask=s["mask"])
    how = case["how"]
    grad = torch.empty_like(logits) if how == "step" else None
    if case["op"] == "top":
        out = scoring.top_logits(logits, case["k"], **common)
        return dict(values=out.values, ids=out.ids, rest=out.rest, status=out.status)
    leaf = logits.detach().requires_grad_() if how == "autograd" else logits
    if case["op"] == "logprobs":
        if how == "step":
            common.update(grad=grad, grad_logprobs=s["grad_out"])
        out = scoring.token_logprobs(leaf, s["tokens"], **common)
        if how == "autograd":
            grad, = torch.autograd.grad((out.logprobs, out.entropy), leaf, (s["grad_out"], s["grad_entropy"]))
        got = dict(logprobs=out.logprobs.detach(), entropy=out.entropy.detach(), status=out.status)
    elif case["op"] == "distill":
        teacher = scoring.TopLogits(s["values"], s["ids"], s["rest"])
        out = scoring.distill_loss(leaf, teacher, weights=s["weights"], tail=case["tail"], grad=grad, **common)
        if how == "autograd":
            grad, = torch.autograd.grad(out.loss, leaf, s["grad_out"])
        got = dict(loss=out.loss.detach(), status=out.status)
    else:
        out = scoring.policy_loss(leaf, s["tokens"], s["old_logprobs"], s["advantages"],
                                  ref_logprobs=s["ref_logprobs"], weights=s["weights"], clip_low=CLIP_LOW,
                                  clip_high=CLIP_HIGH, kl_coef=case["kl"], entropy_coef=case["entropy"], grad=grad,
                                  **common)
        if how == "autograd":
            grad, = torch.autograd.grad(out.loss, leaf, s["grad_out"])
        got = dict(loss=out.loss.detach(), logprobs=out.logprobs, kl=out.kl, entropy=out.entropy, status=out.status)
    if grad is not None:
        got["grad"] = grad
    return got


def _plain_rows(s):
    """The rows' logits over the temperature, masked, in 32 bits."""
    x = s["logits"].float() / s["temperature"]
    if s["mask"] is not None:
        x = x.masked_fill(~_allowed(s["mask"], x.shape[1]), -math.inf)
    return x


def _plain_status(m):
    bad = torch.isnan(m) | (m == math.inf)
    return torch.where(bad, 2, torch.where(m == -math.inf, 1, 0)).to(torch.int32)


def _plain_logsoftmax(s):
    """log p of every token (the sum of exponentials in 64 bits), and the statuses."""
    x = _plain_rows(s)
    m = x.amax(1, keepdim=True)
    x = x - m
    log_sum = x.exp().sum(1, keepdim=True, dtype=torch.float64).log().float()
    return x - log_sum, _plain_status(m[:, 0])


def _plain_entropy(logp):
    p = logp.exp()
    return -torch.where(p > 0, p * logp, 0.0).sum(1), p


def _plain_token_grad(s, logp, p, entropy, on_logprob, on_entropy):
    """Gradient of sum(on_logprob * log p[token] + on_entropy * entropy) by the rows' raw logits."""
    tokens = s["tokens"]
    used = tokens >= 0
    a = torch.where(used, on_logprob, 0.0)[:, None]
    grad = p * -a
    if on_entropy is not None:
        b = torch.where(used, on_entropy, 0.0)[:, None]
        grad -= torch.where(p > 0, p * (logp + entropy[:, None]), 0.0) * b
    at = tokens.clamp(min=0)[:, None]
    grad.scatter_add_(1, at, a)
    return (grad / s["temperature"]).to(s["logits"].dtype)


def _plain_logprobs(s):
    logp, status = _plain_logsoftmax(s)
    entropy, p = _plain_entropy(logp)
    used = s["tokens"] >= 0
    logprobs = logp.gather(1, s["tokens"].clamp(min=0)[:, None])[:, 0]
    got = dict(logprobs=torch.where(used, logprobs, 0.0), entropy=torch.where(used, entropy, 0.0),
               status=torch.where(used, status, 0))
    if s["case"]["how"] != "loss":
        got["grad"] = _plain_token_grad(s, logp, p, entropy, s["grad_out"], s["grad_entropy"])
    return got


def _plain_top(s):
    x = _plain_rows(s)
    vocab = x.shape[1]
    raw = s["logits"].float()
    if s["mask"] is not None:
        raw = raw.masked_fill(x == -math.inf, -math.inf)
    # Distinct keys: the value's bits in order, then the lowest id first.
    bits = (raw + 0.0).view(torch.int32).to(torch.int64)
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    keys = bits * 2**20 + (2**20 - 1 - torch.arange(vocab, device=x.device))
    k = min(s["case"]["k"], vocab)
    ids = keys.topk(k, dim=1).indices
    values = raw.gather(1, ids)
    m = x.amax(1)
    rest = x.scatter(1, ids, -math.inf)
    top = rest.amax(1, keepdim=True).clamp(min=-3e38)
    rest = top[:, 0] + (rest - top).exp().sum(1, dtype=torch.float64).log().float()
    if k < s["case"]["k"]:
        pad = (0, s["case"]["k"] - k)
        values, ids = torch.nn.functional.pad(values, pad, value=-math.inf), torch.nn.functional.pad(ids, pad, value=-1)
    return dict(values=values, ids=torch.where(values > -math.inf, ids, -1), rest=rest, status=_plain_status(m))


def _plain_distill(s):
    case = s["case"]
    x = _plain_rows(s)
    m = x.amax(1, keepdim=True)
    x = x - m
    at = s["ids"].clamp(min=0)
    used = s["ids"][:, 0] >= 0
    mine = x.gather(1, at).double()
    e = x.exp()
    others = e.scatter(1, at, 0.0).sum(1, dtype=torch.float64)
    total = others + mine.exp().sum(1)
    log_total = total.log()[:, None]
    # The teacher: its kept logits and, with the tail, one bucket for the rest.
    t = s["values"].double() / s["temperature"]
    log_t = t.logsumexp(1, keepdim=True)
    if case["tail"]:
        log_t = torch.logaddexp(log_t, s["rest"].double()[:, None])
        t_rest = s["rest"].double() - log_t[:, 0]
    t = t - log_t
    loss = (t.exp() * (t - (mine - log_total))).sum(1)
    pull = torch.ones_like(loss)
    if case["tail"]:
        off = t_rest - (others.log() - log_total[:, 0])
        some = t_rest > -math.inf
        loss = loss + torch.where(some, t_rest.exp() * off, 0.0)
        pull = torch.where(some, 1 - off.exp(), 1.0)
    weights = torch.where(used, s["weights"], 0.0)
    got = dict(loss=torch.where(used, loss.float() * weights, 0.0), status=torch.where(used, _plain_status(m[:, 0]), 0))
    if case["how"] != "loss":
        if case["how"] == "autograd":
            weights = weights * s["grad_out"]
        scale = weights.double() / s["temperature"]
        grad = e * (scale * pull / total).float()[:, None]
        on_top = ((mine - log_total).exp() - t.exp()) * scale[:, None]
        got["grad"] = grad.scatter_(1, at, torch.where(used[:, None], on_top, 0.0).float()).to(s["logits"].dtype)
    return got


def _plain_policy(s):
    case = s["case"]
    logp, status = _plain_logsoftmax(s)
    entropy, p = _plain_entropy(logp)
    used = s["tokens"] >= 0
    logprobs = logp.gather(1, s["tokens"].clamp(min=0)[:, None])[:, 0]
    # Row scalars in 64 bits: the ratio's borders and the KL term's cancellation.
    lp, a = logprobs.double(), s["advantages"].double()
    ratio = (lp - s["old_logprobs"].double()).exp()
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    loss = -torch.minimum(ratio * a, clipped * a)
    slope = torch.where(ratio * a <= clipped * a, -ratio * a, 0.0)
    kl = torch.zeros_like(loss)
    if s["ref_logprobs"] is not None:
        d = s["ref_logprobs"].double() - lp
        kl = torch.expm1(d) - d
        loss = loss + case["kl"] * kl
        slope = slope - case["kl"] * torch.expm1(d)
    loss = (loss - case["entropy"] * entropy.double()) * s["weights"].double()
    zero = torch.zeros_like(entropy)
    got = dict(loss=torch.where(used, loss.float(), zero), logprobs=torch.where(used, logprobs, zero),
               kl=torch.where(used, kl.float(), zero), entropy=torch.where(used, entropy, zero),
               status=torch.where(used, status, 0))
    if case["how"] != "loss":
        weights = s["weights"] * s["grad_out"] if case["how"] == "autograd" else s["weights"]
        on_entropy = -case["entropy"] * weights if case["entropy"] else None
        got["grad"] = _plain_token_grad(s, logp, p, entropy, (slope * weights.double()).float(), on_entropy)
    return got


# ---------------------------------------------------------------- counts
def work(case):
    rows, vocab = case["rows"], case["vocab"]
    read = rows - case["ignored"]  # a row without a token or a teacher need not be read
    size = 4 if case["dtype"] == "f32" else 2
    nbytes = read * vocab * size + rows * 64
    if case["mask"]:
        nbytes += read * ((vocab + 31) // 32) * 4
    # Subtract, scale, exponential and sum of every token; the gradient's exponential and products again.
    flops = 4.0 * read * vocab
    if case["op"] in ("logprobs", "policy"):
        flops += 2.0 * read * vocab  # the entropy's product and sum
    if case["op"] in ("top", "distill"):
        nbytes += rows * case["k"] * 12
    if case["op"] != "top" and case["how"] != "loss":
        nbytes += rows * vocab * size
        flops += 4.0 * read * vocab
    return dict(bytes=nbytes, flops=flops)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    z = s["logits"].double()
    if s["mask"] is not None:
        word = torch.arange(case["vocab"], device=z.device)
        z[((s["mask"][:, word >> 5] >> (word & 31)) & 1) == 0] = -math.inf
    x = z / case["temperature"]
    lse = torch.logsumexp(x, 1)
    how, op = case["how"], case["op"]
    if op == "top":
        k = min(case["k"], case["vocab"])
        order = torch.sort(z, dim=1, descending=True, stable=True)
        values, ids = order.values[:, :k], order.indices[:, :k]
        rest = torch.logsumexp(order.values[:, k:] / case["temperature"], 1) if k < case["vocab"] else \
            torch.full_like(lse, -math.inf)
        if k < case["k"]:
            values = torch.cat([values, values.new_full((case["rows"], case["k"] - k), -math.inf)], 1)
        return dict(values=values, ids=None, rest=rest, status=None)
    n = case["rows"] - case["ignored"]  # the rows behind these have no token and no teacher
    row = torch.arange(n, device=z.device)
    grad = None if how == "loss" else torch.zeros_like(z)
    upstream = s["grad_out"][:n].double() if how == "autograd" else 1.0

    def padded(v):
        out = torch.zeros(case["rows"], dtype=torch.float64, device=z.device)
        out[:n] = v
        return out

    if op == "distill":
        ids = s["ids"][:n]
        t = s["values"][:n].double() / case["temperature"]
        if case["tail"]:
            t = torch.cat([t, s["rest"][:n].double()[:, None]], 1)
        t = torch.log_softmax(t, 1)
        mine = x[:n].gather(1, ids) - lse[:n, None]
        others = torch.logsumexp(x[:n].scatter(1, ids, -math.inf), 1) - lse[:n]
        if case["tail"]:
            mine = torch.cat([mine, others[:, None]], 1)
        loss = torch.where(t > -math.inf, t.exp() * (t - mine), 0.0).sum(1)
        w = s["weights"][:n].double()
        if grad is not None:
            # By each token's own logit: q - target, where the rest's target is spread as q is.
            q = (x[:n] - lse[:n, None]).exp()
            target = torch.zeros_like(q)
            if case["tail"]:
                target = q * (t[:, -1] - others).exp()[:, None]
                target[torch.isnan(target)] = 0.0
            target.scatter_(1, ids, t[:, :ids.shape[1]].exp())
            grad[:n] = (q - target) * (w * upstream / case["temperature"])[:, None]
        out = dict(loss=padded(loss * w), status=None)
    else:
        tokens = s["tokens"][:n]
        logp = x[:n] - lse[:n, None]
        lp = logp[row, tokens]
        p = logp.exp()
        plogp = p * logp
        plogp[p == 0] = 0.0
        h = -plogp.sum(1)
        if op == "logprobs":
            on_lp = on_h = None
            if grad is not None:
                on_lp = s["grad_out"][:n].double()
                on_h = None if s["grad_entropy"] is None else s["grad_entropy"][:n].double()
            out = dict(logprobs=padded(lp), entropy=padded(h), status=None)
        else:
            adv, w = s["advantages"][:n].double(), s["weights"][:n].double()
            r = torch.exp(lp - s["old_logprobs"][:n].double())
            inside = torch.clamp(r, 1 - CLIP_LOW, 1 + CLIP_HIGH)
            value = torch.maximum(-adv * r, -adv * inside)
            d_lp = torch.where(-adv * r >= -adv * inside, -adv * r, torch.zeros_like(r))
            kl = torch.zeros_like(r)
            if s["ref_logprobs"] is not None:
                gap = s["ref_logprobs"][:n].double() - lp
                kl = gap.exp() - 1 - gap
                value = value + case["kl"] * kl
                d_lp = d_lp + case["kl"] * (1 - gap.exp())
            value = (value - case["entropy"] * h) * w
            on_lp, on_h = d_lp * w * upstream, -case["entropy"] * w * upstream
            out = dict(loss=padded(value), logprobs=padded(lp), kl=padded(kl), entropy=padded(h), status=None)
        if grad is not None:
            grad[:n] = -p * on_lp[:, None]
            grad[row, tokens] += on_lp
            if on_h is not None:
                grad[:n] -= (plogp + p * h[:, None]) * on_h[:, None]
            grad /= case["temperature"]
    if grad is not None:
        out["grad"] = grad
    return out
