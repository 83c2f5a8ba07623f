"""The row operators on the GPU where a factor leaves float32's range though
the result does not, and in the calls around them: derivatives that they do not
have, teachers that failed, saving, tracing, gradients handed on to a layer, and
gradients that lie otherwise than the logits do."""
import math

import pytest
import torch

from exactsample_b200 import Status, scoring
from tests import scoring_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def names(value):
    return str(value).replace("torch.", "")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


def sum_error(x, vocab):
    """How far a 32-bit sum of exp(x - max) may be from the exact one,
    relatively: the exponentials 2^-22 and their arguments (three roundings of
    the exponent), one thread's partial sum (128 threads of two partial sums
    over at most 25,600 tokens of a rank, or its share of a longer slice), and
    24 joins of a product and a sum."""
    live = x[x > -math.inf]
    if live.numel() == 0:
        return 0.0
    p, d = torch.softmax(live, 0), (live - live.max()).abs()
    terms = max(100.0, vocab / 16 / 128 / 2)
    return 2.0**-22 + (terms + 48) * 2.0**-24 + 3 * 2.0**-24 * float((p * d).sum())


# ---------------------------------------------------------------- distillation
def distill_exact(z, values, ids, rest, temperature):
    """The loss and its gradient by the row's logits, in 64 bits, from the
    definition: q - t for a kept token, q_j (1 - t_rest / q_rest) for another.
    Also each gradient's two terms, for the error bound."""
    x = z / temperature
    t = torch.log_softmax(torch.cat([values / temperature, rest[None]]), 0)
    others = x.clone()
    others[ids] = -math.inf
    total = torch.logsumexp(x, 0)
    q_rest = torch.logsumexp(others, 0) - total
    mine = torch.cat([x[ids] - total, q_rest[None]])
    loss = torch.where(t > -math.inf, t.exp() * (t - mine), 0.0).sum()
    pushed = (t[-1] + torch.log_softmax(others, 0)).exp()
    pushed[ids] = t[:-1].exp()
    q = (x - total).exp()
    return loss, (q - pushed) / temperature, q, pushed, t, mine, others


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [40, 1000, 50_257])
@pytest.mark.parametrize("gap", [30.0, 87.5, 90.0, 100.0, 104.0, 120.0, 700.0, "lowest"])
@pytest.mark.parametrize("temperature", [1.0, 0.1])
def test_distillation_where_the_student_has_almost_nothing_beside_the_kept(dtype, vocab, gap, temperature):
    """The student's other tokens lie `gap` nats and more below its kept ones,
    while the teacher has mass there: 1 - t_rest / q_rest leaves float32's
    range, the gradient does not."""
    g = torch.Generator().manual_seed(vocab)
    rows = 4
    kept = torch.tensor([1, 0, vocab // 2, vocab - 1])
    x = torch.rand(rows, vocab, generator=g, dtype=torch.float64) * 3 * temperature
    far = torch.finfo(dtype).min if gap == "lowest" else -gap * temperature
    if gap == "lowest":
        x[:] = far
    else:
        x += far - 3 * temperature
    x[:, kept] = torch.rand(rows, 4, generator=g, dtype=torch.float64) * temperature
    x = x.to(dtype)
    values = (torch.rand(rows, 4, generator=g) * temperature).sort(1, descending=True).values
    rest = torch.tensor([-2.2, 0.5, -5.0, 3.0])
    weights = torch.tensor([1.0, 0.7, 1.3, 1.0])
    record = scoring.TopLogits(values.cuda(), kept.expand(rows, 4).cuda(), rest.cuda())
    grad = torch.full_like(x, 5.0, device="cuda")
    args = dict(weights=weights.cuda(), temperature=temperature)
    out = scoring.distill_loss(x.cuda(), record, grad=grad, **args)
    leaf = x.cuda().requires_grad_()
    scoring.distill_loss(leaf, record, **args).loss.sum().backward()
    assert torch.equal(leaf.grad, grad)
    for r in range(rows):
        z, w = x[r].double(), float(weights[r])
        want, slope, q, pushed, t, mine, others = distill_exact(z, values[r].double(), kept, rest[r].double(), temperature)
        # Logits that leave float32's range when divided are held at its
        # lowest number: the loss is then no answer to compare with.
        far_out = float((z / temperature).abs().max()) > 3e38 or w * float(want) > 1e37
        if far_out and int(out.status[r]) != 0:
            assert int(out.status[r]) == int(Status.INVALID_INPUT) and bool((grad[r] == 0).all())
            continue
        assert int(out.status[r]) == 0, r
        error, part = sum_error(others, vocab), 20 * 2.0**-24  # part: see check_distill's derivation in test_gpu_scoring.py
        off = (t - mine).abs()
        if not far_out:
            limit = float((t.exp() * off).sum()) * (part + 6 * 2.0**-24) + 2 * error + 3 * part
            limit += 4 * 2.0**-24 * float(mine.abs().clamp(max=1e38)[:-1].max())
            assert abs(float(out.loss[r]) - w * float(want)) <= w * limit + 2.0**-23 * w * float(want), r
        # Each of a gradient's two terms: both sums' errors, both totals'
        # (part), an exponential (2^-22, and its argument's three roundings)
        # and six products; 2^-126 where an exponential or a share is flushed.
        d = (others - others.max()).clamp(min=-200).abs()
        relative = 2 * error + 2 * part + 2.0**-22 + 3 * 2.0**-24 * d + 6 * 2.0**-24
        limit = w / temperature * ((q + pushed) * relative + 2.0**-125)
        limit = limit + w * slope.abs() * ref.HALF_STEP[dtype] * 1.01 + ref.SMALLEST[dtype]
        difference = (grad[r].cpu().double() - w * slope).abs()
        assert bool((difference <= limit).all()), (r, float((difference / limit).max()))


# ---------------------------------------------------------------- policy
def policy_case(rows=6, vocab=700, dtype=torch.float32, seed=11):
    g = torch.Generator().manual_seed(seed)
    x = ref.test_rows(g, rows, vocab, dtype)
    tokens = torch.randint(vocab, (rows,), generator=g)
    lp = torch.log_softmax(x.double(), 1).gather(1, tokens[:, None])[:, 0]
    return g, x, tokens, lp


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_a_kl_that_is_only_watched_does_not_fail_its_row(dtype):
    """kl_coef 0 with ref_logprobs: a KL beyond float32 is its largest number,
    and the loss, its gradient and the log-probability are those without one."""
    g, x, tokens, lp = policy_case(dtype=dtype)
    gap = torch.tensor([1.0, 88.0, 89.0, 104.0, 800.0, 1e5])
    old, adv = (lp - 0.05).float().cuda(), torch.randn(6, generator=g).cuda()
    grads = [torch.full_like(x, 5.0, device="cuda") for _ in range(2)]
    args = (x.cuda(), tokens.cuda(), old, adv)
    watched = scoring.policy_loss(*args, ref_logprobs=(lp + gap).float().cuda(), entropy_coef=0.01, grad=grads[0])
    without = scoring.policy_loss(*args, entropy_coef=0.01, grad=grads[1])
    assert watched.status.cpu().tolist() == [0] * 6
    for name in ("loss", "logprobs", "entropy", "status"):
        assert torch.equal(getattr(watched, name), getattr(without, name)), name
    assert torch.equal(*grads)
    largest = torch.finfo(torch.float32).max
    assert watched.kl[2:].cpu().tolist() == [largest] * 4
    # exp(d) - 1 - d moves by a factor of d's error: log p's 2^-24 |log p|, the
    # input's own rounding, d's two, and the sums' (2^-18 is above all of them).
    for r, rise in ((0, 1.0), (1, 88.0)):
        d = float((lp + gap).float()[r].double() - lp[r])
        want = math.expm1(d) - d
        assert abs(float(watched.kl[r]) - want) <= want * 2.0**-16 * max(1.0, 1 / rise)


def test_losses_whose_factors_alone_leave_the_range():
    """A ratio or a KL beyond float32 times a small advantage or coefficient."""
    g, x, tokens, lp = policy_case()
    x, tokens, lp = x[:4], tokens[:4], lp[:4]
    old = torch.stack([lp[0] - 100, lp[1] - 95, lp[2], lp[3] - 100]).float()
    adv = torch.tensor([-1e-8, -1e-6, 1.0, -1.0])
    reference = torch.stack([lp[0], lp[1], lp[2] + 100, lp[3]]).float()
    grad = torch.full_like(x, 5.0, device="cuda")
    out = scoring.policy_loss(x.cuda(), tokens.cuda(), old.cuda(), adv.cuda(), ref_logprobs=reference.cuda(),
                              kl_coef=1e-8, grad=grad)
    assert out.status.cpu().tolist() == [0, 0, 0, 2]  # the last row's loss is beyond float32
    p = torch.softmax(x.double(), 1)
    for r in range(3):
        ratio = math.exp(float(lp[r] - old[r].double()))
        d = float(reference[r].double() - lp[r])
        clipped = min(max(ratio, 0.8), 1.2)
        a = float(adv[r])
        through = ratio * a <= clipped * a
        want = -min(ratio * a, clipped * a) + 1e-8 * (math.expm1(d) - d)
        slope = (-ratio * a if through else 0.0) - 1e-8 * math.expm1(d)
        # ratio and exp(d) move with log p: its rounding (2^-24 |log p|) and
        # its sums' (sum_error), 2^-18 with room for their arguments' roundings
        # at 100 (two of 2^-24 100 each).
        relative = 2.0**-24 * (4 * 100 + 2 * abs(float(lp[r]))) + sum_error(x[r].double(), 700) + 2.0**-21
        assert abs(float(out.loss[r]) - want) <= relative * max(abs(want), 1.0), r
        row = -p[r] * slope
        row[tokens[r]] += slope
        limit = abs(slope) * (p[r] + (1 - p[r][tokens[r]]) * (torch.arange(700) == tokens[r])) * (2 * relative + 2.0**-20) + 1e-30
        assert bool(((grad[r].cpu().double() - row).abs() <= limit).all()), r
    assert float(out.kl[2]) == torch.finfo(torch.float32).max


@pytest.mark.parametrize("adv", [1.0, -1.0])
@pytest.mark.parametrize("above", [10.0, 200.0, 1e30])
def test_a_masked_token_is_one_without_probability(adv, above):
    """Whatever its hidden logit is and wherever the ratio goes."""
    g, x, tokens, _ = policy_case(rows=3)
    allowed = torch.ones(3, 700, dtype=torch.bool)
    allowed[torch.arange(3), tokens] = False
    x[torch.arange(3), tokens] = above
    x[1, tokens[1]] = -math.inf
    mask = ref.pack_mask(allowed).cuda()
    column = torch.tensor([-5.0, -5.0, -5.0]).cuda()
    grad = torch.full_like(x, 5.0, device="cuda")
    out = scoring.policy_loss(x.cuda(), tokens.cuda(), column, torch.full((3,), adv, device="cuda"), ref_logprobs=column,
                              kl_coef=0.1, mask=mask, grad=grad)
    alone = scoring.token_logprobs(x.cuda(), tokens.cuda(), mask=mask)
    assert out.status.cpu().tolist() == alone.status.cpu().tolist() == [int(Status.DRAFT_ZERO_PROB)] * 3
    assert bool((grad == 0).all()) and bool((out.loss == 0).all()) and bool((out.kl == 0).all())
    # A bad input says so first, as it does for a token with probability.
    column[2] = math.nan
    out = scoring.policy_loss(x.cuda(), tokens.cuda(), column, torch.full((3,), adv, device="cuda"), mask=mask)
    assert out.status.cpu().tolist() == [3, 3, 2]


# ---------------------------------------------------------------- far logits
@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("far", [-1e30, -1.7e38, -2.3e38, "lowest", "mask", -math.inf])
@pytest.mark.parametrize("incoming", [0.4, 3.0, -700.0, 65536.0, 1e12])
def test_entropy_gradients_beside_very_low_logits(dtype, far, incoming):
    """A token without probability has a gradient of 0, however far below the
    others its logit lies and however large the incoming gradient is."""
    lowest = torch.finfo(dtype).min
    if not isinstance(far, str) and far != -math.inf and far < lowest:
        pytest.skip("not a number of the type")
    g = torch.Generator().manual_seed(3)
    rows, vocab = 3, 4200
    x = ref.test_rows(g, rows, vocab, dtype)
    live = torch.rand(rows, vocab, generator=g) < 0.4
    live[0] = False
    live[0, [7, 4100]] = True       # a row of two tokens
    live[1, :1100] = True           # the others lie behind a warp's first tokens
    tokens = live.float().argmax(1)
    mask = None
    if far == "mask":
        mask = ref.pack_mask(live).cuda()
    else:
        x = torch.where(live, x, torch.tensor(lowest if far == "lowest" else far).to(dtype))
    on_lp = torch.tensor([0.5, -1.0, 2.0])
    for temperature in (1.0, 2.0, 0.2):
        grad = torch.full_like(x, 5.0, device="cuda")
        out = scoring.token_logprobs(x.cuda(), tokens.cuda(), temperature=temperature, mask=mask, grad=grad,
                                     grad_logprobs=on_lp.cuda(), grad_entropy=torch.full((rows,), incoming).cuda())
        assert out.status.cpu().tolist() == [0] * rows
        for r in range(rows):
            logp = ref.logp_of(x[r].double(), live[r], temperature)
            h = float(ref.entropy_of(logp))
            p = logp.exp()
            want = -p * float(on_lp[r]) - incoming * torch.where(live[r], p * (logp + h), 0.0)
            want[tokens[r]] += float(on_lp[r])
            want /= temperature
            bounds = ref.RowBounds(logp, vocab)
            bounds.sum = sum_error(x[r].double() / temperature if far != "mask" else
                                   (x[r].double() / temperature).masked_fill(~live[r], -math.inf), vocab)
            limit = ref.token_grad_bound(bounds, logp, want, int(tokens[r]), float(on_lp[r]), incoming, h, temperature, dtype)
            got = grad[r].cpu().double()
            over = want.abs() > torch.finfo(dtype).max  # (float16 and a large incoming gradient)
            off = (got - want).abs()
            assert bool((off <= limit)[~over].all()), (temperature, r, float((off / limit)[~over].max()))
            assert bool((got[~live[r]] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [2, 40, 129, 300, 600, 1001, 50_257])
@pytest.mark.parametrize("masked", [False, True], ids=["open", "masked"])
def test_logits_at_the_types_highest(dtype, vocab, masked):
    """Rows whose exponents' reference is beyond float32, at sizes that leave
    threads of a warp without tokens."""
    highest = torch.finfo(dtype).max
    x = torch.zeros(3, vocab, dtype=dtype)
    x[0, 0] = highest
    x[1] = highest
    x[2, -1] = highest / 256
    tokens = torch.tensor([0, vocab // 2, vocab - 1])
    mask = ref.pack_mask(torch.ones(3, vocab, dtype=torch.bool)).cuda() if masked else None
    teacher = scoring.TopLogits(torch.zeros(1, 1, device="cuda"), torch.zeros(1, 1, dtype=torch.int64, device="cuda"),
                                torch.full((1,), 0.5, device="cuda"))
    log_v = math.log(vocab)
    for temperature in (1.0, 0.01):
        grad = torch.full_like(x, 5.0, device="cuda")
        ones = torch.ones(3, device="cuda")
        out = scoring.token_logprobs(x.cuda(), tokens.cuda(), temperature=temperature, mask=mask, grad=grad,
                                     grad_logprobs=ones, grad_entropy=ones)
        assert out.status.cpu().tolist() == [0, 0, 0]
        limit = sum_error(torch.zeros(vocab), vocab) + 2.0**-23 * log_v
        for got, want in ((out.logprobs, [0, -log_v, 0]), (out.entropy, [0, log_v, 0])):
            assert float((got.cpu().double() - torch.tensor(want).double()).abs().max()) <= 3 * limit
        want = torch.full((vocab,), -1 / vocab, dtype=torch.float64)
        want[vocab // 2] += 1
        assert bool((grad[[0, 2]] == 0).all())
        bound = (want.abs() * ref.HALF_STEP[dtype] + 6 * limit / vocab) * 1.01 + ref.SMALLEST[dtype]
        bound[vocab // 2] += 6 * limit
        assert bool(((grad[1].cpu().double() * temperature - want).abs() <= bound).all())
        # Distillation against the row of equal logits: t and q of two classes.
        got = scoring.distill_loss(x[1:2].cuda(), teacher, temperature=temperature, mask=None if mask is None else mask[1:2])
        t = torch.softmax(torch.tensor([0.0, 0.5], dtype=torch.float64), 0)
        loss = float((t * (t.log() - torch.tensor([1 / vocab, 1 - 1 / vocab]).double().log())).sum())
        assert int(got.status[0]) == 0
        assert abs(float(got.loss[0]) - loss) <= 3 * limit + 40 * 2.0**-24 * (1 + abs(loss))


# ---------------------------------------------------------------- rows with one likely token
@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [700, 32_000, 151_936])
@pytest.mark.parametrize("kind", ["open", "masked", "infinities"])
@pytest.mark.parametrize("peak", [18, 24, 30, 40])
def test_rows_whose_token_has_most_of_the_mass(dtype, vocab, kind, peak):
    """The digits of small entropies and of log-probabilities near 0, wherever
    in the row the token lies; none past the end of its range."""
    g = torch.Generator(device="cuda").manual_seed(peak)
    rows = 48
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 2
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    tokens[:2] = torch.tensor([0, vocab - 1])
    x.scatter_(1, tokens[:, None], peak + torch.rand(rows, 1, device="cuda", generator=g))
    allowed = torch.ones(rows, vocab, dtype=torch.bool, device="cuda")
    if kind != "open":
        allowed = torch.rand(rows, vocab, device="cuda", generator=g) < 0.6
        allowed.scatter_(1, tokens[:, None], True)
    if kind == "infinities":
        x.masked_fill_(~allowed, -math.inf)
    x = x.to(dtype)
    mask = ref.pack_mask(allowed.cpu()).cuda() if kind == "masked" else None
    grads = [torch.empty_like(x) for _ in range(2)]
    ones = torch.ones(rows, device="cuda")
    out = scoring.token_logprobs(x, tokens, mask=mask, grad=grads[0], grad_entropy=ones)
    step = scoring.policy_loss(x, tokens, out.logprobs, torch.zeros_like(ones), mask=mask, entropy_coef=-1.0, grad=grads[1])
    assert torch.equal(step.logprobs, out.logprobs) and torch.equal(step.entropy, out.entropy)
    logp = torch.log_softmax(x.double().masked_fill(~allowed, -math.inf), 1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    h, lp = -plogp.sum(1), logp.gather(1, tokens[:, None])[:, 0]
    assert bool((out.logprobs <= 0).all()) and bool((out.entropy >= 0).all()) and not bool(out.status.any())
    # The token's exponential is 1 exactly, and the sum is 1 + rest: it is
    # rounded by each of the 26 joins of a row's partial sums and by a thread's
    # 100 additions to 1 while those come to half a unit, all of it at most the
    # rest itself and a few units where the rest is below one.
    rest = -torch.expm1(lp)
    lost = torch.minimum((26 + 100) * 2.0**-24 * torch.ones_like(rest), 4 * 2.0**-24 + 2 * rest)
    relative = 2.0**-15  # of the others' sums: exponents of at most 60 nats (3 * 2^-24 each), 130 roundings
    assert bool(((out.logprobs - lp).abs() <= lost + relative * lp.abs()).all())
    assert bool(((out.entropy - h).abs() <= lost + relative * h).all())
    # A gradient's factor log p + h is a quotient of sums at the token, and far
    # from 0 at the others: each is right to its own digits. (The exponents'
    # reference is rounded to 32 bits, by 2^-24 of the peak at most, and the
    # token's exponent is what that takes away: the quotient's sum has that in
    # it for as many as 130 additions, each rounded by 2^-24 of it, before it is
    # taken back.)
    want = -(plogp + p * h[:, None])
    back = torch.zeros_like(want).scatter_(1, tokens[:, None], 130 * 2.0**-48 * (peak + 1))
    for grad in grads:
        limit = want.abs() * (2 * relative + ref.HALF_STEP[dtype] * 1.01) + ref.SMALLEST[dtype] * 2 + 2.0**-126 * 100 + back
        assert bool(((grad.double() - want).abs() <= limit).all()), float(((grad.double() - want).abs() / limit).max())


def test_a_student_like_its_teacher_has_no_negative_loss():
    g = torch.Generator(device="cuda").manual_seed(17)
    logits = torch.randn(400, 5000, device="cuda", generator=g) * 3
    for k in (1, 20, 256):
        for tail in (True, False):
            out = scoring.distill_loss(logits, scoring.top_logits(logits, k), tail=tail)
            assert bool((out.loss >= 0).all())


# ---------------------------------------------------------------- the calls
def step_inputs(rows=6, vocab=700, seed=21):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(rows, vocab, device="cuda", generator=g)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    columns = [torch.randn(rows, device="cuda", generator=g) - 6 * (i == 0) for i in range(3)]
    return g, logits, tokens, columns, scoring.top_logits(logits * 0.8, 9)


def operator_calls(tokens, columns, teacher):
    return [lambda x, **kw: scoring.token_logprobs(x, tokens, **kw).logprobs,
            lambda x, **kw: scoring.policy_loss(x, tokens, columns[0], columns[1], entropy_coef=0.1, **kw).loss,
            lambda x, **kw: scoring.distill_loss(x, teacher, weights=columns[2], **kw).loss,
            lambda x, **kw: scoring.top_logits(x, 5, **kw).rest]


def test_forward_derivatives_are_refused():
    """None has one: a tangent of zeros would pass for it."""
    import torch.autograd.forward_ad as forward

    _, logits, tokens, columns, teacher = step_inputs()
    for call in operator_calls(tokens, columns, teacher):
        want = call(logits)
        with pytest.raises(RuntimeError, match="forward"):
            torch.func.jvp(call, (logits,), (torch.ones_like(logits),))
        for tracked in (False, True):
            with forward.dual_level():
                dual = forward.make_dual(logits.clone().requires_grad_(tracked), torch.ones_like(logits))
                with pytest.raises(RuntimeError, match="forward"):
                    call(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                    torch.ops.exactsample.token_logprobs(dual, tokens, None, 1.0, None, None, None, None)
        assert torch.equal(call(logits), want)  # nothing is left behind
    with forward.dual_level():  # an input other than the logits
        weights = forward.make_dual(torch.ones(6, device="cuda"), torch.ones(6, device="cuda"))
        with pytest.raises(RuntimeError, match="forward"):
            scoring.policy_loss(logits, tokens, *columns[:2], weights=weights)


def test_a_teacher_that_failed_is_not_padding():
    """Rows whose record is empty because the teacher's row failed have the
    teacher's status; padded rows are as they were."""
    g, logits, tokens, columns, _ = step_inputs()
    teacher_logits = logits * 0.8
    teacher_logits[1, 5] = math.nan
    teacher_logits[3] = -math.inf
    teacher = scoring.top_logits(teacher_logits, 9)
    assert teacher.status.cpu().tolist() == [0, 2, 0, 1, 0, 0]
    teacher.ids[4] = -1  # padding
    kept = torch.tensor([0, 2, 5])
    for weights in (None, columns[2]):
        grad = torch.full_like(logits, 5.0)
        out = scoring.distill_loss(logits, teacher, weights=weights, grad=grad)
        alone = scoring.distill_loss(logits, teacher, weights=weights)
        leaf = logits.clone().requires_grad_()
        tracked = scoring.distill_loss(leaf, teacher, weights=weights)
        tracked.loss.sum().backward()
        assert torch.equal(leaf.grad, grad)
        for got in (out, alone, tracked):
            assert got.status.cpu().tolist() == [0, 2, 0, 1, 0, 0]
            assert bool((got.loss[[1, 3, 4]] == 0).all()) and bool((got.loss[kept.cuda()] != 0).all())
        assert bool((grad[[1, 3, 4]] == 0).all()) and bool((grad[kept.cuda()] != 0).any(1).all())
        # Without the record's statuses an empty row is padding.
        bare = scoring.TopLogits(teacher.values, teacher.ids, teacher.rest)
        again = scoring.distill_loss(logits, bare, weights=weights)
        assert again.status.cpu().tolist() == [0] * 6 and torch.equal(again.loss, out.loss)
    # A strided column of statuses, and one of the wrong type.
    wide = torch.stack([teacher.status, teacher.status + 7], 1)
    strided = scoring.TopLogits(teacher.values, teacher.ids, teacher.rest, wide[:, 0])
    assert scoring.distill_loss(logits, strided).status.cpu().tolist() == [0, 2, 0, 1, 0, 0]
    with pytest.raises(RuntimeError, match="teacher_status has wrong"):
        scoring.distill_loss(logits, scoring.TopLogits(teacher.values, teacher.ids, teacher.rest, teacher.status.long()))


def test_results_are_saved_together(tmp_path):
    """Log-probabilities and statuses of one call in one file."""
    _, logits, tokens, columns, teacher = step_inputs()
    outs = [scoring.token_logprobs(logits, tokens), scoring.policy_loss(logits, tokens, *columns[:2]),
            scoring.distill_loss(logits, teacher), teacher]
    for out in outs:
        whole = {name: getattr(out, name) for name in out.__slots__}
        torch.save(whole, tmp_path / "results.pt")
        again = torch.load(tmp_path / "results.pt")
        assert all(torch.equal(again[name], whole[name]) for name in whole)


def test_grad_through_a_layer():
    """The call's gradient handed on to the layers before the logits: the same
    as through autograd, into memory of its own and into the logits'."""
    g = torch.Generator(device="cuda").manual_seed(22)
    rows, vocab = 12, 900
    hidden = torch.randn(rows, 32, device="cuda", generator=g)
    weight = (torch.randn(vocab, 32, device="cuda", generator=g) * 0.2).requires_grad_()
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    old, adv = torch.full((rows,), -7.0, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    scoring.policy_loss(hidden @ weight.t(), tokens, old, adv, entropy_coef=0.01).loss.sum().backward()
    want, weight.grad = weight.grad, None
    for over in (False, True):
        logits = hidden @ weight.t()
        flat = logits.detach()
        grad = flat if over else torch.empty_like(flat)
        scoring.policy_loss(flat, tokens, old, adv, entropy_coef=0.01, grad=grad)
        logits.backward(grad)
        assert torch.equal(weight.grad, want)
        weight.grad = None
    with pytest.raises(ValueError, match="grad= takes the gradient"):
        logits = hidden @ weight.t()
        scoring.policy_loss(logits, tokens, old, adv, grad=torch.empty_like(logits))


# ---------------------------------------------------------------- many rows, other layouts
def layout(rows, vocab, dtype, kind):
    if kind == "plain":
        return torch.full((rows, vocab), 3.0, dtype=dtype, device="cuda")
    if kind == "even":   # rows on 16 bytes whatever the vocabulary
        return torch.full((rows, (vocab + 7) // 8 * 8 + 8), 3.0, dtype=dtype, device="cuda")[:, :vocab]
    if kind == "words":  # rows on 4 bytes and not on 16
        return torch.full((rows, (vocab + 7) // 8 * 8 + 4), 3.0, dtype=dtype, device="cuda")[:, 2:2 + vocab]
    if kind == "odd":
        return torch.full((rows, vocab + 7 + vocab % 2), 3.0, dtype=dtype, device="cuda")[:, 3:3 + vocab]
    return torch.full((rows, 2 * vocab), 3.0, dtype=dtype, device="cuda")[:, ::2]


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [1003, 1008, 40_001])
@pytest.mark.parametrize("kind", ["even", "words", "odd", "gaps"])
def test_rows_that_share_a_cluster_in_other_layouts(dtype, vocab, kind):
    """Next rows copied while a gradient is written that starts elsewhere than
    the logits do, or over the logits themselves; a temperature for each row."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = 1500 if vocab < 2000 else 700
    logits = layout(rows, vocab, dtype, kind)
    logits.copy_(torch.randn(rows, vocab, device="cuda", generator=g) * 3)
    logits[5::11, ::4] = -math.inf
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    tokens[torch.rand(rows, device="cuda", generator=g) < 0.1] = -1
    columns = [torch.randn(rows, device="cuda", generator=g) for _ in range(4)]
    temperature = 0.5 + torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
    temperature[7::50] = 0.0
    ids = torch.stack([torch.randint(i * vocab // 9, (i + 1) * vocab // 9, (rows,), device="cuda", generator=g) for i in range(9)], 1)
    ids[torch.rand(rows, device="cuda", generator=g) < 0.1] = -1
    values = torch.randn(rows, 9, device="cuda", generator=g)

    def call(which, x, at, grad):
        c, t = [column[at] for column in columns], temperature[at]
        if which == 0:
            return scoring.token_logprobs(x, tokens[at], temperature=t, grad=grad, grad_logprobs=c[0], grad_entropy=c[1])
        if which == 1:
            return scoring.policy_loss(x, tokens[at], c[0], c[1], ref_logprobs=c[2], weights=c[3], kl_coef=0.1,
                                       entropy_coef=0.02, temperature=t, grad=grad)
        return scoring.distill_loss(x, scoring.TopLogits(values[at], ids[at], c[0]), weights=c[3], temperature=t, grad=grad)

    whole = slice(0, rows)
    for which in range(3):
        want = layout(rows, vocab, dtype, "plain")
        pieces = []
        for first in range(0, rows, 40):  # batches whose rows have a cluster each
            at = slice(first, first + 40)
            pieces.append(call(which, logits[at].contiguous(), at, want[at]))
        for grad_kind in ("plain", "even", "words", "odd", "gaps"):
            grad = layout(rows, vocab, dtype, grad_kind)
            out = call(which, logits, whole, grad)
            assert torch.equal(grad, want), grad_kind
            for name in out.__slots__:
                assert torch.equal(getattr(out, name), torch.cat([getattr(o, name) for o in pieces])), name
            if grad_kind != "plain":  # nothing beside the rows is written
                assert int((grad._base == 3).sum()) - int((grad == 3).sum()) == grad._base.numel() - rows * vocab
        over = layout(rows, vocab, dtype, kind)
        over.copy_(logits)
        call(which, over, whole, over)
        assert torch.equal(over, want)
        assert int((over._base == 3).sum()) - int((over == 3).sum()) == over._base.numel() - rows * vocab


# ---------------------------------------------------------------- tracing
def test_compiled_training_step():
    """Traced whole, forward and backward: the same results as in eager mode."""
    _, logits, tokens, columns, teacher = step_inputs()

    def losses(x):
        out = scoring.token_logprobs(x, tokens, temperature=0.8)
        policy = scoring.policy_loss(x, tokens, out.logprobs.detach(), columns[1], entropy_coef=0.1, temperature=0.8)
        distill = scoring.distill_loss(x, teacher, weights=columns[2])
        return out.logprobs.sum() + 0.1 * out.entropy.sum() + policy.loss.sum() + distill.loss.sum(), policy.status

    def with_grad(x, grad):
        top = scoring.top_logits(x, 7)
        out = scoring.policy_loss(x, tokens, columns[0], columns[1], grad=grad)
        return out.loss, out.status, top.values, top.ids, top.rest

    leaf, other = logits.clone().requires_grad_(), logits.clone().requires_grad_()
    want, status = losses(leaf)
    want.backward()
    got, other_status = torch.compile(losses, backend="aot_eager", fullgraph=True)(other)
    got.backward()
    assert torch.equal(status, other_status)
    torch.testing.assert_close(got, want, rtol=1e-6, atol=0)  # (the sum of sums, in another order)
    torch.testing.assert_close(other.grad, leaf.grad, rtol=1e-6, atol=1e-7)  # (three gradients added, likewise)
    grads = [torch.full_like(logits, 5.0) for _ in range(2)]
    eager = with_grad(logits, grads[0])
    traced = torch.compile(with_grad, backend="aot_eager", fullgraph=True)(logits, grads[1])
    assert all(torch.equal(a, b) for a, b in zip(eager, traced)) and torch.equal(*grads)
