"""The row operators on the GPU against their formulas in 64 bits
(tests/scoring_ref.py), at the sizes, types, masks, alignments and bad values
where they can go wrong; the same bits for a row in any batch; streams,
graphs and autograd; and a run of them together around a decode step."""
import math

import numpy as np
import pytest
import torch

from exactsample_b200 import Status, scoring
from tests import scoring_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# One token to several slices: a rank's slice holds 50 KB of a row (16 ranks at most).
VOCABS = [1, 2, 7, 31, 33, 128, 129, 1000, 4099, 19_500, 50_257]


def names(value):
    return str(value).replace("torch.", "")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


def place(x, layout):
    """The CPU rows on the GPU in a memory layout."""
    rows, vocab = x.shape
    if layout == "plain":
        return x.cuda()
    if layout == "odd":  # rows at every alignment: an odd row stride and an odd start
        backing = torch.full((rows, vocab + 7 + (vocab + 7 + 1) % 2), math.nan, dtype=x.dtype, device="cuda")
        view = backing[:, 3:3 + vocab]
    elif layout == "columns":  # no unit stride
        view = torch.empty((vocab, rows), dtype=x.dtype, device="cuda").t()
    elif layout == "gaps":
        view = torch.full((rows, 2 * vocab), math.nan, dtype=x.dtype, device="cuda")[:, ::2]
    view.copy_(x)
    return view


def random_mask(g, rows, vocab, keep=0.5):
    allowed = torch.rand(rows, vocab, generator=g) < keep
    allowed[:, 0] = True
    return allowed


# ---------------------------------------------------------------- token_logprobs
def check_logprobs(x, tokens, temperatures, allowed, out, grad=None, on_lp=None, on_h=None):
    rows, vocab = x.shape
    z = x.double()
    for r in range(rows):
        got = [float(v[r]) for v in (out.logprobs, out.entropy)]
        t, temperature = int(tokens[r]), float(temperatures[r])
        if t < 0:
            assert got == [0, 0] and int(out.status[r]) == 0
            if grad is not None:
                assert bool((grad[r] == 0).all())
            continue
        status = ref.row_status(z[r], allowed[r], temperature)
        if status == Status.OK and t >= vocab:
            status = Status.INVALID_INPUT
        if status == Status.OK and (not allowed[r, t] or z[r, t] == -math.inf):
            status = Status.DRAFT_ZERO_PROB
        assert int(out.status[r]) == int(status), r
        if status != Status.OK:
            assert got == [-math.inf, 0]
            if grad is not None:
                assert bool((grad[r] == 0).all())
            continue
        logp = ref.logp_of(z[r], allowed[r], temperature)
        h = float(ref.entropy_of(logp))
        bounds = ref.RowBounds(logp, vocab)
        # (a log-probability below float32's range is held at its lowest number)
        assert abs(got[0] - max(float(logp[t]), torch.finfo(torch.float32).min)) <= bounds.logprob(logp[t])
        assert abs(got[1] - h) <= bounds.entropy(h)
        if grad is not None:
            a, b = float(on_lp[r]), float(on_h[r])

            def f(v):
                lp = ref.logp_of(v, allowed[r], temperature)
                return a * lp[t] + b * ref.entropy_of(lp)
            leaf = z[r].clone().requires_grad_()
            f(leaf).backward()
            want = torch.where(allowed[r] & (z[r] > -math.inf), leaf.grad, 0.0)
            limit = ref.token_grad_bound(bounds, logp, want, t, a, b, h, temperature, x.dtype)
            off = (grad[r].cpu().double() - want).abs()
            assert bool((off <= limit).all()), (r, float((off / limit).max()))


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("layout", ["plain", "odd", "columns", "gaps"])
def test_token_logprobs(dtype, vocab, layout):
    g = torch.Generator().manual_seed(vocab)
    rows = 5
    x = ref.test_rows(g, rows, vocab, dtype)
    tokens = torch.randint(vocab, (rows,), generator=g)
    tokens[3] = -1
    masked = layout in ("odd", "columns")
    allowed = random_mask(g, rows, vocab) if masked else torch.ones(rows, vocab, dtype=torch.bool)
    temperatures = torch.tensor([1.0, 0.6, 2.5, 1.0, 0.05], dtype=torch.float64)
    on_lp, on_h = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    logits = place(x, layout)
    args = dict(temperature=temperatures.cuda(), mask=ref.pack_mask(allowed).cuda() if masked else None)
    out = scoring.token_logprobs(logits, tokens.cuda(), **args)
    check_logprobs(x, tokens, temperatures, allowed, out)
    # The gradient, into memory of another and of the same layout, and over the logits.
    grads = [place(x, "plain"), place(x, "odd"), logits]
    for grad in grads:
        again = scoring.token_logprobs(logits, tokens.cuda(), grad=grad, grad_logprobs=on_lp.cuda(),
                                       grad_entropy=on_h.cuda(), **args)
        assert torch.equal(again.logprobs, out.logprobs) and torch.equal(again.entropy, out.entropy)
        check_logprobs(x, tokens, temperatures, allowed, again, grad, on_lp, on_h)
        assert torch.equal(grad, grads[0])  # the same bits wherever it lies
    if layout in ("odd", "gaps"):  # what lies between the rows' elements is untouched
        backing = logits._base
        assert int(torch.isnan(backing).sum()) == backing.numel() - rows * vocab


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [40, 1003, 19_500, 50_257])
def test_token_logprobs_of_rows_with_infinities(dtype, vocab):
    """Rows masked by -inf before: a fifth of them, nearly all, only late ones,
    and beside the type's lowest values, with and without an entropy gradient."""
    g = torch.Generator().manual_seed(vocab + 1)
    x = ref.test_rows(g, 9, vocab, dtype)
    few = torch.randperm(vocab, generator=g)[:5]
    lowest = torch.finfo(dtype).min
    x[0, ::5] = -math.inf
    x[1, torch.rand(vocab, generator=g) < 0.9] = -math.inf
    x[2] = -math.inf
    x[2, few] = torch.randn(5, generator=g).to(dtype)
    x[3, vocab // 2:] = -math.inf
    x[4, vocab - 1] = -math.inf
    x[5] = -math.inf
    x[5, few] = lowest                    # all that is left
    x[6, ::3] = -math.inf
    x[6, 1::3] = lowest
    x[7, ::2] = -math.inf
    x[7, 1] = math.nan
    x[8, :vocab // 3] = -math.inf
    tokens = torch.stack([(row > -math.inf).float().argmax() for row in x])
    tokens[5] = few[0]
    tokens[1:3] = torch.stack([row.float().argmax() for row in x[1:3]])
    allowed = torch.ones(x.shape, dtype=torch.bool)
    for temperature in (1.0, 0.3, 1e9):
        temperatures = torch.full((9,), temperature, dtype=torch.float64)
        for with_entropy in (True, False):
            on_lp = torch.randn(9, generator=g)
            on_h = torch.randn(9, generator=g) if with_entropy else torch.zeros(9)
            grad = torch.full_like(x, 3.0, device="cuda")
            out = scoring.token_logprobs(x.cuda(), tokens.cuda(), temperature=temperature, grad=grad, grad_logprobs=on_lp.cuda(),
                                         grad_entropy=on_h.cuda() if with_entropy else None)
            check_logprobs(x, tokens, temperatures, allowed, out, grad, on_lp, on_h)


def test_lowest_values_over_a_small_temperature():
    """A teacher and a student masked by float32's lowest value, which leaves
    the range when divided: the same as masked by -inf."""
    g = torch.Generator(device="cuda").manual_seed(9)
    rows, vocab, k = 4, 900, 16
    lowest = torch.finfo(torch.float32).min
    student = torch.randn(rows, vocab, device="cuda", generator=g)
    hidden = torch.rand(rows, vocab, device="cuda", generator=g) < 0.995
    hidden[:, 3] = False
    teacher = (student + 0.1).masked_fill(hidden, lowest)
    assert bool((hidden.sum(1) > vocab - k).all())  # some of the k are lowest values
    top = scoring.top_logits(teacher, k, temperature=0.25)
    exact = scoring.top_logits(teacher.masked_fill(hidden, -math.inf), k, temperature=0.25)
    kept = exact.ids >= 0
    assert torch.equal(top.values[kept], exact.values[kept]) and bool((top.values[~kept] == lowest).all())
    assert bool((top.rest == lowest).all()) and not bool(top.status.any())
    grads = [torch.empty_like(student) for _ in range(2)]
    for x in (student, student.masked_fill(hidden, lowest)):
        one = scoring.distill_loss(x, top, temperature=0.25, grad=grads[0])
        two = scoring.distill_loss(x, exact, temperature=0.25, grad=grads[1])
        assert not bool(one.status.any()) and not bool(two.status.any())
        torch.testing.assert_close(one.loss, two.loss, rtol=1e-5, atol=1e-6)
        torch.testing.assert_close(grads[0], grads[1], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_token_logprobs_without_an_entropy_gradient(dtype):
    g = torch.Generator().manual_seed(8)
    x = ref.test_rows(g, 4, 777, dtype)
    tokens, on_lp = torch.randint(777, (4,), generator=g), torch.randn(4, generator=g)
    ones, allowed = torch.ones(4), torch.ones(4, 777, dtype=torch.bool)
    grad = torch.empty_like(x, device="cuda")
    out = scoring.token_logprobs(x.cuda(), tokens.cuda(), grad=grad, grad_logprobs=on_lp.cuda())
    check_logprobs(x, tokens, ones, allowed, out, grad, on_lp, torch.zeros(4))
    out = scoring.token_logprobs(x.cuda(), tokens.cuda(), grad=grad, grad_entropy=on_lp.cuda())
    check_logprobs(x, tokens, ones, allowed, out, grad, torch.zeros(4), on_lp)


def hard_rows(dtype, vocab):
    """Rows of bad, empty and extreme values, with their tokens, masks and temperatures."""
    g = torch.Generator().manual_seed(1)
    lowest, highest = torch.finfo(dtype).min, torch.finfo(dtype).max
    base = ref.test_rows(g, 24, vocab, dtype)
    allowed = torch.ones(24, vocab, dtype=torch.bool)
    tokens = torch.randint(vocab, (24,), generator=g)
    temperatures = torch.ones(24, dtype=torch.float64)
    base[0] = -math.inf
    base[1, vocab // 2] = math.nan
    base[2, vocab - 1] = math.inf
    base[3, vocab // 3] = math.nan
    allowed[3, vocab // 3] = False          # a NaN behind the mask
    base[4, vocab // 3] = math.inf
    allowed[4, vocab // 3] = False          # an infinity behind the mask
    allowed[5] = False                      # nothing allowed
    base[6] = lowest                        # a row of the type's lowest value is uniform
    base[7] = lowest
    base[7, 5] = 1.0
    tokens[7] = 5
    base[8] = -math.inf
    base[8, vocab - 1] = 2.0                # one token
    tokens[8] = vocab - 1
    base[9, 0] = highest                    # all of the mass
    tokens[9] = 0
    base[10, int(tokens[10])] = -math.inf   # the token has no mass
    allowed[11, int(tokens[11])] = False    # the token is masked
    tokens[12] = vocab                      # not a token
    tokens[13] = 2**40
    tokens[14] = -2**40                     # no token
    temperatures[15] = 0.0
    temperatures[16] = -1.0
    temperatures[17] = math.nan
    temperatures[18] = math.inf
    temperatures[19] = 1e-45                # the reciprocal is beyond float32
    base[20] = lowest
    allowed[20, ::2] = False
    tokens[20] = 1
    base[21, 1:] = -math.inf
    allowed[21] = False
    allowed[21, 1] = True                   # the one allowed token is -inf
    base[22] = highest                      # uniform at the type's highest
    base[23, ::2] = lowest
    temperatures[23] = 3.0
    tokens[23] = 1
    return base, tokens, temperatures, allowed


def hard_status(base, tokens, temperatures, allowed, r):
    temperature = float(temperatures[r])
    if r == 19:
        return Status.INVALID_INPUT
    return ref.row_status(base[r].double(), allowed[r], temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [40, 1001, 45_000])
def test_token_logprobs_of_hard_rows(dtype, vocab):
    x, tokens, temperatures, allowed = hard_rows(dtype, vocab)
    g = torch.Generator().manual_seed(2)
    on_lp, on_h = torch.randn(24, generator=g), torch.randn(24, generator=g)
    grad = torch.full_like(x, 7.0, device="cuda")
    out = scoring.token_logprobs(x.cuda(), tokens.cuda(), temperature=temperatures.cuda(),
                                 mask=ref.pack_mask(allowed).cuda(), grad=grad, grad_logprobs=on_lp.cuda(),
                                 grad_entropy=on_h.cuda())
    assert int(out.status[19]) == int(Status.INVALID_INPUT) and bool((grad[19] == 0).all())
    keep = torch.tensor([r for r in range(24) if r != 19])
    scoring_out = scoring.TokenLogprobs(out.logprobs[keep.cuda()], out.entropy[keep.cuda()], out.status[keep.cuda()])
    check_logprobs(x[keep], tokens[keep], temperatures[keep], allowed[keep], scoring_out, grad[keep.cuda()],
                   on_lp[keep], on_h[keep])


# ---------------------------------------------------------------- top_logits
def check_top(x, k, temperatures, allowed, out):
    rows, vocab = x.shape
    z = x.double()
    for r in range(rows):
        temperature = float(temperatures[r])
        status = ref.row_status(z[r], allowed[r], temperature)
        assert int(out.status[r]) == int(status), r
        if status != Status.OK:
            assert bool((out.values[r] == -math.inf).all()) and bool((out.ids[r] == -1).all())
            assert float(out.rest[r]) == -math.inf
            continue
        values, ids, rest = ref.top_of(z[r], allowed[r], temperature, k)
        assert out.ids[r].cpu().tolist() == ids.tolist(), r
        assert torch.equal(out.values[r].cpu().double(), values), r
        got = float(out.rest[r])
        if rest == -math.inf:
            assert got == -math.inf
        else:
            others = (z[r] / temperature).masked_fill(~allowed[r], -math.inf)
            others[ids[ids >= 0]] = -math.inf
            bounds = ref.RowBounds(torch.log_softmax(others, 0), vocab)
            assert abs(got - rest) <= bounds.sum + 2.0**-23 * abs(rest), (r, got, rest)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("layout", ["plain", "odd", "gaps"])
def test_top_logits(dtype, vocab, layout):
    g = torch.Generator().manual_seed(vocab)
    rows = 4
    x = ref.test_rows(g, rows, vocab, dtype)
    masked = layout != "plain"
    allowed = random_mask(g, rows, vocab) if masked else torch.ones(rows, vocab, dtype=torch.bool)
    temperatures = torch.tensor([1.0, 0.6, 2.5, 0.05], dtype=torch.float64)
    for k in (1, 5, 64, 256):
        out = scoring.top_logits(place(x, layout), k, temperature=temperatures.cuda(),
                                 mask=ref.pack_mask(allowed).cuda() if masked else None)
        check_top(x, k, temperatures, allowed, out)


def awkward_rows(dtype, vocab):
    """Rows whose largest values tie, cluster in one place, or span the type."""
    g = torch.Generator().manual_seed(4)
    rows = [torch.zeros(vocab), torch.full((vocab,), -3.0), torch.arange(vocab) % 3 * 1.0,
            torch.arange(vocab) * 1.0, -torch.arange(vocab) * 1.0, torch.randint(-2, 3, (vocab,), generator=g) * 1.0]
    rows[0][::2] = -0.0                               # zeros of both signs are equal
    cluster = torch.randn(vocab, generator=g)
    cluster[vocab // 2:vocab // 2 + 300] += 50        # all of the largest side by side
    rows.append(cluster)
    steps = torch.full((vocab,), -5.0)
    steps[::37] = 4.0                                 # more equal leaders than any list
    rows.append(steps)
    few = torch.full((vocab,), -math.inf)
    few[::vocab // 7 + 1] = 1.0                       # fewer tokens than k
    rows.append(few)
    wide = torch.randn(vocab, generator=g).double() * 10
    wide = (wide.sign() * 10.0 ** wide.abs().clamp(max=math.log10(torch.finfo(dtype).max) - 0.1)).float()
    rows.append(wide)
    low = torch.full((vocab,), torch.finfo(dtype).min)
    low[3] = 0.0
    rows.append(low)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [40, 513, 5000, 50_257, 120_000])
def test_top_logits_of_awkward_rows(dtype, vocab):
    x = awkward_rows(dtype, vocab)
    rows = x.shape[0]
    for k in (1, 20, 256):
        out = scoring.top_logits(x.cuda(), k)
        check_top(x, k, torch.ones(rows), torch.ones(rows, vocab, dtype=torch.bool), out)


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_top_logits_of_hard_rows(dtype):
    x, _, temperatures, allowed = hard_rows(dtype, 1001)
    out = scoring.top_logits(x.cuda(), 9, temperature=temperatures.cuda(), mask=ref.pack_mask(allowed).cuda())
    assert int(out.status[19]) == int(Status.INVALID_INPUT)
    keep = torch.tensor([r for r in range(24) if r != 19])
    kept = scoring.TopLogits(*(t[keep.cuda()] for t in (out.values, out.ids, out.rest, out.status)))
    check_top(x[keep], 9, temperatures[keep], allowed[keep], kept)


# ---------------------------------------------------------------- policy_loss
def policy_inputs(g, x, temperatures, allowed):
    rows, vocab = x.shape
    tokens = torch.stack([torch.nonzero(allowed[r])[:, 0][torch.randint(int(allowed[r].sum()), (1,), generator=g)[0]]
                          for r in range(rows)])
    lp = torch.stack([ref.logp_of(x[r].double(), allowed[r], float(temperatures[r]))[tokens[r]] for r in range(rows)])
    ratio = 0.3 * torch.randn(rows, generator=g)
    for border in (math.log(0.8), math.log(1.3)):  # the gradient jumps there: keep clear of rounding
        ratio = torch.where((ratio - border).abs() < 1e-3, ratio + 3e-3, ratio)
    return dict(tokens=tokens, old_logprobs=(lp - ratio).float(), advantages=torch.randn(rows, generator=g),
                ref_logprobs=(lp + 0.4 * torch.randn(rows, generator=g)).float(),
                weights=torch.rand(rows, generator=g) + 0.5)


def check_policy(x, temperatures, allowed, inputs, out, grad, kl_coef, entropy_coef, with_ref, with_weights):
    rows, vocab = x.shape
    for r in range(rows):
        z, temperature, t = x[r].double(), float(temperatures[r]), int(inputs["tokens"][r])
        old, adv = inputs["old_logprobs"][r].double(), inputs["advantages"][r].double()
        ref_lp = inputs["ref_logprobs"][r].double() if with_ref else None
        w = float(inputs["weights"][r]) if with_weights else 1.0
        logp = ref.logp_of(z, allowed[r], temperature)
        h = ref.entropy_of(logp)
        bounds = ref.RowBounds(logp, vocab)
        loss, kl = ref.policy_of(logp[t], h, old, adv, ref_lp, w, 0.2, 0.3, kl_coef, entropy_coef)
        assert int(out.status[r]) == 0
        assert abs(float(out.logprobs[r]) - float(logp[t])) <= bounds.logprob(logp[t])
        assert abs(float(out.entropy[r]) - float(h)) <= bounds.entropy(h)
        # lp is exact to bounds.sum before its own rounding; the loss and the KL term move with it.
        ratio = float((logp[t] - old).exp())
        rise = abs(math.expm1(float(ref_lp - logp[t]))) if with_ref else 0.0
        assert abs(float(out.kl[r]) - float(kl)) <= rise * bounds.sum + bounds.sum**2 + 2.0**-24 * float(kl)
        slope = abs(float(adv)) * ratio + kl_coef * rise
        limit = w * (slope * bounds.sum * 1.01 + kl_coef * bounds.sum**2 + entropy_coef * bounds.entropy(h))
        assert abs(float(out.loss[r]) - float(loss)) <= limit + 2.0**-24 * abs(float(loss))
        if grad is None:
            continue

        def f(v):
            lp = ref.logp_of(v, allowed[r], temperature)
            return ref.policy_of(lp[t], ref.entropy_of(lp), old, adv, ref_lp, w, 0.2, 0.3, kl_coef, entropy_coef)[0]
        leaf = z.clone().requires_grad_()
        f(leaf).backward()
        want = torch.where(allowed[r], leaf.grad, 0.0)
        # The slope itself moves with lp: ratio and the KL term's exponential, relatively by bounds.sum.
        size = w * (slope + kl_coef * (rise + 1) * with_ref)
        limit = ref.token_grad_bound(bounds, logp, want, t, size, w * entropy_coef, float(h), temperature, x.dtype)
        limit[t] += size * bounds.sum / temperature
        off = (grad[r].cpu().double() - want).abs()
        assert bool((off <= limit).all()), (r, float((off / limit).max()))


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [2, 33, 1000, 19_500, 50_257])
@pytest.mark.parametrize("terms", ["plain", "kl", "entropy", "both"])
def test_policy_loss(dtype, vocab, terms):
    g = torch.Generator().manual_seed(vocab)
    rows = 8
    x = ref.test_rows(g, rows, vocab, dtype)
    masked = terms in ("kl", "both")
    allowed = random_mask(g, rows, vocab) if masked else torch.ones(rows, vocab, dtype=torch.bool)
    temperatures = torch.tensor([1.0, 0.6, 2.5, 1.0, 0.5, 1.0, 1.5, 1.0], dtype=torch.float64)
    inputs = policy_inputs(g, x, temperatures, allowed)
    kl_coef = 0.05 if terms in ("kl", "both") else 0.0
    entropy_coef = 0.02 if terms in ("entropy", "both") else 0.0
    with_ref, with_weights = terms != "plain", terms != "entropy"
    args = dict(ref_logprobs=inputs["ref_logprobs"].cuda() if with_ref else None,
                weights=inputs["weights"].cuda() if with_weights else None, temperature=temperatures.cuda(),
                mask=ref.pack_mask(allowed).cuda() if masked else None, clip_low=0.2, clip_high=0.3, kl_coef=kl_coef,
                entropy_coef=entropy_coef)
    given = [inputs[n].cuda() for n in ("tokens", "old_logprobs", "advantages")]
    logits = place(x, "odd" if masked else "plain")
    out = scoring.policy_loss(logits, *given, **args)
    check_policy(x, temperatures, allowed, inputs, out, None, kl_coef, entropy_coef, with_ref, with_weights)
    grad = place(x, "plain")
    step = scoring.policy_loss(logits, *given, grad=grad, **args)
    check_policy(x, temperatures, allowed, inputs, step, grad, kl_coef, entropy_coef, with_ref, with_weights)
    assert all(torch.equal(getattr(out, n), getattr(step, n)) for n in ("loss", "logprobs", "kl", "entropy", "status"))
    # Autograd: the same bits for an incoming gradient of ones.
    leaf = logits.detach().requires_grad_()
    scoring.policy_loss(leaf, *given, **args).loss.sum().backward()
    assert torch.equal(leaf.grad, grad)


def test_policy_loss_of_bad_rows():
    g = torch.Generator().manual_seed(5)
    rows, vocab = 10, 500
    x = ref.test_rows(g, rows, vocab, torch.float32)
    temperatures, allowed = torch.ones(rows, dtype=torch.float64), torch.ones(rows, vocab, dtype=torch.bool)
    inputs = policy_inputs(g, x, temperatures, allowed)
    inputs["old_logprobs"][0] = math.nan
    inputs["advantages"][1] = math.inf
    inputs["ref_logprobs"][2] = -math.inf
    inputs["tokens"][3] = -1
    inputs["old_logprobs"][3] = math.nan          # not read: the row has no token
    inputs["old_logprobs"][4] = -500.0            # the ratio is beyond float32
    inputs["advantages"][4] = -1.0
    inputs["tokens"][5] = vocab
    x[6, 17] = math.nan
    x[7] = -math.inf
    x[8, int(inputs["tokens"][8])] = -math.inf
    grad = torch.full_like(x, 3.0, device="cuda")
    out = scoring.policy_loss(x.cuda(), *(inputs[n].cuda() for n in ("tokens", "old_logprobs", "advantages")),
                              ref_logprobs=inputs["ref_logprobs"].cuda(), kl_coef=0.1, entropy_coef=0.01, grad=grad)
    assert out.status.cpu().tolist() == [2, 2, 2, 0, 2, 2, 2, 1, 3, 0]
    assert out.loss[:9].cpu().tolist() == [0] * 9 and float(out.loss[9]) != 0
    assert out.kl[:9].cpu().tolist() == [0] * 9 and out.entropy[:9].cpu().tolist() == [0] * 9
    assert out.logprobs[:9].cpu().tolist() == [-math.inf] * 3 + [0.0] + [-math.inf] * 5
    assert bool((grad[:9] == 0).all()) and bool((grad[9] != 0).any())


def test_infinite_weights_show_in_the_gradient():
    # An overflowed loss scale must not pass for a gradient of zeros.
    g = torch.Generator().manual_seed(6)
    x = ref.test_rows(g, 3, 300, torch.float32)
    tokens = torch.tensor([1, 2, 3]).cuda()
    weights = torch.tensor([1.0, math.inf, math.nan]).cuda()
    old = torch.full((3,), -5.0).cuda()
    grad = torch.zeros_like(x, device="cuda")
    out = scoring.policy_loss(x.cuda(), tokens, scoring.token_logprobs(x.cuda(), tokens).logprobs, old, weights=weights,
                              grad=grad)
    assert out.status.cpu().tolist() == [0, 0, 0]
    assert bool(torch.isfinite(grad[0]).all()) and not bool(torch.isfinite(grad[1:]).any(1).all())
    teacher = scoring.top_logits(x.cuda() * 1.5, 4)
    scoring.distill_loss(x.cuda(), teacher, weights=weights, grad=grad)
    assert bool(torch.isfinite(grad[0]).all()) and not bool(torch.isfinite(grad[1:]).any(1).all())


# ---------------------------------------------------------------- distill_loss
def check_distill(x, values, ids, rest, weights, temperatures, allowed, out, grad):
    rows, vocab = x.shape
    for r in range(rows):
        z, temperature = x[r].double(), float(temperatures[r])
        v, i, w = values[r].double(), ids[r], float(weights[r])
        rr = None if rest is None else rest[r].double()
        if not bool((i >= 0).any()):
            assert float(out.loss[r]) == 0 and int(out.status[r]) == 0
            assert grad is None or bool((grad[r] == 0).all())
            continue
        logp = ref.logp_of(z, allowed[r], temperature)
        want, lost = ref.distill_of(logp, v, i, rr, temperature)
        assert int(out.status[r]) == (Status.DRAFT_ZERO_PROB if lost else Status.OK), r
        if lost:
            assert float(out.loss[r]) == 0 and (grad is None or bool((grad[r] == 0).all()))
            continue
        # All in 32 bits. The others' sum is off by `error`. The kept tokens'
        # exponentials t and q are off by an expf (2^-23) and two products;
        # sums of them add at most K / 128 + 10 joins (12 here), and shares of
        # the totals a reciprocal and three products: 20 roundings at most,
        # `part`. In the loss, a term t (lt - lq) has the error of t and three
        # roundings of its own, 24 with the sum's joins; the logs of the
        # totals move by the totals' relative errors, and their difference is
        # rounded with what multiplies it.
        others = (z / temperature).masked_fill(~allowed[r], -math.inf)
        others[i[i >= 0]] = -math.inf
        error = ref.RowBounds(torch.log_softmax(others, 0), vocab).sum if bool((others > -math.inf).any()) else 0.0
        part = 20 * 2.0**-24
        kept = i >= 0
        scale = 1 / temperature
        x_kept = (z / temperature).masked_fill(~allowed[r], -math.inf)[i[kept]]
        lt, lq = v[kept] * scale, x_kept
        t = torch.log_softmax(torch.cat([lt, rr[None]]) if rr is not None else lt, 0).exp()
        live = t[:lt.numel()] > 0
        gaps = ((lt - lt.max()) - (lq - lq.max()))[live].abs()
        gap_of_totals = abs(float(torch.logsumexp(lt - lt.max(), 0) - torch.logsumexp(lq - lq.max(), 0)))
        gap_of_totals += abs(float(rr - lt.max())) if rr is not None and float(rr) > -math.inf else 0.0
        limit = 24 * 2.0**-24 * float((t[:lt.numel()][live] * gaps).sum()) + (part + 2.0**-23) * (1 + gap_of_totals) + 2 * part
        limit = w * (limit + 2 * error) + 3 * 2.0**-24 * abs(w * float(want))
        assert abs(float(out.loss[r]) - w * float(want)) <= limit, r
        if grad is None:
            continue
        leaf = z.clone().requires_grad_()
        (w * ref.distill_of(ref.logp_of(leaf, allowed[r], temperature), v, i, rr, temperature)[0]).backward()
        g = torch.where(allowed[r] & (z > -math.inf), leaf.grad, 0.0)
        q = logp.exp()
        pull = torch.ones(())
        if rr is not None:
            q_rest = torch.logsumexp(others, 0) - torch.logsumexp((z / temperature).masked_fill(~allowed[r], -math.inf), 0)
            pull = 1 + (t[-1].log() - q_rest).exp() if q_rest > -math.inf else pull
        d = (others - others.max()).clamp(min=-200).abs() if bool((others > -math.inf).any()) else torch.zeros(vocab)
        # 1 - t_rest / q_rest moves with both logs (part and error each), and
        # the coefficient has six roundings more. A kept token's w (q - t) has
        # both shares' errors and three roundings.
        # (2^-126: exponentials below it are flushed to zero.)
        relative = 2 * error + 2.0**-22 + 3 * 2.0**-24 * d + 2 * part + 6 * 2.0**-24
        size = (q * relative + 2.0**-126) * pull
        size[i[kept]] += t[:lt.numel()] * (part + 3 * 2.0**-24) + 2.0**-126
        limit = w / temperature * size + g.abs() * ref.HALF_STEP[x.dtype] * 1.01 + ref.SMALLEST[x.dtype]
        off = (grad[r].cpu().double() - g).abs()
        assert bool((off <= limit).all()), (r, float((off / limit).max()))


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [2, 33, 1000, 19_500, 50_257])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("layout", ["plain", "odd", "columns"])
def test_distill_loss(dtype, vocab, tail, layout):
    g = torch.Generator().manual_seed(vocab)
    rows = 6
    x = ref.test_rows(g, rows, vocab, dtype)
    teacher = (x.double() + torch.randn(rows, vocab, generator=g)).to(dtype)
    masked = layout != "plain"
    allowed = random_mask(g, rows, vocab) if masked else torch.ones(rows, vocab, dtype=torch.bool)
    mask = ref.pack_mask(allowed).cuda() if masked else None
    temperatures = torch.tensor([1.0, 0.6, 2.5, 1.0, 1.0, 2.0], dtype=torch.float64)
    weights = torch.rand(rows, generator=g) + 0.5
    for k in (1, 20, 256):
        record = scoring.top_logits(teacher.cuda(), k, temperature=temperatures.cuda(), mask=mask)
        record.ids[3] = -1                       # a padded row
        record.ids[4, ::2] = -1                  # unused entries
        if not bool((record.ids[4] >= 0).any()):
            record.ids[4, 0] = 0
        # Unused entries keep their mass out of the teacher: the record is taken as it is.
        args = dict(weights=weights.cuda(), temperature=temperatures.cuda(), mask=mask, tail=tail)
        host = (record.values.cpu(), record.ids.cpu(), record.rest.cpu() if tail else None)
        logits = place(x, layout)
        grads = [place(x, "plain"), logits]
        out = scoring.distill_loss(logits, record, **args)
        check_distill(x, *host, weights, temperatures, allowed, out, None)
        for grad in grads:
            step = scoring.distill_loss(logits, record, grad=grad, **args)
            check_distill(x, *host, weights, temperatures, allowed, step, grad)
            assert torch.equal(step.loss, out.loss) and torch.equal(grad, grads[0])
        leaf = place(x, layout).detach().requires_grad_()
        scoring.distill_loss(leaf, record, **args).loss.sum().backward()
        assert torch.equal(leaf.grad, grads[0])


def test_distill_loss_of_bad_rows():
    g = torch.Generator().manual_seed(9)
    rows, vocab, k = 14, 700, 5
    x = ref.test_rows(g, rows, vocab, torch.float32)
    record = scoring.top_logits(x.cuda() + 0.1, k)
    values, ids, rest = record.values.cpu(), record.ids.cpu(), record.rest.cpu()
    allowed = torch.ones(rows, vocab, dtype=torch.bool)
    ids[0, 4] = ids[0, 1]                         # the same id twice
    ids[1, 0] = vocab                             # not a token
    ids[2, 2] = 2**40
    values[3, 1] = math.nan
    values[4, 1] = math.inf
    rest[5] = math.nan
    rest[6] = math.inf
    values[7] = -math.inf
    rest[7] = -math.inf                           # no mass at all
    x[8, int(ids[8, 0])] = math.nan
    x[9, int(ids[9, 0]) - 1 if int(ids[9, 0]) else 1] = math.inf
    x[10] = -math.inf
    x[11, int(ids[11, 3])] = -math.inf            # no mass where the teacher has some
    allowed[12] = False
    allowed[12, ids[12]] = True                   # nothing outside the kept ids
    values[13, 4] = -math.inf                     # a kept token without mass
    grad = torch.full_like(x, 3.0, device="cuda")
    out = scoring.distill_loss(x.cuda(), scoring.TopLogits(values.cuda(), ids.cuda(), rest.cuda()),
                               mask=ref.pack_mask(allowed).cuda(), grad=grad)
    assert out.status.cpu().tolist() == [2] * 10 + [1, 3, 3, 0]
    assert out.loss[:13].cpu().tolist() == [0] * 13 and bool((grad[:13] == 0).all())
    last = slice(13, 14)
    check_distill(x[last], values[last], ids[last], rest[last], torch.ones(1), torch.ones(1), allowed[last],
                  scoring.DistillLoss(out.loss[last], out.status[last]), grad[last])
    # A teacher renormalised over its kept tokens does not ask for the others.
    out = scoring.distill_loss(x.cuda()[12:13], scoring.TopLogits(values.cuda()[12:13], ids.cuda()[12:13], None),
                               mask=ref.pack_mask(allowed[12:13]).cuda(), tail=False)
    check_distill(x[12:13], values[12:13], ids[12:13], None, torch.ones(1), torch.ones(1), allowed[12:13], out, None)


# ---------------------------------------------------------------- the calls
def all_outputs(logits, tokens, teacher, columns, **common):
    grads = [torch.empty_like(logits) for _ in range(3)]
    one = scoring.token_logprobs(logits, tokens, grad=grads[0], grad_logprobs=columns[0], grad_entropy=columns[1], **common)
    two = scoring.top_logits(logits, 33, **common)
    three = scoring.policy_loss(logits, tokens, columns[0], columns[1], ref_logprobs=columns[2], weights=columns[3],
                                kl_coef=0.1, entropy_coef=0.02, grad=grads[1], **common)
    four = scoring.distill_loss(logits, teacher, weights=columns[3], grad=grads[2], **common)
    return [getattr(o, n) for o in (one, two, three, four) for n in o.__slots__] + grads


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [1003, 151_936])
def test_a_row_has_the_same_bits_in_any_batch(dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = 40
    logits = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype)
    teacher = scoring.top_logits(logits * 0.9, 20)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    columns = [torch.randn(rows, device="cuda", generator=g) * 0.5 - 10 * (i in (0, 2)) for i in range(4)]
    whole = all_outputs(logits, tokens, teacher, columns)
    for first, last in [(0, 1), (17, 18), (39, 40), (5, 12)]:
        at = slice(first, last)
        part = scoring.TopLogits(teacher.values[at], teacher.ids[at], teacher.rest[at])
        moved = place(logits[at].cpu(), "odd")
        for got, want in zip(all_outputs(moved, tokens[at], part, [c[at] for c in columns]), whole):
            assert torch.equal(got, want[at])


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("vocab", [1003, 1008, 13_001, 60_016])
@pytest.mark.parametrize("masked", [False, True], ids=["open", "masked"])
def test_rows_that_share_a_cluster(dtype, vocab, masked):
    """More rows than clusters run at a time, so that rows are copied beside
    the row before: bad, hard and padded ones between others, with and without
    a gradient, against the same rows in small batches."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows, piece = 1400 if vocab < 20_000 else 520, 50
    logits = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype)
    logits[3::7, ::5] = -math.inf   # the careful form
    logits[5::11, 1] = math.nan
    logits[8::13] = -math.inf
    logits[10::17, :900] = -math.inf
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    tokens[torch.rand(rows, device="cuda", generator=g) < 0.3] = -1
    allowed = torch.rand(rows, vocab, device="cuda", generator=g) < 0.5
    allowed[4::9] = False
    mask = ref.pack_mask(allowed.cpu()).cuda() if masked else None
    ids = torch.stack([torch.randint(i * vocab // 9, (i + 1) * vocab // 9, (rows,), device="cuda", generator=g) for i in range(9)], 1)
    ids[torch.rand(rows, device="cuda", generator=g) < 0.3] = -1
    values, rest = torch.randn(rows, 9, device="cuda", generator=g), torch.randn(rows, device="cuda", generator=g)
    columns = [torch.randn(rows, device="cuda", generator=g) for _ in range(4)]

    def calls(at, with_grad):
        x = logits[at]
        common = dict(temperature=0.7, mask=None if mask is None else mask[at])
        grads = [torch.full_like(x, 7.0) if with_grad else None for _ in range(3)]
        c = [column[at] for column in columns]
        incoming = dict(grad_logprobs=c[0], grad_entropy=c[1]) if with_grad else {}
        outs = [scoring.token_logprobs(x, tokens[at], grad=grads[0], **incoming, **common),
                scoring.policy_loss(x, tokens[at], c[0], c[1], ref_logprobs=c[2], weights=c[3], kl_coef=0.1, entropy_coef=0.02,
                                    grad=grads[1], **common),
                scoring.distill_loss(x, scoring.TopLogits(values[at], ids[at], rest[at]), weights=c[3], grad=grads[2], **common)]
        return [getattr(o, n) for o in outs for n in o.__slots__], grads
    whole, whole_grads = calls(slice(0, rows), True)
    forward, _ = calls(slice(0, rows), False)
    for got, want in zip(forward, whole):
        assert torch.equal(got, want)
    for first in range(0, rows, piece):
        at = slice(first, first + piece)
        part, part_grads = calls(at, True)
        for got, want in zip(part + part_grads, whole + whole_grads):
            assert torch.equal(got, want[at])


def test_broadcast_and_strided_columns():
    g = torch.Generator(device="cuda").manual_seed(2)
    rows, vocab = 6, 900
    logits = torch.randn(1, vocab, device="cuda", generator=g).expand(rows, vocab)  # the same row for all
    tokens = torch.randint(vocab, (rows, 2), device="cuda", generator=g)[:, 0]
    temperature = torch.full((1,), 0.8, dtype=torch.float64, device="cuda").expand(rows)
    columns = [(torch.randn(rows, 3, device="cuda", generator=g) * 0.3 - 6)[:, 1] for _ in range(2)]
    columns += [columns[0].contiguous() + 0.2, torch.ones(1, device="cuda").expand(rows)]
    teacher = scoring.top_logits(logits + 0.1, 8, temperature=temperature)
    got = all_outputs(logits, tokens, teacher, columns, temperature=temperature)
    plain = all_outputs(logits.contiguous(), tokens.contiguous(), teacher, [c.contiguous() for c in columns],
                        temperature=temperature.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, plain))
    # Differentiating a broadcast leaf sums over its rows.
    leaf = logits[:1].detach().clone().requires_grad_()
    out = scoring.token_logprobs(leaf.expand(rows, vocab), tokens)
    out.logprobs.sum().backward()
    full = logits.contiguous().requires_grad_()
    scoring.token_logprobs(full, tokens).logprobs.sum().backward()
    torch.testing.assert_close(leaf.grad, full.grad.sum(0, keepdim=True), rtol=0, atol=0)


def test_incoming_gradients_multiply():
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, vocab = 7, 1234
    logits = torch.randn(rows, vocab, device="cuda", generator=g)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    weights = torch.rand(rows, device="cuda", generator=g)
    upstream = torch.randn(rows, device="cuda", generator=g)
    old, adv = torch.full((rows,), -7.0, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    teacher = scoring.top_logits(logits * 1.1, 9)
    for call in (lambda z, **kw: scoring.policy_loss(z, tokens, old, adv, entropy_coef=0.1, **kw),
                 lambda z, **kw: scoring.distill_loss(z, teacher, **kw)):
        leaf = logits.clone().requires_grad_()
        (got,) = torch.autograd.grad(call(leaf, weights=weights).loss, leaf, upstream)
        want = torch.empty_like(logits)
        call(logits, weights=weights * upstream, grad=want)
        assert torch.equal(got, want)
        (got,) = torch.autograd.grad(call(leaf).loss, leaf, upstream)
        call(logits, weights=upstream, grad=want)
        assert torch.equal(got, want)
    # One of the two results alone, and both.
    leaf = logits.clone().requires_grad_()
    out = scoring.token_logprobs(leaf, tokens)
    parts = [torch.autograd.grad(v, leaf, upstream, retain_graph=True)[0] for v in (out.logprobs, out.entropy)]
    for got, kw in zip(parts, (dict(grad_logprobs=upstream), dict(grad_entropy=upstream))):
        want = torch.empty_like(logits)
        scoring.token_logprobs(logits, tokens, grad=want, **kw)
        assert torch.equal(got, want)
    assert not out.status.requires_grad
    with torch.no_grad():
        assert not scoring.token_logprobs(leaf, tokens).logprobs.requires_grad


def test_a_changed_input_is_noticed_by_autograd():
    logits = torch.randn(3, 50, device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    leaf = logits.clone().requires_grad_()
    hidden = leaf * 1.0
    out = scoring.token_logprobs(hidden, tokens)
    scoring.token_logprobs(hidden.detach(), tokens, grad=hidden.detach(), grad_logprobs=torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()


def test_autograd_once_and_no_more():
    g = torch.Generator(device="cuda").manual_seed(31)
    rows, vocab = 6, 700
    logits = torch.randn(rows, vocab, device="cuda", generator=g)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    columns = [torch.randn(rows, device="cuda", generator=g) for _ in range(2)]
    teacher = scoring.top_logits(logits * 0.8, 9)
    calls = [lambda x: scoring.token_logprobs(x, tokens).logprobs, lambda x: scoring.token_logprobs(x, tokens).entropy,
             lambda x: scoring.policy_loss(x, tokens, *columns, entropy_coef=0.1).loss,
             lambda x: scoring.distill_loss(x, teacher, weights=columns[0]).loss]
    for call in calls:
        leaf = logits.clone().requires_grad_()
        out = call(leaf)
        (first,) = torch.autograd.grad(out.sum(), leaf, retain_graph=True)
        (again,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)  # the graph is kept: the same once more
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="differentiable once"):
            again.square().sum().backward()
        call(leaf).sum().backward()
        assert torch.equal(leaf.grad, first)
        call(leaf).sum().backward()  # gradients add up
        assert torch.equal(leaf.grad, first + first)
        out = call(leaf)
        out.sum().backward()
        with pytest.raises(RuntimeError, match="second time"):
            out.sum().backward()
    # Through what broadcasts the logits, and half of the rows through each of two calls.
    leaf = logits[:1].clone().requires_grad_()
    scoring.token_logprobs(leaf.expand(rows, vocab), tokens).logprobs.sum().backward()
    whole = logits[:1].expand(rows, vocab).contiguous().requires_grad_()
    scoring.token_logprobs(whole, tokens).logprobs.sum().backward()
    assert torch.equal(leaf.grad, whole.grad.sum(0, keepdim=True))
    leaf = logits.clone().requires_grad_()
    loss = scoring.token_logprobs(leaf[:2], tokens[:2]).logprobs.sum() + scoring.token_logprobs(leaf[2:], tokens[2:]).logprobs.sum()
    loss.backward()
    whole = logits.clone().requires_grad_()
    scoring.token_logprobs(whole, tokens).logprobs.sum().backward()
    assert torch.equal(leaf.grad, whole.grad)
    status = scoring.token_logprobs(leaf, tokens).status
    assert not status.requires_grad
    with pytest.raises(ValueError, match="need grad"):
        scoring.token_logprobs(leaf, tokens, grad_logprobs=columns[0])
    with pytest.raises(RuntimeError, match="tokens has wrong"):
        scoring.token_logprobs(leaf, tokens.int())
    with torch.no_grad():
        assert not scoring.token_logprobs(leaf, tokens).logprobs.requires_grad
    with torch.inference_mode():
        scoring.policy_loss(leaf, tokens, *columns)


def test_rows_without_any_and_refusals_on_the_device():
    logits = torch.randn(4, 64, device="cuda")
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    empty = scoring.token_logprobs(logits[:0], tokens[:0])
    assert empty.logprobs.shape == (0,)
    assert scoring.top_logits(logits[:0], 5).ids.shape == (0, 5)
    for call, message in [
        (lambda: scoring.token_logprobs(logits.double(), tokens), "float16/bfloat16/float32"),
        (lambda: scoring.token_logprobs(logits, tokens.int()), "tokens has wrong"),
        (lambda: scoring.token_logprobs(logits, tokens.cpu()), "tokens has wrong device"),
        (lambda: scoring.token_logprobs(logits, tokens[:3]), "one value per row"),
        (lambda: scoring.token_logprobs(logits, tokens, temperature=0.0), "temperature must be"),
        (lambda: scoring.token_logprobs(logits, tokens, temperature=torch.ones(4, device="cuda")), "temperature has wrong"),
        (lambda: scoring.token_logprobs(logits, tokens, grad=logits[:, 1:]), "grad shape"),
        (lambda: scoring.token_logprobs(logits, tokens, grad=torch.empty(1, 64, device="cuda").expand(4, 64)), "overlapping"),
        (lambda: scoring.top_logits(logits, 0), "k must be"),
        (lambda: scoring.top_logits(logits, 257), "k must be"),
        (lambda: scoring.policy_loss(logits, tokens, logits[:, 0], logits[:, 1], kl_coef=0.1), "kl_coef needs"),
        (lambda: scoring.distill_loss(logits, scoring.TopLogits(logits[:, :3], tokens, logits[:, 0])), "ids has wrong"),
        (lambda: scoring.token_logprobs(logits[0], tokens), "2D CUDA"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()


def test_two_streams_at_once():
    g = torch.Generator(device="cuda").manual_seed(4)
    sets = []
    for _ in range(4):
        logits = torch.randn(60, 50_257, device="cuda", generator=g)
        tokens = torch.randint(50_257, (60,), device="cuda", generator=g)
        columns = [torch.randn(60, device="cuda", generator=g) - 10 for _ in range(4)]
        sets.append((logits, tokens, scoring.top_logits(logits + 0.1, 20), columns))
    want = [all_outputs(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for stream, s in zip(streams, sets):
        with torch.cuda.stream(stream):
            got.append(all_outputs(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_inputs_freed_while_a_side_stream_reads_them():
    side = torch.cuda.Stream()
    tokens = torch.zeros(64, dtype=torch.int64, device="cuda")
    scoring.token_logprobs(torch.zeros(64, 20_000, device="cuda"), tokens)
    logits = torch.zeros(64, 20_000, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        out = scoring.token_logprobs(logits, tokens)
    del logits
    torch.full((64, 20_000), math.nan, device="cuda")  # would take the freed memory at once
    torch.cuda.synchronize()
    assert out.status.cpu().tolist() == [0] * 64


def test_captured_calls_replay():
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, vocab = 12, 33_000
    logits = torch.randn(rows, vocab, device="cuda", generator=g).to(torch.bfloat16)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    columns = [torch.randn(rows, device="cuda", generator=g) - 10 for _ in range(4)]
    teacher = scoring.top_logits(logits, 20)
    all_outputs(logits, tokens, teacher, columns)
    graphs = []
    for _ in range(2):  # two graphs of the same calls share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = all_outputs(logits, tokens, teacher, columns)
        graphs.append((graph, kept))
    for turn in range(3):
        logits.copy_(torch.randn(rows, vocab, device="cuda", generator=g))
        tokens.copy_(torch.randint(vocab, (rows,), device="cuda", generator=g))
        want = all_outputs(logits, tokens, teacher, columns)
        for graph, kept in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, want)), turn


def test_captured_training_step_through_autograd():
    # Forward and backward in one capture, on leaves that no eager graph holds.
    g = torch.Generator(device="cuda").manual_seed(6)
    rows, vocab = 9, 5000
    weight = torch.randn(vocab, 32, device="cuda", generator=g).mul_(0.1).requires_grad_()
    hidden = torch.randn(rows, 32, device="cuda", generator=g)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    old, adv = torch.full((rows,), -8.0, device="cuda"), torch.randn(rows, device="cuda", generator=g)

    def step():
        out = scoring.policy_loss(hidden @ weight.t(), tokens, old, adv, entropy_coef=0.01)
        return torch.autograd.grad(out.loss.sum(), weight)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    hidden.normal_(generator=g)
    graph.replay()
    torch.cuda.synchronize()
    torch.testing.assert_close(kept, step(), rtol=0, atol=0)


def test_offsets_beyond_32_bits():
    rows, vocab = 14_500, 151_936  # 2.2e9 elements
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    tokens = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    last = torch.randn(3, vocab, device="cuda", generator=g).to(torch.bfloat16)
    logits[-3:] = last
    tokens[-3:] = torch.tensor([5, 70_000, vocab - 1])
    ones = torch.ones(rows, device="cuda")
    out = scoring.token_logprobs(logits, tokens, grad=logits, grad_logprobs=ones)
    grad = torch.empty_like(last)
    want = scoring.token_logprobs(last, tokens[-3:], grad=grad, grad_logprobs=ones[:3])
    assert torch.equal(out.logprobs[-3:], want.logprobs) and torch.equal(logits[-3:], grad)
    assert bool((logits[:-3:101] == 0).all()) and bool((out.status == 0).all())


# ---------------------------------------------------------------- together
def test_a_decode_step_then_training_on_it():
    """Tokens from ``verify``, their log-probabilities and top logits, then a
    policy step on them and a distillation step against them."""
    from exactsample_b200 import bridge
    from exactsample_b200.cuda import CudaRequestParams, CudaRngKey, plan, verify

    g = torch.Generator(device="cuda").manual_seed(8)
    requests, vocab, temperature = 24, 32_000, 0.7
    logits = (torch.randn(requests, vocab, device="cuda", generator=g) * 3).to(torch.bfloat16)
    allowed = torch.rand(requests, vocab, device="cuda", generator=g) < 0.5
    allowed[7] = False  # a request whose grammar allows nothing fails and has no token
    mask = ref.pack_mask(allowed.cpu()).cuda()
    ints = dict(dtype=torch.int64, device="cuda")
    work = plan(requests, requests, 0, vocab)
    sampled = verify(logits, torch.arange(requests + 1, **ints), torch.empty((requests, 0), **ints),
                     params=CudaRequestParams(torch.full((requests,), temperature, dtype=torch.float64, device="cuda"),
                                              torch.zeros(requests, **ints),
                                              torch.ones(requests, dtype=torch.float64, device="cuda"),
                                              torch.zeros(requests, dtype=torch.float64, device="cuda"),
                                              torch.zeros(requests, **ints)),
                     rng=CudaRngKey(torch.arange(requests, **ints), torch.zeros(requests, **ints),
                                    torch.arange(requests, **ints)),
                     plan=work, out=work.allocate_output(), mask=mask)
    tokens = bridge.committed_row_tokens(sampled, torch.arange(requests + 1, **ints), requests)
    assert torch.equal(tokens, sampled.tokens[:, 0])
    common = dict(temperature=temperature, mask=mask)
    old = scoring.token_logprobs(logits, tokens, **common)
    assert int(tokens[7]) == -1 and float(old.logprobs[7]) == 0
    assert bool((old.status == 0).all()) and bool((old.logprobs[:7] < 0).all())
    top = scoring.top_logits(logits, 20, **common)
    assert int(top.status[7]) == int(Status.NO_VALID_TOKEN)
    # The sampled token, where it is among the top, has the record's log-probability.
    total = torch.logaddexp(torch.logsumexp(top.values.double() / temperature, 1), top.rest.double())
    for r, k in (top.ids == tokens[:, None]).nonzero().tolist():
        if r != 7:
            assert abs(float(top.values[r, k]) / temperature - float(total[r]) - float(old.logprobs[r])) < 1e-5
    # The first policy step after sampling: every ratio is 1, the loss is -A.
    adv = torch.randn(requests, device="cuda", generator=g)
    grad = torch.empty_like(logits)
    step = scoring.policy_loss(logits, tokens, old.logprobs, adv, ref_logprobs=old.logprobs, kl_coef=0.1, grad=grad, **common)
    assert torch.equal(step.logprobs, old.logprobs)
    want = torch.where(tokens >= 0, -adv, 0.0)
    # log p was rounded to float32 (half a step, 2^-24 of it), the ratio is an expf (2^-23) and the loss a product.
    torch.testing.assert_close(step.loss, want, rtol=2.0**-24 * float(old.logprobs.abs().max()) + 2.0**-22, atol=0)
    assert bool((grad[7] == 0).all()) and bool((grad[~allowed] == 0).all())
    # A student equal to its teacher: no loss and, but for rounding, no gradient.
    out = scoring.distill_loss(logits, top, grad=grad, **common)
    assert float(out.loss.abs().max()) < 1e-5 and float(grad.float().abs().max()) < 1e-4
