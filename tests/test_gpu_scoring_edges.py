"""The row operators on the GPU where a factor leaves float32's range though
the result does not."""
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
