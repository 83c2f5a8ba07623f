"""The row operators without a GPU: the C ABI's refusals, the Python API's,
and the 64-bit formulas that the GPU tests compare with (their gradients
against finite differences)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from exactsample_b200 import capi, scoring
from tests import scoring_ref as ref
from tests.test_abi import Host

F32, I32, I64, F64 = capi.ES_F32, capi.ES_I32, capi.ES_I64, capi.ES_F64


def arguments(name, rows=3, vocab=40, k=4, optional=(), **override):
    """Valid arguments over host buffers (never dereferenced by the checks)."""
    h = Host()
    a = capi.ROW_OPERATORS[name]()
    a.rows.logits = h.t((rows, vocab), np.float32, F32)
    a.rows.temperature_all = 1.0
    if "mask" in optional:
        a.rows.mask = h.t((rows, (vocab + 31) // 32), np.int32, I32)
    if "temperature" in optional:
        a.rows.temperature = h.t((rows,), np.float64, F64)
    needed = {"es_token_logprobs": ["tokens", "logprobs", "entropy", "status"],
              "es_top_logits": ["values", "ids", "rest", "status"],
              "es_policy_loss": ["tokens", "old_logprobs", "advantages", "loss", "logprobs", "kl", "entropy", "status"],
              "es_distill_loss": ["values", "ids", "loss", "status"]}[name]
    for field in [*needed, *(f for f in optional if f not in ("mask", "temperature"))]:
        if field == "grad":
            value = h.t((rows, vocab), np.float32, F32)
        elif field in ("values", "ids"):
            value = h.t((rows, k), *((np.float32, F32) if field == "values" else (np.int64, I64)))
        else:
            kind = {"tokens": (np.int64, I64), "status": (np.int32, I32)}.get(field, (np.float32, F32))
            value = h.t((rows,), *kind)
        setattr(a, field, value)
    for field, value in override.items():
        setattr(a, field, value(h, a) if callable(value) else value)
    a._host = h
    return a


def call(name, a):
    lib = capi.load()
    code = getattr(lib, name)(ctypes.byref(a), None)
    return code, lib.es_last_error().decode()


OPERATORS = sorted(capi.ROW_OPERATORS)


@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("optional", [(), ("mask", "temperature")])
def test_valid_arguments_reach_the_device_check(name, optional):
    code, message = call(name, arguments(name, optional=optional))
    assert code == -7 and ("GPU" in message or "device" in message)


@pytest.mark.parametrize("name", [n for n in OPERATORS if n != "es_top_logits"])
def test_gradient_may_be_the_logits_and_nothing_else(name):
    assert call(name, arguments(name, optional=("grad",)))[0] == -7

    def over(h, a):
        return a.rows.logits
    assert call(name, arguments(name, grad=over))[0] == -7

    def shifted(h, a):
        t = capi.Tensor.from_buffer_copy(a.rows.logits)
        t.data += 4
        return t
    assert call(name, arguments(name, grad=shifted)) == (-4, "exactsample input/output aliasing is forbidden")

    def transposed(h, a):
        t = capi.Tensor.from_buffer_copy(a.rows.logits)
        t.stride[0], t.stride[1] = 1, t.size[0]
        return t
    assert call(name, arguments(name, grad=transposed))[0] == -4

    def other_type(h, a):
        return h.t((3, 40), np.float16, capi.ES_F16)
    assert call(name, arguments(name, grad=other_type)) == (-1, "grad has wrong device, dtype or rank")

    def narrow(h, a):
        return h.t((3, 39), np.float32, F32)
    assert call(name, arguments(name, grad=narrow)) == (-1, "grad shape mismatch")


@pytest.mark.parametrize("name", OPERATORS)
def test_logits_are_checked(name):
    for make, code, message in [
        (lambda h: h.t((3,), np.float32, F32), -1, "logits must be a 2D CUDA tensor"),
        (lambda h: h.t((3, 40), np.float64, F64), -1, "row operators require float16/bfloat16/float32 logits"),
        (lambda h: h.t((3, 0), np.float32, F32), -1, "at least one column"),
    ]:
        a = arguments(name)
        a.rows.logits = make(a._host)
        got, text = call(name, a)
        assert got == code and message in text
    a = arguments(name)
    a.rows.logits.stride[1] = -1
    assert call(name, a) == (-1, "logits has a negative stride")
    a = arguments(name)
    a.rows.logits.data += 2
    assert call(name, a) == (-3, "logits must be aligned to their elements")
    a = arguments(name)
    a.rows.logits.stride[0] = 1 << 46
    assert call(name, a) == (-1, "logits exceeds the kernels' index range")


@pytest.mark.parametrize("name", OPERATORS)
def test_masks_and_temperatures_are_checked(name):
    a = arguments(name)
    a.rows.mask = a._host.t((3, 1), np.int32, I32)
    assert call(name, a) == (-1, "mask shape mismatch")
    a = arguments(name)
    a.rows.mask = a._host.t((3, 2), np.int64, I64)
    assert call(name, a) == (-1, "mask has wrong device, dtype or rank")
    a = arguments(name)
    a.rows.temperature = a._host.t((3,), np.float32, F32)
    assert call(name, a) == (-1, "temperature has wrong device, dtype or rank")
    a = arguments(name)
    a.rows.temperature = a._host.t((2,), np.float64, F64)
    assert call(name, a) == (-1, "temperature must have one value per row")
    for bad in (0.0, -1.0, math.inf, math.nan):
        a = arguments(name)
        a.rows.temperature_all = bad
        assert call(name, a) == (-1, "temperature must be positive and finite")


@pytest.mark.parametrize("name,field", [(n, f) for n in OPERATORS for f in
                                        (f for f, kind in capi.ROW_OPERATORS[n]._fields_[1:] if kind is capi.Tensor)])
def test_every_tensor_is_checked(name, field):
    def wrong(h, a):
        return h.t((3,), np.uint8, capi.ES_U8)
    optional = ("grad",) if field in ("grad_logprobs", "grad_entropy") else ()
    code, message = call(name, arguments(name, optional=optional, **{field: wrong}))
    assert code == -1 and message == f"{field} has wrong device, dtype or rank"


def test_numbers_are_checked():
    for override, message in [(dict(clip_low=-0.1), "clip_low"), (dict(clip_low=1.5), "clip_low"),
                              (dict(clip_high=-1.0), "clip_low"), (dict(clip_high=math.inf), "clip_low"),
                              (dict(kl_coef=math.nan), "finite"), (dict(entropy_coef=math.inf), "finite"),
                              (dict(kl_coef=0.1), "kl_coef needs ref_logprobs")]:
        code, text = call("es_policy_loss", arguments("es_policy_loss", **override))
        assert code == -1 and message in text
    for name in ("es_top_logits", "es_distill_loss"):
        for k in (0, capi.MAX_TOP + 1):
            assert call(name, arguments(name, k=k)) == (-1, "k must be in [1, 256]")
    assert call("es_token_logprobs", arguments("es_token_logprobs", optional=("grad_logprobs",))) == \
        (-1, "grad_logprobs and grad_entropy need grad")


def test_outputs_may_not_overlap():
    a = arguments("es_token_logprobs")
    a.entropy = a.logprobs
    assert call("es_token_logprobs", a) == (-4, "exactsample outputs alias")
    a = arguments("es_policy_loss")
    a.loss = a.advantages
    assert call("es_policy_loss", a) == (-4, "exactsample input/output aliasing is forbidden")
    a = arguments("es_top_logits")
    a.values.stride[0] = 0
    assert call("es_top_logits", a) == (-4, "output has overlapping strides")


def test_vocabularies_beyond_a_cluster_are_refused():
    for name in OPERATORS:
        a = arguments(name)
        a.rows.logits.data = 1 << 44
        a.rows.logits.size[1] = 4_000_000
        a.rows.logits.stride[0] = 4_000_000
        code, text = call(name, a)
        assert code == -5 and "vocabulary too large" in text


@pytest.mark.parametrize("name", OPERATORS)
def test_no_rows_is_no_work(name):
    assert call(name, arguments(name, rows=0)) == (0, "")


def test_null_arguments():
    lib = capi.load()
    for name in OPERATORS:
        assert getattr(lib, name)(None, None) == -1
        assert lib.es_last_error().decode() == "null arguments"


def test_python_refusals():
    logits = torch.zeros(2, 8, requires_grad=True)
    tokens = torch.zeros(2, dtype=torch.int64)
    column = torch.zeros(2)
    with pytest.raises(ValueError, match="grad= takes the gradient"):
        scoring.token_logprobs(logits, tokens, grad=torch.zeros(2, 8))
    with pytest.raises(ValueError, match="by the logits only"):
        scoring.policy_loss(logits, tokens, column.clone().requires_grad_(), column)
    with pytest.raises(ValueError, match="tail=True needs"):
        scoring.distill_loss(logits, scoring.TopLogits(column, tokens, None))


def test_committed_row_tokens():
    from exactsample_b200 import bridge
    from exactsample_b200.cuda import CudaOutput

    tokens = torch.tensor([[5, 6, 7], [8, -1, -1], [9, 10, -1], [1, 2, 3]])
    out = CudaOutput(tokens, torch.tensor([2, 0, 1, 0], dtype=torch.int32), torch.tensor([0, 0, 0, 2], dtype=torch.int32),
                     torch.zeros(4, dtype=torch.int32), 4)
    cu_rows = torch.tensor([0, 3, 5, 8, 9])  # request 2 accepted one of two drafts, request 3 failed
    for offsets in (cu_rows, cu_rows.int()):
        assert bridge.committed_row_tokens(out, offsets, 9).tolist() == [5, 6, 7, 8, -1, 9, 10, -1, -1]
        # Logits padded to more rows than the requests have, fewer rows, none, and no requests.
        assert bridge.committed_row_tokens(out, offsets, 16).tolist() == [5, 6, 7, 8, -1, 9, 10, -1, -1] + [-1] * 7
        assert bridge.committed_row_tokens(out, offsets, 4).tolist() == [5, 6, 7, 8]
        assert bridge.committed_row_tokens(out, offsets, 0).tolist() == []
        assert bridge.committed_row_tokens(out, offsets[:1], 3).tolist() == [-1, -1, -1]
    # A request with no rows between others.
    gap = CudaOutput(out.tokens[:3], out.accepted_len[:3], out.status[:3], out.path_used[:3], 3)
    assert bridge.committed_row_tokens(gap, torch.tensor([0, 3, 3, 6]), 6).tolist() == [5, 6, 7, 9, 10, -1]


# ---------------------------------------------------------------- the formulas
def differences(f, z, step=1e-6):
    grad = torch.zeros_like(z)
    for i in range(z.numel()):
        up, down = z.clone(), z.clone()
        up[i] += step
        down[i] -= step
        grad[i] = (f(up) - f(down)) / (2 * step)
    return grad


def by_autograd(f, z):
    z = z.clone().requires_grad_()
    f(z).backward()
    return z.grad


@pytest.mark.parametrize("temperature", [1.0, 0.6])
@pytest.mark.parametrize("old_gap,adv", [(0.1, 1.0), (0.1, -1.0), (0.5, 1.0), (0.5, -1.0), (-0.5, 1.0), (-0.5, -1.0)])
def test_reference_gradients_match_differences(temperature, old_gap, adv):
    g = torch.Generator().manual_seed(3)
    z = torch.randn(12, generator=g, dtype=torch.float64)
    allowed = torch.ones(12, dtype=torch.bool)
    allowed[3] = False
    lp0 = ref.logp_of(z, allowed, temperature)[5]

    def policy(x):
        logp = ref.logp_of(x, allowed, temperature)
        return ref.policy_of(logp[5], ref.entropy_of(logp), lp0 - old_gap, torch.tensor(adv).double(), lp0 + 0.3, 0.7,
                             0.2, 0.3, 0.05, 0.01)[0]

    values, ids, rest = ref.top_of(z + 0.3 * torch.randn(12, generator=g, dtype=torch.float64), allowed, temperature, 4)
    for f in (policy,
              lambda x: ref.distill_of(ref.logp_of(x, allowed, temperature), values, ids, torch.tensor(rest), temperature)[0],
              lambda x: ref.distill_of(ref.logp_of(x, allowed, temperature), values, ids, None, temperature)[0]):
        # Central differences: rounding 2^-52 |f| / step = 4e-10 and step^2 times a third derivative.
        torch.testing.assert_close(by_autograd(f, z), differences(f, z), rtol=0, atol=1e-8)
