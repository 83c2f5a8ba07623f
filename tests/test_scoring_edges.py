"""Refusals of the row operators without a GPU, beside those of test_scoring.py."""
import ctypes

import numpy as np
import pytest
import torch

from exactsample_b200 import capi, scoring
from tests.test_scoring import OPERATORS, arguments, call

OPTIONAL = {"es_token_logprobs": ("grad", "grad_logprobs", "grad_entropy"), "es_top_logits": (),
            "es_policy_loss": ("ref_logprobs", "weights", "grad"), "es_distill_loss": ("rest", "weights", "grad")}


@pytest.mark.parametrize("name,field", [(n, f) for n in OPERATORS for f in
                                        ["mask", "temperature", *(f for f, kind in capi.ROW_OPERATORS[n]._fields_[1:]
                                                                  if kind is capi.Tensor)]])
def test_every_tensor_is_aligned_to_its_elements(name, field):
    """A pointer between two elements would be a misaligned access on the GPU."""
    for shift in (1, 2, 3):
        a = arguments(name, optional=("mask", "temperature", *OPTIONAL[name]))
        assert call(name, a)[0] == -7  # as it is, it gets to the device check
        tensor = getattr(a.rows if field in ("mask", "temperature") else a, field)
        tensor.data += shift
        assert call(name, a) == (-3, f"{field} must be aligned to its elements"), shift


def test_forward_derivatives_are_refused():
    """None of the operators has one: a tangent of zeros would pass for it.
    (The check comes before the device's, so that it needs no GPU.)"""
    import torch.autograd.forward_ad as forward

    x, tokens, column = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    teacher = scoring.TopLogits(torch.zeros(3, 2), torch.arange(6).view(3, 2), column)
    calls = [lambda z: scoring.token_logprobs(z, tokens).logprobs, lambda z: scoring.top_logits(z, 2).values,
             lambda z: scoring.policy_loss(z, tokens, column, column).loss, lambda z: scoring.distill_loss(z, teacher).loss]
    for call_of in calls:
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(call_of, (x,), (torch.ones_like(x),))
        for tracked in (False, True):
            with forward.dual_level():
                dual = forward.make_dual(x.clone().requires_grad_(tracked), torch.ones_like(x))
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call_of(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call_of(dual)
    with forward.dual_level():  # of an input beside the logits
        weights = forward.make_dual(torch.ones(3), torch.ones(3))
        for z in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                scoring.policy_loss(z, tokens, column, column, weights=weights)


def test_a_teachers_statuses_are_checked():
    lib = capi.load()

    def with_status(a, status):
        code = lib.es_distill_loss_status(ctypes.byref(a), None if status is None else ctypes.byref(status), None)
        return code, lib.es_last_error().decode()
    a = arguments("es_distill_loss")
    good = a._host.t((3,), np.int32, capi.ES_I32)
    assert with_status(a, good)[0] == with_status(a, None)[0] == with_status(a, capi.Tensor())[0] == -7
    assert with_status(a, a._host.t((3,), np.int64, capi.ES_I64)) == (-1, "teacher_status has wrong device, dtype or rank")
    assert with_status(a, a._host.t((2,), np.int32, capi.ES_I32)) == (-1, "teacher_status must have one value per row")
    between = capi.Tensor.from_buffer_copy(good)
    between.data += 2
    assert with_status(a, between) == (-3, "teacher_status must be aligned to its elements")
    assert with_status(a, a.status) == (-4, "exactsample input/output aliasing is forbidden")
    assert lib.es_distill_loss_status(None, None, None) == -1
    empty = arguments("es_distill_loss", rows=0)
    assert with_status(empty, empty._host.t((0,), np.int32, capi.ES_I32)) == (0, "")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_shapes_and_types_without_memory(dtype):
    """What a tracer asks for: results of tensors without memory, forward and backward."""
    rows, vocab, k = 3, 40, 4
    x = torch.empty(rows, vocab, dtype=dtype, device="meta")
    tokens = torch.empty(rows, dtype=torch.int64, device="meta")
    column = torch.empty(rows, device="meta")
    teacher = scoring.top_logits(x, k)
    calls = [lambda z, **kw: scoring.token_logprobs(z, tokens, **kw),
             lambda z, **kw: scoring.policy_loss(z, tokens, column, column, weights=column, **kw),
             lambda z, **kw: scoring.distill_loss(z, teacher, weights=column, **kw)]
    outs = [call_of(x) for call_of in calls] + [call_of(x, grad=torch.empty_like(x)) for call_of in calls]
    for out in outs + [teacher]:
        for name in out.__slots__:
            kind = {"status": torch.int32, "ids": torch.int64}.get(name, torch.float32)
            value = getattr(out, name)
            assert value.dtype == kind and not value.requires_grad
            assert value.shape == ((rows, k) if name in ("values", "ids") else (rows,))
    for call_of in calls:
        leaf = x.clone().requires_grad_()
        out = call_of(leaf)
        sum(getattr(out, name).sum() for name in out.__slots__ if getattr(out, name).requires_grad).backward()
        assert leaf.grad.shape == x.shape and leaf.grad.dtype == dtype and not out.status.requires_grad
    with pytest.raises(RuntimeError, match="float16/bfloat16/float32"):
        scoring.token_logprobs(x.double(), tokens)
    with pytest.raises(RuntimeError, match="k must be"):
        scoring.top_logits(x, 257)


def test_a_training_step_is_traced():
    """Into one graph: each operator, and its gradient's call in the backward pass."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, tokens, column):
        leaf = x.detach().requires_grad_()
        loss = scoring.policy_loss(leaf, tokens, column, column).loss.sum()
        loss = loss + scoring.token_logprobs(leaf, tokens).logprobs.sum()
        loss = loss + scoring.distill_loss(leaf, scoring.top_logits(x, 5)).loss.sum()
        return torch.autograd.grad(loss, leaf)
    with FakeTensorMode():
        inputs = (torch.empty(3, 8, device="meta"), torch.empty(3, dtype=torch.int64, device="meta"),
                  torch.empty(3, device="meta"))
        nodes = [str(node.target) for node in make_fx(step)(*inputs).graph.nodes]
    counts = {name: sum(f"exactsample.{name}.default" == node for node in nodes)
              for name in ("token_logprobs", "policy_loss", "distill_loss", "top_logits")}
    assert counts == dict(token_logprobs=2, policy_loss=2, distill_loss=2, top_logits=1)
