"""Refusals of the row operators without a GPU, beside those of test_scoring.py."""
import pytest

from exactsample_b200 import capi
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
