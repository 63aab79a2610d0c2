"""Bounds of the arguments of include/edsl_hip_lm.h, decided on the host before any
device is looked at."""
import pytest

from mlir_edsl_hip import last_plan
from test_lm_refusals import call, message


@pytest.mark.parametrize("op", ["token_logprobs", "token_logprobs_backward"])
def test_scale(op):
    """scale log2(e) has to be a finite 32-bit number: the logits' maximum times it is 0 or the row's largest value."""
    for scale in (2.4e38, 3.4e38, 2.0 ** 127 * (1 + 2.0 ** -23)):
        assert call(op, dict(scale=scale)) != 0
        assert "2^127" in message()
    assert call(op, dict(scale=2.0 ** 127, M=0)) == 0
    assert last_plan() == "empty"
