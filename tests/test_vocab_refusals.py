"""Calls at a language model's two ends that have to be refused: outputs in the place of an input that is not the logits."""
import pytest

from katsu_b200 import cabi
from test_adjust_logits import BASE as LOGITS
from test_adjust_logits import NAMES as LOGITS_NAMES
from test_block_norm import anywhere  # noqa: F401 (fixture)
from test_distill import BASE as DISTILL
from test_distill import NAMES as DISTILL_NAMES


@pytest.mark.parametrize("other", ["teacher", "index", "labels", "weight", "g"])
def test_a_loss_in_place_of_its_logits_and_of_another_input(anywhere, other):  # noqa: F811
    """The gradient may be written where the logits are; a list, a label or a weight that is there too would be overwritten under way."""
    args = {**DISTILL, "dlogits": DISTILL["logits"], other: DISTILL["logits"]}
    lib = cabi.load()
    assert lib.katsu_cuda_distill_bwd(anywhere, *(args[n] for n in DISTILL_NAMES)) == cabi.ERR_INVALID_ARG
    assert "overlaps" in lib.katsu_cuda_last_error_string().decode()


@pytest.mark.parametrize("other", ["history", "prompts", "lengths", "repetition", "presence", "frequency", "bias_tokens", "bias", "allowed"])
def test_logits_adjusted_in_place_and_in_that_of_another_input(anywhere, other):  # noqa: F811
    args = {**LOGITS, "out": LOGITS["logits"], other: LOGITS["logits"]}
    lib = cabi.load()
    assert lib.katsu_cuda_adjust_logits(anywhere, *(args[n] for n in LOGITS_NAMES)) == cabi.ERR_INVALID_ARG
    assert "overlaps" in lib.katsu_cuda_last_error_string().decode()
