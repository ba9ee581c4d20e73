"""Limits of the vocabulary's operators that need no GPU to be seen."""
import pytest

from tests.test_vocab_host import _distill, _fails
from sdmchat_amd import _lib


@pytest.mark.parametrize("temperature", [1e-30, 9e-19, 2e18, 3e38])
def test_a_temperature_whose_square_float32_does_not_hold(temperature):
    """Its square would be 0 (no teacher at all) or infinite."""
    lib = _lib.load()
    dims, a, head = _distill(temperature=temperature)
    _fails(lib.sdm_rt_distill_loss(*head, a["loss"], a["stats"], a["dz"], a["dzs"], a["ws"], a["nws"], None), -1, "temperature")
    _fails(lib.sdm_rt_distill_grad(*head, a["stats"], a["go"], 1, a["dz"], a["dzs"], None), -1, "temperature")
