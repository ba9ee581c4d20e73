"""Limits of the vocabulary's operators that need no GPU to be seen."""
import pytest
import torch

from sdmchat_amd import _lib, core
from tests.test_vocab_host import _distill, _fails


@pytest.mark.parametrize("temperature", [1e-30, 9e-19, 2e18, 3e38])
def test_a_temperature_whose_square_float32_does_not_hold(temperature):
    """Its square would be 0 (no teacher at all) or infinite."""
    lib = _lib.load()
    dims, a, head = _distill(temperature=temperature)
    _fails(lib.sdm_rt_distill_loss(*head, a["loss"], a["stats"], a["dz"], a["dzs"], a["ws"], a["nws"], None), -1, "temperature")
    _fails(lib.sdm_rt_distill_grad(*head, a["stats"], a["go"], 1, a["dz"], a["dzs"], None), -1, "temperature")


def test_apart_goes_by_addresses():
    """Tensors that share memory without sharing a storage object (through dlpack)."""
    buf = torch.zeros(9, 24)

    def shared(t):
        return torch.utils.dlpack.from_dlpack(torch.utils.dlpack.to_dlpack(t))
    for a, b, want in ((buf, shared(buf), True), (buf[:4], shared(buf[1:5]), False), (buf[:4], shared(buf[4:8]), True),
                       (buf[:, :8], shared(buf[:, 8:16]), True), (buf[:, :8], shared(buf[:, 7:15]), False),
                       (buf, torch.zeros(9, 24), True)):
        assert core._apart(a, b) is want and core._apart(b, a) is want
