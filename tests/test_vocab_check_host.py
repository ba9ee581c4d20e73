"""Token ids outside the embedding's table, what needs no GPU."""
import pytest
import torch

from sdmchat_amd import OneSdmLM, _lib

P = 0x1000   # a pointer that no check reads


def test_a_model_on_the_cpu_raises_at_once():
    m = OneSdmLM(20, d=16, layers=1, mlp_f=16, mem=False, ffn="none", heads=4, n_sub=4, d_a=4, k=2)
    with pytest.raises(IndexError):
        m.enfold(torch.tensor([[1, 20]]))


@pytest.mark.parametrize("over,code", [((P, -1, P, 8, 0, 10, 8, 1.0, P, 8), -1), ((P, 4, None, 8, 0, 10, 8, 1.0, P, 8), -1),
                                       ((P, 4, P, 7, 0, 10, 8, 1.0, P, 8), -1), ((P, 4, P, 8, 0, (1 << 21) + 1, 8, 1.0, P, 8), -3),
                                       ((None, 0, None, 8, 0, 10, 8, 1.0, None, 8), 0)])
def test_checked_lookup_checks_its_arguments(over, code):
    assert _lib.load().sdm_rt_embed_checked(*over, P, None) == code
