"""The balance loss at the edges of what its calls allow."""
import numpy as np
import pytest

import balance as B

pytestmark = pytest.mark.gpu


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("E", [1, 512, 852, 853, 1000, 1024])
def test_no_tokens(E, bf):
    """on either side of where one workgroup's tables fit"""
    import helexa_amd as hx
    x, idx = B.inputs(1, 0, E, 1)
    for counts in (None, cuda(np.arange(E, dtype=np.int32))):
        out = hx.balance_loss(cuda(x, bf), cuda(idx), counts=counts)
        assert float(out["loss"]) == 0.0 and out["dlogits"].shape == (0, E)
        assert out["probs"].shape == (E,) and not out["probs"].any() and not out["counts"].any()
    assert not hx.expert_counts(cuda(idx), E).any()
