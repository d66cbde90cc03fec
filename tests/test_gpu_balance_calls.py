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


@pytest.mark.parametrize("T,E,bf", [(8192, 16, False), (8192, 64, True), (3000, 5, False), (700, 128, True)])
def test_workgroups_have_rows(T, E, bf):
    """a workgroup leaves a row of E + 1 sums; where a row of logits takes few lanes, its 8 waves take
    8 (64 / lanes) rows at a time, and there are no more workgroups than that needs"""
    import helexa_amd as hx
    import torch
    x, idx = B.inputs(T, T, E, 3)
    t, i = cuda(x, bf), cuda(idx)
    want = hx.balance_loss(t, i)
    ws = torch.full((hx.balance_workspace_size(T, E),), 0x5a, dtype=torch.uint8, device="cuda")
    out = hx.balance_loss(t, i, workspace=ws)
    assert all(torch.equal(out[n], want[n]) for n in want)
    per = 8 if bf else 4
    chunks, lanes = E // per if E % per == 0 else E, 64
    while lanes > 1 and lanes // 2 >= chunks:
        lanes //= 2
    groups = -(-T // (8 * (64 // lanes)))
    most = 4 * (E + 1) * (groups + -(-T // 1024)) + 512   # and a row of counts for each 1024 tokens; the tables' starts
    assert int((ws.view(torch.int32) != 0x5a5a5a5a).sum()) * 4 <= most
