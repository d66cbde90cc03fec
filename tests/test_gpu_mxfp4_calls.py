"""Calls of the MXFP4 experts whose sizes or arguments meet an edge of a kernel or of an
entry point: rows that fill only some lanes of the combine."""
import numpy as np
import pytest

import mxfp4 as M
from test_gpu_mxfp4_experts import BF16, F32, check, cuda, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("H,k,Is", [(32, 64, 32), (64, 10, 0), (64, 33, 64), (544, 64, 32), (1056, 24, 0)])
def test_more_entries_than_lanes_with_outputs(H, k, Is, act):
    """the combine's lanes hold a token's entries also where they hold none of its outputs:
    rows of 32 and 64, and rows whose last segment is 32 wide"""
    E, I = 80, 32
    rows, vals = M.block(H + k, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, act)
    for T in (2, 5, 9, 40):
        print("case", H, k, act, T, flush=True)
        x, idx, w, sw = inputs(T, T, H, E, k, act)
        check(blk.experts(cuda(x, act), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None), x, idx, w, vals,
              sw if Is else None, act)
    blk.close()
