"""Calls of the encoder block's operators that their documentation allows and tests/test_gpu_encoder_block.py does not make: outputs beside the main ones, graphs and optimizers in
states that a program reaches, inputs at the ends of their ranges.  Bounds: tests/encoder_block_reference.py."""
import math

import pytest
import torch

import encoder_block_reference as R
import test_gpu_encoder_block as T
from test_gpu_encoder_block import G, H, dev  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
F32, BF16, F16 = T.F32, T.BF16, T.F16


# ------------------------------------------------------------------------------------------------ neighbour attention
@pytest.mark.parametrize("heads,kv,dim,kind", [(4, 4, 25, F32), (8, 2, 64, BF16), (1, 1, 1, F16)])
@pytest.mark.parametrize("masked", [None, 2, 6])
def test_log_sum_exp_beside_the_output(H, dev, masked, heads, kv, dim, kind):
    """the log-sum-exp of every list: the sum of its two statistics, rounded once; -inf where nothing is live; short lists, none, one that is cut and joined.  The other
    results are those of the call without it."""
    index, offsets = T.lists(6, 30, [5, 0, 400, 30, 1, 2], 3)
    bias = None if masked is None else T.relation_bias(heads, 7, masked)(index.numel()).to(dev)
    q, k, v = T.rows_of(6, heads, dim, kind, dev, 1), T.rows_of(30, kv, dim, kind, dev, 2), T.rows_of(30, kv, dim, kind, dev, 3)
    plan = H.NeighborPlan(index.to(dev), offsets.to(dev), 30)
    out, stats, lse = H.neighbor_attention(q, k, v, plan, None, bias, return_lse=True)
    assert lse.shape == (6, heads) and lse.dtype == F32 and torch.equal(lse, stats[..., 0] + stats[..., 1])
    assert all(torch.equal(a, b) for a, b in zip((out, stats), H.neighbor_attention(q, k, v, plan, None, bias)))
    rows, owner = R.lists_of(index, offsets, 6)
    value, mag = R.attention(q, k, v, rows, owner, dim ** -0.5, None if bias is None else bias.cpu())["stats"]
    R.close(lse, value.sum(-1), mag.sum(-1), 1, "lse")
    assert bool((lse[1] == -math.inf).all()) and (masked != 6 or bool((lse == -math.inf).all()))
