"""tests/test_gpu_encoder_block_calls.py on the CPU build of its kernel files (tests/emul), and what is refused there."""
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emul"))

import test_gpu_encoder_block_calls as T  # noqa: E402
from test_encoder_block_emul_cpu import CPU, refused  # noqa: E402
from test_kernels_emul_cpu import HE, emulated_library  # noqa: E402,F401  (fixtures)

F32, BF16, F16 = T.F32, T.BF16, T.F16


@pytest.mark.parametrize("masked", [None, 2, 6])
def test_emulated_log_sum_exp(HE, masked):
    T.test_log_sum_exp_beside_the_output(HE, CPU, masked, 8, 2, 64, BF16)
    T.test_log_sum_exp_beside_the_output(HE, CPU, masked, 4, 4, 25, F32)


# ------------------------------------------------------------------------------------------------ refusals
def test_residual_norm_refuses_wide_rows_even_where_there_are_none(HE):
    """gradients of weights over 8192 elements, which nothing would have written"""
    x, w = torch.zeros(0, 9000), torch.ones(9000)
    refused(HE, "1 to 8192", HE.residual_norm, x, pre_weight=w)
    refused(HE, "1 to 8192", HE.residual_norm_backward, x, x, x, x, w, w, w, w, w, post_norm=True)
    got = HE.residual_norm_backward(*(torch.zeros(0, 8192) for _ in range(4)), *(torch.ones(8192) for _ in range(5)), post_norm=True)
    assert all(not got[k].any() for k in ("dgate", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias"))
    assert HE.residual_norm(torch.zeros(0, 0))[1].shape == (0, 0)
