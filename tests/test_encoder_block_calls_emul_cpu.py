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
