"""Calls of the operators that serve from 4 bits that would give wrong numbers or touch memory where they may not are refused by name before anything is
launched (no GPU needed)."""

import pytest
import torch

from dryft_b200.ops import kernels as K

BF, F32 = torch.bfloat16, torch.float32


def test_a_sum_into_nothing():
    """``out += x @ w.T`` needs an ``out``."""
    w4 = K.pack_weight4(torch.randn(48, 64))
    with pytest.raises(K.KernelError, match="no out was given"):
        K.linear4(torch.zeros(1, 64, dtype=BF), w4, mode="residual")
