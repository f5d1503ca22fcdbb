"""Calls that the operators from 4 bits take as their 16-bit forms do."""

import importlib

import pytest
import torch

import plain_four_bit as P
from test_gpu_four_bit import Cache, _near, _weights, i32
from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("m", [1, 64, 65, 200])
@pytest.mark.parametrize("n", [40, 250])
def test_32_bit_activations_and_a_result_of_16(m, n, monkeypatch):
    """The 32-bit product, rounded once; weights taken out whole and in parts."""
    L = importlib.import_module("dryft_b200.parts.linear")
    from dryft_b200.parts.base import Runtime

    w, x = _weights(n, 320, F32), torch.randn(m, 320)
    w4, rt = K().pack_weight4(w.to(DEV), 64), Runtime(dtype=F32, device=torch.device(DEV))
    for size in (L.EXPAND_BYTES, 64 * 320 * 4):
        monkeypatch.setattr(L, "EXPAND_BYTES", size)
        got, whole = L.linear(x.to(DEV), w4, rt, out_dtype=BF), L.linear(x.to(DEV), w4, rt)
        values, s, _ = P.group_values(w, 64)
        assert got.dtype == BF and torch.equal(got, whole.to(BF))
        _near(whole, P.linear(x, values), P.linear_slack(x, values, s, 64, F32))


@pytest.mark.parametrize("n", [1, 5])
def test_one_tensor_as_keys_and_values(n):
    """Rows that lie apart, the same for both."""
    c = Cache([n], 2, 64, 64)
    rows = torch.randn(n, 5 * 64).to(BF)
    c.keys[0] = c.values[0] = rows[:, 64:3 * 64].reshape(n, 2, 64)
    c.fill()
    want = c.k.clone(), c.v.clone()
    c.k.fill_(255), c.v.fill_(255)
    both = rows.to(DEV)[:, 64:3 * 64].view(n, 2, 64)
    K().kv4_store(both, both, i32([0] * n), i32(range(n)), c.k, c.v, c.pt, 64)
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
