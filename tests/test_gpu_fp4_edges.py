"""Microscaled 4-bit floating point on the GPU at the edges of what its calls allow."""

import pytest
import torch

from dryft_b200.ops import kernels as K
from test_gpu_fp4 import near, rows_of

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
KINDS = ("mx", "nv")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [2, 40])
def test_gates_whose_exponential_is_nearly_too_large(kind, m):
    """1 + exp(-g) between 2^126 and the largest 32-bit number: silu(g) is a bfloat16 number like any other, and counts where what it is multiplied by is large.  Two roundings to
    bfloat16 (2^-8 each, at most), an exponential of 2 + 1.173 |g| ulp at most (106: 2^-16.2) and a division of two."""
    k, n = 256, 200
    gate = torch.arange(-88.5, -85.75, 0.5, device="cuda").repeat(m * k)[:m * k].view(m, k)
    up = torch.randn(m, k, device="cuda") * 2.0**118
    x = torch.cat([gate, up], 1).to(BF)
    assert float(x[:, :k].float().min()) == -88.5
    want = (x[:, :k].double() * torch.sigmoid(x[:, :k].double()) * x[:, k:].double())
    act = torch.empty(m, k, dtype=BF, device="cuda")
    K.silu_mul(x, act)
    assert bool(((act.double() - want).abs() <= (2 * 2.0**-8 + 2.0**-15) * want.abs()).all())
    w = rows_of(n, k, BF)
    q = K.fp4_quantise(w, kind)
    got = K.linear_fp4(x, q, silu=True)
    assert torch.equal(got, K.linear_fp4(act, q))
    near(got, act, w, kind, k)
    # rows of an odd width, which silu_mul takes number by number: at most two of them have a neighbour's code somewhere (as in the test of silu in front)
    odd = torch.cat([x[:, :k - 1], x[:, k:2 * k - 1]], 1)
    act = torch.empty(m, k - 1, dtype=BF, device="cuda")
    K.silu_mul(odd, act)
    q = K.fp4_quantise(w[:, :k - 1], kind)
    got, want = K.linear_fp4(odd, q, silu=True), K.linear_fp4(act, q)
    assert int((got != want).any(1).sum()) <= 2 and bool(((got.float() - want.float()).norm(dim=1) <= 0.5 * want.float().norm(dim=1)).all())
