"""Microscaled 4-bit floating point on the GPU at the edges of what its calls allow."""

import pytest
import torch

import plain_fp4 as P
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


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [16, 100, 300])
def test_stages_that_end_anywhere_in_a_ring(monkeypatch, kind, m):
    """Fewer inputs than a ring of stages holds, as many, and more; one tile and several to a block."""
    n = 700
    for k in (100, 600, 1100, 1300, 1700, 2100, 2900):
        x, w = rows_of(m, k, BF), rows_of(n, k, BF)
        q, h = K.fp4_quantise(w, kind), K.fp4_quantise(x, kind)
        want, terms = P.product(x, w, kind)
        room = (k / 64 + 10) * 2.0**-21 * terms + 2.0**-22 * want.abs()
        plans = [(next(b for b in (16, 32, 64, 128) if m <= b or b == 128), blocks, 1) for blocks in (1, 2, 5)]
        plans += [(nb, blocks, 0) for nb in (128, 192, 256) for blocks in (2, 4) if m > 16]
        for plan in plans:
            monkeypatch.setattr(K, "linear_fp4_plan", lambda *a: plan)
            for operand in (h, x):
                y = K.linear_fp4(operand, q, out_dtype=F32)
                assert bool(((y.double().cpu() - want).abs() <= room).all()), (k, plan)
    K.check_error_flags()
