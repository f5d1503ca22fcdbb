"""Activations that are infinite, not a number, or so large that parts of a product leave 32 bits: products with 4-bit weights give what their definition
gives, whichever kernel the number of rows chooses."""

import pytest
import torch

import plain_four_bit as P
from test_gpu_four_bit import _weights
from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def _inputs(m, n, k, dtype):
    """Weights whose rows have either sign at every input, a row of zeros, a group of zeros and one of NaN; of up to eight kinds of rows of activations as many as fit: a positive and a
    negative infinity, two of the same and of opposite signs, a NaN, a number whose product with 31 (a code's largest 16 + c) leaves 32 bits,
    one in the middle and one in the last input."""
    w, x = _weights(n, k, BF), torch.randn(m, k).to(dtype)
    w[1], w[2, :16] = 0.0, 0.0
    w[n - 1, 16] = float("nan")
    kinds = [{5: INF}, {k - 1: -INF}, {0: INF, 16: INF}, {3: INF, k - 2: -INF}, {7: float("nan")}, {k // 2: 2e37}, {0: -INF}, {k - 1: -2e37}]
    odd = [(i * 5) % m for i in range(min(m, 8))] if m % 5 else list(range(min(m, 8)))
    for row, kind in zip(odd, kinds):
        for at, v in kind.items():
            x[row, at] = v
    return w, x


def _check(got, x, values):
    """Infinities and NaN are those of the sum over the inputs in 64 bits; where it is finite, weights and result may each be rounded to bfloat16 (2^-8), and 32-bit sums are
    off by less than that again."""
    terms = x.double()[:, None] * values[None]
    want, slack = terms.sum(-1).to(F32).double(), 3 * 2.0**-8 * terms.abs().sum(-1)
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    whole = want.isfinite()
    assert torch.equal(got[~whole & ~want.isnan()], want[~whole & ~want.isnan()])
    assert ((got - want).abs()[whole] <= slack[whole]).all()


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("n,k,group", [(40, 80, 16), (37, 128, 64), (250, 1280, 128), (48, 9728, 32)])
@pytest.mark.parametrize("m", [1, 2, 5, 8, 9, 16])
def test_few_rows(m, n, k, group, out):
    w, x = _inputs(m, n, k, BF)
    w4 = K().pack_weight4(w.to(DEV), group)
    for row in range(min(m, 4)):        # every kind alone, too
        _check(K().linear4(x[row:row + 1].to(DEV), w4, out_dtype=out), x[row:row + 1], P.group_values(w, group)[0])
    _check(K().linear4(x.to(DEV), w4, out_dtype=out), x, P.group_values(w, group)[0])


@pytest.mark.parametrize("m", [1, 5, 16])
def test_few_rows_with_a_sum_or_activation_behind(m):
    n, k, group = 96, 256, 64
    w, x = _inputs(m, n, k, BF)
    w4, xd, y0 = K().pack_weight4(w.to(DEV), group), x.to(DEV), torch.randn(m, n, device=DEV).to(BF)
    plain = K().linear4(xd, w4)
    assert not plain.isfinite().all()
    total, act, want = y0.clone(), torch.empty(m, n // 2, dtype=BF, device=DEV), torch.empty(m, n // 2, dtype=BF, device=DEV)
    K().linear4(xd, w4, total, mode="residual")
    assert torch.equal(total.nan_to_num(nan=7.0), (y0.float() + plain.float()).to(BF).nan_to_num(nan=7.0)) and torch.equal(total.isnan(), plain.isnan())
    K().linear4(xd, w4, act, mode="silu")
    K().silu_mul(plain, want)
    assert torch.equal(act.isnan(), want.isnan()) and torch.equal(act.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("n,k,group", [(40, 80, 16), (37, 128, 64), (250, 1280, 128), (129, 2432, 32)])
@pytest.mark.parametrize("m", [17, 48, 130, 256])
def test_weights_taken_out_tile_by_tile(m, n, k, group, out):
    w, x = _inputs(m, n, k, BF)
    values = P.group_values(w, group)[0]
    y = K().linear4(x.to(DEV), K().pack_weight4(w.to(DEV), group), out_dtype=out)
    K().check_error_flags()
    for i in range(0, m, 16):
        _check(y[i:i + 16], x[i:i + 16], values)


@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("n", [40, 37])
def test_many_rows(n, dtype, out):
    from dryft_b200.parts.base import Runtime
    from dryft_b200.parts.linear import linear

    w, x = _inputs(300, n, 320, dtype)
    y = linear(x.to(DEV), K().pack_weight4(w.to(DEV), 64), Runtime(dtype=dtype, device=torch.device(DEV)), out_dtype=out)
    _check(y, x, P.group_values(w, 64)[0])


@pytest.mark.parametrize("m,n", [(16, 5000), (256, 20000)])
def test_every_result_not_finite(m, n):
    """All of a launch's results are worked out again: slowly, and no bounded wait runs out over it."""
    w4 = K().pack_weight4(torch.rand(n, 2560, device=DEV).to(BF) + 0.5)
    y = K().linear4(torch.full((m, 2560), INF, dtype=BF, device=DEV), w4, out_dtype=F32)
    K().check_error_flags()
    assert (y == INF).all()
