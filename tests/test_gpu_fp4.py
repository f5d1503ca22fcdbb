"""Microscaled 4-bit floating point on the GPU: rounding, values and products against the definition in 64 bits."""

import pytest
import torch

import plain_fp4 as P
from dryft_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
KINDS = ("mx", "nv")


def rows_of(m, k, dtype, wide=0, grow=0.5):
    x = torch.randn(m, k + wide, device="cuda") * torch.exp(grow * torch.randn(1, k + wide, device="cuda"))
    return x.to(dtype)[:, wide // 2:wide // 2 + k]


def odd_rows(k, dtype):
    """Rows with what is rare: nothing but zeros, tiny and large numbers, ties, groups of very different size, infinities and NaN."""
    x = torch.randn(12, k, device="cuda")
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 1e37
    x[3] *= 1e-30
    x[4, ::2] *= 1e-6
    x[5] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 0.3, 7.9], device="cuda").repeat(k // 12 + 1)[:k]
    x[6, k // 2] = float("nan")
    x[7, k - 1] = float("inf")
    x[8, :k // 3] = 0
    x[9] *= torch.exp(8 * torch.randn(k, device="cuda"))
    x[10] = -x[10].abs()
    x[11, 0] = torch.finfo(dtype).max
    return x.to(dtype)


def same_values(got, want, dtype):
    """Equal to the definition's values but for the factor's product (one 32-bit rounding) and the result's own."""
    assert torch.equal(got.isnan().cpu(), want.isnan())
    tiny = 2.0**-149 if dtype == F32 else 2.0**-133       # half a step of the smallest numbers, twice
    room = (torch.finfo(dtype).eps / 2 + 2.0**-24) * want.abs() + tiny
    assert bool(((got.double().cpu() - want).abs() <= room)[~want.isnan()].all())


def near(got, x, w, kind, k):
    """Sums of k terms: the tensor cores take 64 at a time and cut off what is below 2^-23 of the largest, at most, in each of 64 terms and the sum so far (2^-21 of the terms'
    magnitudes, an instruction); the factors' products and the result are rounded."""
    want, terms = P.product(x, w, kind)
    assert torch.equal(got.isnan().cpu(), want.isnan())
    room = (torch.finfo(got.dtype).eps / 2 + 2.0**-22) * want.abs() + (k / 64 + 2) * 2.0**-21 * terms
    off = (got.double().cpu() - want).abs()
    assert bool((off <= room)[~want.isnan()].all()), float((off / room).nan_to_num().max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k,wide", [(1, 16, 0), (1, 1, 0), (3, 17, 0), (130, 256, 0), (5, 2560, 0), (300, 333, 7), (2, 9728, 16), (129, 64, 8), (1, 30000, 2)])
def test_rounding_and_values(kind, dtype, m, k, wide):
    x = rows_of(m, k, dtype, wide)
    q = K.fp4_quantise(x, kind)
    want = P.values(x, kind)
    for out in (BF, F32):
        same_values(K.fp4_expand(q, out_dtype=out), want, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("k", [48, 1000])
def test_rounding_of_rare_rows(kind, dtype, k):
    x = odd_rows(k, dtype)
    same_values(K.fp4_expand(K.fp4_quantise(x, kind), out_dtype=F32), P.values(x, kind), F32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 128, 64), (1, 128, 256), (2, 256, 5120), (16, 300, 4100), (13, 129, 9728), (16, 128, 512), (5, 389, 83), (17, 200, 1000), (33, 130, 300), (100, 256, 2560), (129, 128, 256), (257, 300, 777),
                                   (700, 384, 320), (8, 40000, 320)])
def test_products(kind, m, n, k):
    x, w = rows_of(m, k, BF), rows_of(n, k, BF)
    near(K.linear_fp4(x, K.fp4_quantise(w, kind), out_dtype=F32), x, w, kind, k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,out", [(BF, BF), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("m,n,k", [(1, 129, 1), (3, 50, 31), (20, 260, 2560), (200, 1000, 96)])
def test_products_of_other_types(kind, dtype, out, m, n, k):
    x, w = rows_of(m, k, dtype, 3), rows_of(n, k, dtype)
    near(K.linear_fp4(x, K.fp4_quantise(w, kind), out_dtype=out), x, w, kind, k)
