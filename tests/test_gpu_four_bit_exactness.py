"""How exact the work from 4 bits is as a whole: bfloat16 attention, where the outputs' own rounding may be the only error that counts, and 32-bit results of products."""

import pytest
import torch

import plain_four_bit as P
from test_gpu_four_bit import Cache, i32
from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _far(c, of, rows, max_kv=None):
    """Off by how much of the whole: the root of the squares' sum over all outputs of all rows."""
    q = torch.randn(len(rows), c.kv * of, c.d).to(BF)
    out = torch.empty(len(rows), c.kv * of * c.d, dtype=BF, device=DEV)
    K().attn4_rows(q.to(DEV), c.k, c.v, c.pt, i32([b for b, _ in rows]), i32([p for _, p in rows]), out, P.scale_of(c.d), None, c.group, max_kv or max(c.lens))
    held = {b: (P.group_values(c.keys[b], c.group)[0], P.group_values(c.values[b], c.group)[0]) for b in {b for b, _ in rows}}
    want = torch.stack([P.attention(q[i].double(), *held[b], p, P.scale_of(c.d))[0].flatten() for i, (b, p) in enumerate(rows)])
    return float((out.double().cpu() - want).norm() / want.norm())


# A rounding to bfloat16 moves a number by up to 2^-8 of it, less towards the next power of two: below 2^-9 in the mean square over many numbers.  Weights have 11 bits (2^-12) and
# sums 32, which together move the whole by less than a hundredth of that.
MOST = 2.0**-9


@pytest.mark.parametrize("lens,kv,of,d,group", [([700] * 40, 2, 4, 128, 64), ([3000] * 2, 8, 4, 128, 64), ([333] * 9, 2, 2, 256, 16), ([500] * 12, 3, 3, 48, 16), ([900] * 12, 4, 4, 64, 64),
                                                ([100] * 30, 2, 2, 32, 32), ([400] * 9, 2, 8, 192, 64)])
@pytest.mark.parametrize("size,uneven", [(1.0, 0.0), (1e-6, 0.0), (1e6, 0.0), (1.0, 2.0), (1e-3, 6.0), (1e12, 0.0), (1e-12, 1.0)])
def test_the_whole_is_off_by_the_results_rounding(lens, kv, of, d, group, size, uneven):
    """Values of any size, and tokens whose values differ in size by orders of magnitude, the largest anywhere among them."""
    c = Cache(lens, kv, d, group)
    for b, n in enumerate(lens):
        c.values[b] = (c.values[b].float() * size * torch.exp(uneven * torch.randn(n, kv, 1))).to(BF)
    c.fill()
    e = _far(c, of, [(b, n - 1) for b, n in enumerate(lens)])
    assert e <= MOST, f"off by {e:.5f} of the whole ({MOST:.5f} allowed)"


def test_long_rows_in_one_split():
    """Nothing accumulates: a warp walks 128 tiles."""
    c = Cache([16383], 7, 128, 64)
    c.fill()
    assert K().attn4_plan(20 * 7, 16383, None, True) == (1, 8, 8, False)
    e = _far(c, 1, [(0, 16382 - i) for i in range(20)])
    assert e <= MOST, f"off by {e:.5f} of the whole ({MOST:.5f} allowed)"


@pytest.mark.parametrize("d,group", [(128, 64), (256, 16), (48, 16)])
def test_values_of_zero_and_of_one_number(d, group):
    """Scales of zero: of all tokens, and of those before the first one that has values of its own; then a token a million times larger than all before it."""
    c = Cache([200] * 3, 1, d, group)
    c.values[0].zero_()
    c.values[1][:] = torch.randn(200, 1, 1).to(BF)
    c.values[2][:150] = 0.5
    c.values[2][190] *= 2.0**20
    c.fill()
    of = {128: 2, 256: 2, 48: 3}[d]
    q = torch.randn(3, of, d).to(BF)
    out = torch.empty(3, of * d, dtype=BF, device=DEV)
    K().attn4_rows(q.to(DEV), c.k, c.v, c.pt, i32(range(3)), i32([199] * 3), out, P.scale_of(d), None, group, 200)
    assert torch.count_nonzero(out[0]) == 0
    for b in (1, 2):
        want = P.attention(q[b].double(), P.group_values(c.keys[b], group)[0], P.group_values(c.values[b], group)[0], 199, P.scale_of(d))[0].flatten()
        assert ((out[b].double().cpu() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-11 * want.abs().max() + 1e-5).all()


@pytest.mark.parametrize("n,k,group", [(6886, 11184, 16), (20000, 5120, 64), (2560, 2560, 128), (19000, 528, 16), (389, 4096, 32), (129, 80, 16)])
@pytest.mark.parametrize("m", [4, 17, 48, 128, 256, 300])
def test_32_bit_results_of_many_inputs(m, n, k, group):
    """Sums of 512 inputs are 64 additions on the tensor cores, which cut off less than 2^-24 of the sum each, half of that in the mean; what is summed in 32 bits from there on
    rounds both ways.  Every row of weights is held against 64 bits over some rows of activations."""
    from dryft_b200.parts.base import Runtime
    from dryft_b200.parts.linear import linear

    w = (torch.randn(n, k, device=DEV) * torch.exp(0.3 * torch.randn(n, 1, device=DEV))).to(BF)
    x = (torch.randn(m, k, device=DEV) * torch.exp(0.5 * torch.randn(1, k, device=DEV))).to(BF)
    w4, values = K().pack_weight4(w, group), torch.empty(n, k, device=DEV)
    K().weight4_expand(w4, values)           # (held against 64 bits elsewhere)
    y = linear(x, w4, Runtime(dtype=BF, device=torch.device(DEV)), out_dtype=torch.float32)
    K().check_error_flags()
    for rows in (slice(0, 8), slice(max(0, m - 8), m)):
        want = x[rows].double() @ values.double().T
        e = float((y[rows].double() - want).norm() / want.norm())
        assert e <= 64 * 2.0**-25, f"off by {e:.3g} of the whole ({64 * 2.0**-25:.3g} allowed)"
