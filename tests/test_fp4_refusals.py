"""What the operators of microscaled 4-bit floating point do not take is refused by name before anything is compiled or launched (no GPU needed); and the definition that their
tests go by."""

import pytest
import torch

import plain_fp4 as P
from dryft_b200.ops import kernels as K
from dryft_b200.parts.base import Runtime
from dryft_b200.parts.linear import linear

BF, F32 = torch.bfloat16, torch.float32


def held(n, k, kind="nv"):
    size = {"mx": 17408, "nv": 18432}[kind]
    blocks = torch.zeros((n + 127) // 128, (k + 255) // 256, size, dtype=torch.uint8)
    return K.Fp4(blocks, torch.ones(n) if kind == "nv" else None, n, k, kind)


def refused(word, call):
    with pytest.raises(K.KernelError) as e:
        call()
    assert word in str(e.value), str(e.value)


def test_kinds():
    for kind in ("mxfp4", "", None, 1, ["nv"]):
        refused("mx, nv", lambda: K.fp4_quantise(torch.zeros(2, 32), kind))


def test_numbers_that_are_not_rows():
    for x in (torch.zeros(32), torch.zeros(2, 3, 4)):
        refused("rows", lambda: K.fp4_quantise(x, "mx"))
    refused("behind one another", lambda: K.fp4_quantise(torch.zeros(32, 4).t(), "mx"))
    refused("float32 or bfloat16", lambda: K.fp4_quantise(torch.zeros(2, 32, dtype=torch.float16), "mx"))
    refused("tensor", lambda: K.fp4_quantise([[1.0]], "mx"))
    refused("fewer than", lambda: K.fp4_quantise(torch.zeros(1).expand(2**31, 1), "mx"))


def test_tensors_on_the_cpu():
    w, x = held(16, 64), torch.zeros(1, 64)
    for call in (lambda: K.fp4_quantise(x, "nv"), lambda: K.fp4_expand(w), lambda: K.linear_fp4(x, w), lambda: K.linear_fp4(held(3, 64), w),
                 lambda: linear(x, w, Runtime(dtype=F32, device=torch.device("cpu")))):
        refused("CUDA", call)


def test_held_forms_that_are_not_what_they_say():
    good = held(130, 300)
    for h, f, n, k, kind in [(good.held[:1], good.factors, 130, 300, "nv"), (good.held, good.factors, 300, 300, "nv"), (good.held, good.factors, 130, 600, "nv"),
                             (good.held, None, 130, 300, "nv"), (good.held, good.factors[:129], 130, 300, "nv"), (good.held, good.factors, 130, 300, "mx"),
                             (good.held, good.factors.double(), 130, 300, "nv"), (good.held.to(torch.int32), good.factors, 130, 300, "nv"),
                             (good.held, good.factors, 0, 300, "nv"), (good.held, good.factors, 130, 300, "xx"), (good.held.transpose(0, 1), good.factors, 130, 300, "nv")]:
        with pytest.raises(K.KernelError):
            K.Fp4(h, f, n, k, kind)


def test_row_ranges_start_at_blocks():
    w = held(400, 300)
    assert w[128:300].shape == (172, 300) and w[:400].shape == (400, 300) and w[256:].shape == (144, 300) and w[128:].factors.shape == (272,)
    assert held(400, 300, "mx")[128:].factors is None
    for at in (slice(1, 200), slice(128, 128), slice(0, 400, 2), 3, slice(400, 500)):
        refused("Fp4", lambda: w[at])
    assert w.nbytes() == 4 * 2 * 18432 + 1600 and w.dtype == torch.uint8


def test_definition():
    """The plain form's own numbers, by hand."""
    x = torch.zeros(1, 40)
    x[0, :8] = torch.tensor([6.0, 5.0, 3.5, 2.5, 1.75, 0.75, 0.25, -0.3])
    x[0, 32] = 7.9
    got = P.values(x, "mx")[0]
    assert got[:8].tolist() == [6.0, 4.0, 4.0, 2.0, 2.0, 1.0, 0.0, -0.5] and got[32] == 6.0 and got[33] == 0.0   # 7.9: above 6 where the scale is 1
    row = torch.tensor([[2688.0] * 16 + [6.0] * 16])
    got = P.values(row, "nv")[0]
    assert torch.equal(got, row[0].double())                       # factor 1, scales 448 and 1
    assert P.values(torch.tensor([[1.0, float("inf")] + [2.0] * 15]), "nv")[0].isnan().tolist() == [True] * 16 + [False]
    assert len(P.E4M3) == 127 and P.E4M3[-1] == 448.0 and P.E4M3[1] == 2.0**-9
