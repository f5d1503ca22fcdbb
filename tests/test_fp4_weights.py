"""Matrices in microscaled 4-bit floating point as objects: what copies and row ranges of them share (no GPU needed)."""

import copy
import pickle

import pytest
import torch

from dryft_b200.ops import kernels as K


def held(n, k, kind="nv"):
    size = {"mx": 17408, "nv": 18432}[kind]
    blocks = torch.zeros((n + 127) // 128, (k + 255) // 256, size, dtype=torch.uint8)
    return K.Fp4(blocks, torch.ones(n) if kind == "nv" else None, n, k, kind)


@pytest.mark.parametrize("kind", ["mx", "nv"])
def test_a_copy_is_a_matrix_that_no_product_has_read(kind):
    """Its memory was written later than that of what it was copied from: its first product is one that overlaps nothing."""
    w = held(300, 512, kind)
    w.read.append(True)
    for other in (copy.deepcopy(w), copy.copy(w), pickle.loads(pickle.dumps(w))):
        assert other.read == [] and w.read == [True]
        other.read.append(True)
        assert len(w.read) == 1
        assert (other.shape, other.kind) == (w.shape, kind) and torch.equal(other.held, w.held) and (other.factors is None) == (kind == "mx")


def test_ranges_of_rows_have_it_in_common_whether_a_product_has_read_them():
    """They are one memory, written at once: a first product of any is the first one of all."""
    w = held(400, 300)
    first, rest = w[:128], w[128:]
    assert first.read == [] and rest[128:].read == []
    rest.read.append(True)
    assert w.read == first.read == rest[128:].read == w[256:].read == [True]
    assert copy.deepcopy(rest).read == []
