"""Matrices in microscaled 4-bit floating point as objects: what copies and row ranges of them share, and the order of the options beside them (no GPU needed)."""

import copy
import dataclasses
import pickle

import pytest
import torch

from dryft_b200.engine.api import EngineOptions
from dryft_b200.ops import kernels as K
from dryft_b200.parts.base import Runtime


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


def test_options_keep_their_places():
    """A program that gives options by place goes on meaning what it meant: what came later stands behind."""
    assert [f.name for f in dataclasses.fields(EngineOptions)][:19] == ["dtype", "max_batch", "max_seq_len", "max_tokens", "page_size", "cuda_graphs", "device", "small_m_max", "stream_m_max", "fuse_decode", "pdl",
                                         "norm_ahead", "weight_bits", "cache_bits", "bits_group", "tcgen05", "branch_rows", "prefill_chunk_tokens", "weight_format"]
    assert [f.name for f in dataclasses.fields(Runtime)][:17] == ["dtype", "device", "page_size", "sm_count", "small_m_max", "stream_m_max", "ffn_chunk_rows", "fuse_decode", "pdl", "norm_ahead", "tcgen05", "weight_bits",
                              "cache_bits", "bits_group", "branch_rows", "side_streams", "weight_format"]
