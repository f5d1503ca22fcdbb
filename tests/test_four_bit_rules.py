"""Rules that choose between forms of the work from 4 bits, on the host (no GPU needed)."""

import importlib

import pytest
import torch

from dryft_b200.ops import kernels as K
from dryft_b200.parts.base import Runtime

L = importlib.import_module("dryft_b200.parts.linear")


def _weight(n, k):
    tiles, wide = -(-n // 16), -(-k // 128) * 128
    return K.Weight4(torch.empty(tiles, wide // 64, 512, dtype=torch.uint8), torch.empty(tiles, wide // 64, 8, 2, 2, dtype=torch.bfloat16), n, k, 64)


@pytest.mark.parametrize("width,most", [(1024, 4), (2048, 4), (2560, 4), (4096, 2), (5120, 2), (8192, 1)])
def test_norms_left_to_products_cost_as_rows_are_wide(monkeypatch, width, most):
    """As many rows as are faster that way at their width; a second product's inputs are not normed."""
    monkeypatch.setattr(L, "fused_rms", lambda norm: norm)
    rt, weights = Runtime(dtype=torch.bfloat16, device=torch.device("cpu")), (_weight(64, width), _weight(width, 9728))
    assert [L.four_bits_fuse(rows, "norm", rt, *weights) for rows in range(1, 8)] == [rows <= most for rows in range(1, 8)]


def test_the_command_lines_numbers_that_share_a_scale(monkeypatch):
    """``--bits-group`` reaches the engine, as its other two options for 4 bits do."""
    from dryft_b200 import cli
    from dryft_b200.engine import api

    class Made(Exception):
        pass

    def made(*a, **kw):
        raise Made(kw)

    monkeypatch.setattr(api, "Engine", made)
    for more, group in (([], 64), (["--bits-group", "128"], 128)):
        with pytest.raises(Made) as e:
            cli.main(["generate", "--model", "somewhere", "--prompt-ids", "1", "--weight-bits", "4"] + more)
        assert e.value.args[0]["bits_group"] == group and e.value.args[0]["weight_bits"] == 4
