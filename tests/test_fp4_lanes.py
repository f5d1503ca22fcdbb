"""How many lanes round a row to microscaled 4-bit floating point: a rule on sizes and on the device's multiprocessors (no GPU needed)."""

import pytest

from dryft_b200.ops import kernels as K


@pytest.mark.parametrize("multiprocessors", [16, 74, 148, 160])
@pytest.mark.parametrize("is_bf16,kind,silu", [(1, 0, 0), (1, 0, 1), (1, 1, 0), (1, 1, 1), (0, 0, 0), (0, 1, 0)])
def test_lanes_of_a_row(multiprocessors, is_bf16, kind, silu):
    lanes = lambda words, rows, k: K.fp4_lib().dryft_fp4_lanes(is_bf16, kind, silu, words, rows, k, multiprocessors)  # noqa: E731
    wide = 25600
    # a row that has a multiprocessor to itself has up to 1,024 lanes, more rows 256, or 512 where their numbers would be worked out or read twice
    assert lanes(1, multiprocessors, 16 * 4 * 1024) == 1024
    assert lanes(1, multiprocessors + 1, wide) == (512 if kind == 1 and (silu or not is_bf16) else 256)
    for rows in (1, multiprocessors, multiprocessors + 1, 512, 513, 100000):
        for k in (1, 16, 256, 257, 512, 2560, 9728, wide, 10**6):
            for words in (0, 1):
                n = lanes(words, rows, k)
                assert n in (32, 64, 128, 256, 512, 1024) and (words or n <= 256)
                assert n <= 2 * max(16, -(-k // 256) * 16)   # no more than twice what has something to do
