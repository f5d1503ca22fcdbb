"""Attention over the 4-bit cache against 64 bits in every way that its keys are cut over blocks: each case says which way it is meant to take."""

import pytest
import torch

from test_gpu_four_bit import Cache, _attend
from test_gpu_kernels import K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _plan(rows, kv, of, keys, window=None, dtype=BF):
    return K().attn4_plan(rows * kv * ((of + 7) // 8), keys, window, dtype == BF)


@pytest.mark.parametrize("page", [16, 64])
def test_more_blocks_than_multiprocessors_in_one_split(page):
    lens = [700, 1, 16, 333, 64] * 8
    c = Cache(lens, 8, 128, 64, page)
    c.fill()
    assert _plan(40, 8, 1, 700) == (1, 1, 4, False)
    _attend(c, 8, [(b, n - 1) for b, n in enumerate(lens)], None)


@pytest.mark.parametrize("kv,of,d,group", [(1, 2, 64, 64), (2, 4, 128, 64), (1, 2, 256, 16), (1, 1, 16, 16), (1, 9, 80, 16)])
@pytest.mark.parametrize("window", [None, 2500])
def test_more_blocks_than_multiprocessors_in_joined_splits(kv, of, d, group, window):
    """Rows with keys in the first split alone, in all of them, at the edges of splits; padding between them."""
    lens = [1, 17, 1024, 1025, 2049, 3000, 5000]
    c = Cache(lens, kv, d, group)
    c.fill()
    rows = [(-1, 9)] + [(b, n - 1 - i) for i in range(26) for b, n in enumerate(lens) if n > 7 * i] + [(-1, 0)] + [(6, 1023 + i) for i in range(4)] + [(6, 2047), (6, 2048), (6, 3071), (6, 4095)]
    rows += [(6, 40 * i) for i in range(160 - len(rows))]
    splits, least, warps, cluster = _plan(len(rows), kv, of, 5000, window)
    assert splits == (5 if window is None else 3) and (least, warps, cluster) == (64, 4, False)
    _attend(c, kv * of, rows, window)


@pytest.mark.parametrize("kv,of,d,group", [(1, 2, 256, 16), (1, 16, 256, 128), (1, 8, 192, 64), (2, 2, 256, 16), (1, 8, 128, 64)])
def test_few_rows_in_clusters_of_every_size(kv, of, d, group):
    """Heads above 128, whose blocks take most of a multiprocessor's shared memory each, in clusters of two to sixteen; rows that leave most of their cluster without keys."""
    lens = [4300, 3, 600]
    c = Cache(lens, kv, d, group)
    c.fill()
    for splits, keys in ((16, 4300), (7, 1800), (2, 600)):
        assert _plan(1, kv, of, keys) == (splits, 8, 8, True)
        _attend(c, kv * of, [(0, keys - 1)], None, max_kv=keys)
    assert _plan(3, kv, of, 4300)[3]
    _attend(c, kv * of, [(0, 4299), (1, 2), (2, 599)], None)
    _attend(c, kv * of, [(2, 599), (0, 4000), (-1, 5)], 1500, max_kv=4300)


@pytest.mark.parametrize("kv,of,d,group", [(2, 2, 64, 64), (1, 2, 256, 16)])
def test_splits_in_32_bits(kv, of, d, group):
    lens = [4300, 3, 600]
    c = Cache(lens, kv, d, group, 64, F32)
    c.fill()
    assert _plan(3, kv, of, 4300, dtype=F32)[0] > 8
    _attend(c, kv * of, [(0, 4299), (1, 2), (2, 599)], None)
