"""How products in microscaled 4-bit floating point are cut into tiles, blocks and clusters: every plan of the rule is one that the launcher takes and covers the result (no GPU needed)."""

import random

import pytest

from dryft_b200.ops import kernels as K

CLUSTERS = (0, 0, 148, 90, 66, 52, 44, 30, 30)   # as a B200 answers


def tiles_of(m, n, nb, split):
    return -(-n // 256) * -(-m // nb) if split == 0 else -(-n // 128) * -(-m // nb)


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("sms,clusters", [(148, CLUSTERS), (16, (0, 0, 8, 4, 2, 2, 2, 0, 0)), (1, (0,) * 9)])
def test_every_plan_is_one_that_the_launcher_takes(seed, sms, clusters):
    rng = random.Random(seed)
    for _ in range(400):
        m, n, k = (int(round(2 ** rng.uniform(0, top))) for top in (13, 18, 15))
        nb, blocks, split = K._fp4_plan(m, n, k, max(sms, 2), clusters)
        units, tiles = (k + 255) // 256, tiles_of(m, n, nb, split)
        if split == 0:
            assert nb in (128, 192, 256) and 0 < blocks <= 2 * tiles and blocks % 2 == 0
        else:
            assert nb in (16, 32, 64, 128) and (m <= nb or nb == 128) and 1 <= split <= min(8, units)
            assert blocks == tiles * split if split > 1 else 0 < blocks <= tiles
            assert split == 1 or tiles <= clusters[split]   # all at once
        for kind in K.FP4_KINDS:
            if K._fp4_fused(m, k, kind, nb, split) or K._fp4_fused(m, k, kind, nb, split, True, True):
                assert m <= 16 and nb == 16 and split >= 1 and -(-units // split) <= 12


def test_blocks_that_a_tile_reads_are_there():
    """The index arithmetic of both kernels, block by block: nothing outside of what fp4_quantise allocates is read, and every result is somebody's once."""
    for m in [1, 2, 15, 16, 17, 31, 64, 100, 127, 128, 129, 160, 191, 192, 193, 255, 256, 257, 300, 383, 384, 385, 500, 777, 1000]:
        for n in [1, 127, 128, 129, 255, 256, 257, 389, 512, 1000]:
            x_blocks, w_blocks = -(-m // 128), -(-n // 128)
            for nb in (16, 32, 64, 128):
                if m > nb and nb < 128:
                    continue
                x_tiles = -(-m // nb)
                for t in range(w_blocks * x_tiles):
                    assert t // x_tiles < w_blocks and t % x_tiles < x_blocks
            for nb in (128, 192, 256):
                w_tiles, whole = -(-w_blocks // 2), m // nb
                seen = set()
                for t in range(w_tiles * -(-m // nb)):
                    last = t >= w_tiles * whole
                    w = (t - w_tiles * whole if last else t // whole) * 2
                    x0 = (whole if last else t % whole) * nb
                    cols = (m - x0 + 31) // 32 * 32 if last else nb
                    assert 32 <= cols <= nb and (w, x0) not in seen and w < w_blocks and x0 % 64 == 0
                    seen.add((w, x0))
                    off, block = x0 % 128, x0 // 128
                    assert off + cols <= 256 and block < x_blocks
                    if off + cols > 128:
                        assert block + 1 < x_blocks
                    for rank in (0, 1):
                        begin = off + rank * (cols // 2)
                        end = begin + cols // 2
                        head = (min(end, 128) - begin) if begin < 128 else 0
                        tail = (end - max(begin, 128)) if end > 128 else 0
                        assert head + tail == cols // 2 and head % 8 == 0 and tail % 8 == 0 and begin % 8 == 0
                        assert tail == 0 or off + cols > 128
                assert seen == {(2 * w, x) for w in range(w_tiles) for x in range(0, m, nb)}
