"""What the operators that serve from 4 bits do not take is refused by name before anything is compiled or launched (no GPU needed), and the layout of
weights in 4 bits."""

import pytest
import torch

import plain_four_bit as P
from dryft_b200.cache.slots import CacheError
from dryft_b200.cache.store import KVNeed, SequenceCache
from dryft_b200.ops import kernels as K

BF = torch.bfloat16


@pytest.mark.parametrize("k,group", [(64, 48), (64, 8), (80, 32), (64, 256), (0, 16)])
def test_groups_of_weights(k, group):
    with pytest.raises(K.KernelError) as e:
        K.pack_weight4(torch.zeros(4, k), group)
    assert str(group) in str(e.value)


def test_weights_of_other_types_and_shapes():
    for w in (torch.zeros(4, 64, dtype=torch.float16), torch.zeros(4, 64, 1), torch.zeros(0, 64)):
        with pytest.raises(K.KernelError):
            K.pack_weight4(w)
    with pytest.raises(K.KernelError) as e:
        K.linear4(torch.zeros(1, 64), torch.zeros(4, 64), torch.zeros(1, 4))
    assert "pack_weight4" in str(e.value)


def test_row_ranges_of_weights_start_at_tiles():
    w4 = K.pack_weight4(torch.randn(70, 64))
    assert w4[16:50].shape == (34, 64) and w4[:70].shape == (70, 64) and w4[48:].shape == (22, 64)
    for at in (slice(8, 20), slice(32, 32), slice(0, 70, 2), 3):
        with pytest.raises(K.KernelError):
            w4[at]


@pytest.mark.parametrize("head_dim,heads,page,group", [(40, 2, 64, 16), (272, 2, 64, 16), (64, 17, 64, 64), (64, 0, 64, 64), (64, 2, 40, 64), (64, 2, 64, 48), (96, 2, 64, 64)])
def test_attention_sizes(head_dim, heads, page, group):
    with pytest.raises(K.KernelError):
        K.attn4_lib(head_dim, heads, page, group)


def test_tensors_on_the_cpu():
    w4 = K.pack_weight4(torch.randn(16, 64))
    with pytest.raises(K.KernelError) as e:
        K.linear4(torch.zeros(1, 64), w4, torch.zeros(1, 16))
    assert "CUDA" in str(e.value)
    pages, ints = torch.zeros(2, 1, 64 * K.kv4_token_bytes(64, 64), dtype=torch.uint8), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: K.kv4_store(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), ints, ints, pages, pages, ints[None], 64),
                 lambda: K.kv4_expand(pages, pages, ints[None], ints, ints[:1], ints, torch.zeros(2, 1, 64, 64), torch.zeros(2, 1, 64, 64), 64, 64),
                 lambda: K.attn4_rows(torch.zeros(1, 1, 64), pages, pages, ints[None], ints, ints, torch.zeros(1, 64), 0.1, None, 64, 64)):
        with pytest.raises(K.KernelError) as e:
            call()
        assert "CUDA" in str(e.value)


@pytest.mark.parametrize("need", [KVNeed(2, 64, bits=8), KVNeed(2, 72, bits=4), KVNeed(2, 96, bits=4, bits_group=64), KVNeed(2, 64, bits=4, bits_group=24),
                                  KVNeed(2, 64, values=False, bits=4), KVNeed(2, 64, v_head_dim=32, bits=4), KVNeed(2, 64, 64, pool=16, bits=4)])
def test_cache_needs(need):
    with pytest.raises(CacheError):
        SequenceCache([(need, None)], [None], max_tokens=256, max_slots=2, max_seq_len=128, page_size=64, dtype=BF, device=torch.device("cpu"))


def test_a_cache_in_four_bits_is_smaller_by_its_format():
    make = lambda **kw: SequenceCache([(KVNeed(2, 128, **kw), None)] * 8, [None] * 8, max_tokens=640, max_slots=4, max_seq_len=128, page_size=64, dtype=BF,
                                      device=torch.device("cpu"))
    small, whole = make(bits=4), make()
    assert small.entry(0).k.shape == (10, 2, 64 * 72) and whole.entry(0).scratch is None
    assert small.bytes() == whole.bytes() * 72 // 256 + 2 * 640 * 2 * 128 * 2      # 72 bytes a token and head instead of 256, and pages of one layer


@pytest.mark.parametrize("n,k,group,dtype", [(5, 48, 16, torch.float32), (40, 128, 64, BF), (17, 320, 32, BF)])
def test_layout_of_packed_weights(n, k, group, dtype):
    """Every number's code and scale are where the layout says."""
    w = torch.randn(n, k).to(dtype)
    w[0, :group] = 0.5
    w4 = K.pack_weight4(w, group)
    values, s, z = P.group_values(w, group)
    codes, scales = w4.codes.view(-1, (k + 127) // 128 * 2, 32, 4, 4), w4.scales.double()
    for row in range(n):
        tile, h, r = row // 16, (row % 16) // 8, row % 8
        for col in range(k):
            block, step, c, e = col // 64, col % 64 // 16, col % 16 // 4, col % 4
            word = sum(int(codes[tile, block, 4 * r + c, step, i]) << (8 * i) for i in range(4))
            code = word >> (4 * (2 * (e // 2) + h) + 16 * (e % 2)) & 15
            sz = scales[tile, col // group, r, h]
            assert float(sz[0]) == float(s[row, col]) and float(sz[1]) == float(z[row, col])
            assert float(sz[1] + (code - 7.5) * sz[0]) == float(values[row, col])
