"""Calls of the operators that serve from 4 bits that would give wrong numbers or touch memory where they may not are refused by name before anything is
launched (no GPU needed)."""

from types import SimpleNamespace

import pytest
import torch

from dryft_b200.ops import kernels as K

BF, F32 = torch.bfloat16, torch.float32


class OnDevice(torch.Tensor):
    """A tensor that says it is on a GPU; where launches are replaced, too (``launches``), checks of arguments run as there."""

    is_cuda = property(lambda self: True)


def on(t):
    return t.as_subclass(OnDevice)


def begins_at(shape, dtype, numbers):
    """A contiguous tensor that begins ``numbers`` numbers behind a 64-byte boundary."""
    size = torch.Size(shape).numel()
    buf = torch.zeros(size + 64, dtype=dtype)
    first = -(buf.data_ptr() // buf.element_size()) % (64 // buf.element_size()) + numbers
    return on(buf[first:first + size].view(shape))


@pytest.fixture
def launches(monkeypatch):
    """Every launch of these operators is counted instead of made."""
    made = []

    def launch(*a):
        made.append(a)
        return 0

    lib = SimpleNamespace(dryft_weight4_expand=launch, dryft_kv4_rope_store=launch, dryft_attn4_rows=launch)
    monkeypatch.setattr(K, "linear4_lib", lambda: lib)
    monkeypatch.setattr(K, "kv4_lib", lambda: lib)
    monkeypatch.setattr(K, "_kv4_calls", lambda: (launch, launch))
    monkeypatch.setattr(K, "attn4_lib", lambda *a: lib)
    monkeypatch.setattr(K, "_variants", {})
    monkeypatch.setattr(K, "_stream", lambda: 0)
    return made


def test_a_sum_into_nothing():
    """``out += x @ w.T`` needs an ``out``."""
    w4 = K.pack_weight4(torch.randn(48, 64))
    with pytest.raises(K.KernelError, match="no out was given"):
        K.linear4(torch.zeros(1, 64, dtype=BF), w4, mode="residual")


@pytest.mark.parametrize("dtype,word", [(BF, 8), (F32, 16)])
def test_expanded_weights_begin_on_a_word(launches, dtype, word):
    w4 = K.pack_weight4(torch.randn(16, 64))
    w4 = K.Weight4(on(w4.codes), on(w4.scales), w4.n, w4.k, w4.group)
    for numbers in range(9):
        out = begins_at((16, 64), dtype, numbers)
        if out.data_ptr() % word:
            with pytest.raises(K.KernelError, match="boundary"):
                K.weight4_expand(w4, out)
        else:
            K.weight4_expand(w4, out)
    assert len(launches) == 3


def _pages(d, group, kv=1):
    pages = [on(torch.zeros(2, kv, 64 * K.kv4_token_bytes(d, group), dtype=torch.uint8)) for _ in range(2)]
    return *pages, on(torch.zeros(1, 2, dtype=torch.int32))


ints = lambda *v: on(torch.tensor(v, dtype=torch.int32))


@pytest.mark.parametrize("dtype,word", [(BF, 8), (F32, 16)])
@pytest.mark.parametrize("which", [0, 1])
def test_expanded_pages_begin_on_a_word(launches, dtype, word, which):
    for numbers in range(9):
        out = [begins_at((2, 1, 64, 64), dtype, numbers if i == which else 0) for i in range(2)]
        call = lambda: K.kv4_expand(*_pages(64, 64), ints(0, 1), ints(0), ints(0), *out, 64, 64)
        if out[which].data_ptr() % word:
            with pytest.raises(K.KernelError, match="_out: begins"):
                call()
        else:
            call()
    assert len(launches) == 3


@pytest.mark.parametrize("q_at,out_at,dtype,fine", [(0, 0, BF, True), (4, 2, BF, True), (2, 0, BF, False), (1, 0, BF, False), (0, 1, BF, False), (1, 1, F32, True)])
def test_queries_and_outputs_begin_on_a_word(launches, q_at, out_at, dtype, fine):
    q, out = begins_at((1, 2, 64), dtype, q_at), begins_at((1, 128), dtype, out_at)
    call = lambda: K.attn4_rows(q, *_pages(64, 64), ints(0), ints(0), out, 0.125, None, 64, 64)
    if fine:
        call()
    else:
        with pytest.raises(K.KernelError, match="boundary"):
            call()
    assert len(launches) == fine


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("at", [0, 1, 2, 3, 4])
def test_a_projections_rows_begin_on_a_word(launches, dtype, at):
    qkv, q = begins_at((1, 4 * 64), dtype, at), begins_at((1, 2, 64), dtype, 0)
    call = lambda: K.kv4_rope_store(qkv, None, None, None, ints(0), ints(0), q, *_pages(64, 64), 2, 1, 64, 0, 1e-6, 64)
    if at % 2:
        with pytest.raises(K.KernelError, match="qkv: begins"):
            call()
    else:
        call()
    assert len(launches) == (at % 2 == 0)


@pytest.mark.parametrize("n,k", [(40, 64), (70, 128)])
def test_a_launch_stands_behind_the_last_write_of_packed_weights(n, k):
    """A product that overlaps the launch in front of it asks for its weights before that launch has ended: that launch must not be the one that wrote them."""
    from torch.utils._python_dispatch import TorchDispatchMode

    made = []   # of every operation that writes: the memory it writes to

    class Ops(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            to = [a for a, info in zip(args, func._schema.arguments) if info.alias_info is not None and info.alias_info.is_write]
            if not to and not any(r.alias_info for r in func._schema.returns) and "empty" not in str(func):
                to = [out] if isinstance(out, torch.Tensor) else []
            made.extend(t.untyped_storage().data_ptr() for t in to)
            return out

    with Ops():
        w4 = K.pack_weight4(torch.randn(n, k))
    mine = {t.untyped_storage().data_ptr() for t in (w4.codes, w4.scales)}
    assert mine <= set(made) and made[-1] not in mine
