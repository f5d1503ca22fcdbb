"""The operators that serve from 4 bits: products with 4-bit weights, the paged cache in 4 bits, attention over it, against 64 bits."""

import importlib

import pytest
import torch

import plain_four_bit as P
from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)


def _near(got, want, slack, what=""):
    far = (got.double().cpu() - want).abs() - slack
    assert torch.isfinite(got).all(), what
    assert far.max() <= 0, f"{what}: {int((far > 0).sum())} of {far.numel()} values off by more than they may, the worst by {float(far.max()):.3g} more"


# ------------------------------------------------------------------------------------------------ products
def _weights(n, k, dtype):
    return (torch.randn(n, k) * torch.exp(0.5 * torch.randn(n, 1)) + 0.3 * torch.randn(n, 1)).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k,group", [(1, 16, 16), (15, 80, 16), (17, 64, 64), (389, 96, 32), (64, 2560, 128), (250, 1280, 64), (33, 9728, 64), (2000, 128, 128)])
def test_expanded_weights_are_the_codes_values(n, k, group, dtype):
    w = _weights(n, k, dtype)
    w[0] = 0.25                                                   # a group whose numbers are all the same
    w4 = K().pack_weight4(w.to(DEV), group)
    out = torch.full((n, k), 9.0, dtype=dtype, device=DEV)
    K().weight4_expand(w4, out)
    values, _, _ = P.group_values(w, group)
    assert torch.equal(out.cpu(), values.to(F32).to(dtype))       # one 32-bit rounding of z + (c - 7.5) s, then the type's


@pytest.mark.parametrize("m,dtype,out", [(m, *types) for types in ((BF, BF), (BF, F32), (F32, F32)) for m in ((1, 2, 7, 8, 9, 16) if types[0] == BF else (1, 2, 8, 9, 31, 64))])
@pytest.mark.parametrize("n,k,group", [(1, 16, 16), (389, 80, 16), (17, 64, 64), (250, 1280, 64), (100, 96, 32), (160, 2560, 128), (48, 9728, 64), (5000, 128, 128)])
def test_products_with_four_bit_weights(n, k, group, m, dtype, out):
    w, x = _weights(n, k, dtype), torch.randn(m, k).to(dtype)
    values, s, _ = P.group_values(w, group)
    y = torch.full((m, n), float("nan"), dtype=out, device=DEV)
    K().linear4(x.to(DEV), K().pack_weight4(w.to(DEV), group), y)
    slack = P.linear_slack(x, values, s, group, out)
    if K().linear4_plan(m, n, k, group, dtype == BF, out == F32):    # x does not fit beside the kernel's rings: weights are taken out tile by tile, as below
        slack = slack + (2.0**-8 if out == BF else 2.0**-17) * (x.double().abs() @ values.abs().T)
    _near(y, P.linear(x, values), slack)


@pytest.mark.parametrize("m", [17, 32, 33, 64, 65, 128, 129, 200, 256])
@pytest.mark.parametrize("n,k,group", [(1, 16, 16), (389, 80, 16), (17, 64, 64), (250, 1280, 64), (100, 96, 32), (160, 2560, 128), (128, 9728, 64), (20000, 128, 128)])
@pytest.mark.parametrize("out", [BF, F32])
def test_products_on_weights_taken_out_tile_by_tile(m, n, k, group, out):
    """Tiles that one block finishes, that several share, and that outnumber the blocks.  Weights are multiplied as bfloat16 numbers, one (off by
    up to 2^-8 of each) or, for 32-bit results, two (up to 2^-16, 2^-18 in the mean square)."""
    w, x = _weights(n, k, BF), torch.randn(m, k).to(BF)
    values, s, _ = P.group_values(w, group)
    w4, y = K().pack_weight4(w.to(DEV), group), torch.full((m, n), float("nan"), dtype=out, device=DEV)
    for _ in range(2):
        K().linear4(x.to(DEV), w4, y, pdl=True)
    K().check_error_flags()
    _near(y, P.linear(x, values), P.linear_slack(x, values, s, group, out) + (2.0**-8 if out == BF else 2.0**-17) * (x.double().abs() @ values.abs().T))


@pytest.mark.parametrize("m", [257, 300])
@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32)])
def test_products_of_many_rows(m, dtype, out, monkeypatch):
    """More rows than the kernel takes: weights out of their 4 bits, in parts (here of 64 rows of W)."""
    L = importlib.import_module("dryft_b200.parts.linear")
    from dryft_b200.parts.base import Runtime

    monkeypatch.setattr(L, "EXPAND_BYTES", 64 * 320 * (2 if dtype == BF else 4))
    n, k, group = 250, 320, 64
    w, x = _weights(n, k, dtype), torch.randn(m, k).to(dtype)
    values, s, _ = P.group_values(w, group)
    y = L.linear(x.to(DEV), K().pack_weight4(w.to(DEV), group), Runtime(dtype=dtype, device=torch.device(DEV)), out_dtype=out)
    slack = P.linear_slack(x, values, s, group, out)
    if dtype == BF:   # the values are rounded to bfloat16 for this product, once or (32-bit results) as two numbers: up to 2^-8 of each, or 2^-16 (allowed: 2^-17)
        slack = slack + (2.0**-8 if out == BF else 2.0**-17) * (x.double().abs() @ values.abs().T)
    _near(y, P.linear(x, values), slack)


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16])
@pytest.mark.parametrize("n,k,group", [(32, 16, 16), (64, 64, 64), (96, 96, 32), (1312, 2560, 128), (192, 80, 16), (10016, 128, 64)])
def test_products_with_the_norm_before_and_the_sum_or_activation_behind(m, n, k, group):
    """The norm against 64 bits (its two roundings are allowed one unit, 2^-8, of each number; the other half is left to their signs).  What follows a product
    is held to the last bit: the same kernel's plain product, rounded where the products of bfloat16 weights round, and the activation of its own launch."""
    w, x, norm = _weights(n, k, BF) / k**0.5, torch.randn(m, k).to(BF), (1 + 0.2 * torch.randn(k)).to(DEV)
    values, s, _ = P.group_values(w, group)
    w4, eps, xd = K().pack_weight4(w.to(DEV), group), 1e-6, x.to(DEV)
    h = x.double() * torch.rsqrt((x.double()**2).mean(1, keepdim=True) + eps) * norm.double().cpu()
    new = lambda cols, dtype=BF: torch.full((m, cols), float("nan"), dtype=dtype, device=DEV)
    out32 = new(n, F32)
    K().linear4(xd, w4, out32, norm_w=norm, eps=eps)
    _near(out32, P.linear(h, values), P.linear_slack(h.to(BF), values, s, group, F32) + (2.0**-8 + 1e-5) * (h.abs() @ values.abs().T))
    y0 = torch.randn(m, n, device=DEV).to(BF)
    for more in ({}, dict(norm_w=norm, eps=eps)):
        plain, wide, total, act, want = new(n), new(n, F32), y0.clone(), new(n // 2), new(n // 2)
        K().linear4(xd, w4, plain, **more)
        K().linear4(xd, w4, wide, **more)
        assert torch.equal(plain, wide.to(BF))
        K().linear4(xd, w4, total, pdl=True, mode="residual", **more)
        assert torch.equal(total, (y0.float() + plain.float()).to(BF))
        K().linear4(xd, w4, act, pdl=True, mode="silu", **more)
        K().silu_mul(plain, want)
        assert torch.equal(act, want)


def test_many_rows_of_results_that_begin_anywhere():
    """685 rows of 439 outputs, held against 64 bits as a whole: roundings to bfloat16, of the weights and of the result, may be its only errors.  Either is below
    2^-9 in the mean square (up to 2^-8 of a number, less towards the next power of two), so the whole is off by 2^-9 times the square root of 2 at most."""
    L = importlib.import_module("dryft_b200.parts.linear")
    from dryft_b200.parts.base import Runtime

    m, n, k = 685, 439, 8496
    w, x = torch.randn(n, k).to(BF), torch.randn(m, k).to(BF)
    want = P.linear(x, P.group_values(w, 16)[0])
    y = L.linear(x.to(DEV), K().pack_weight4(w.to(DEV), 16), Runtime(dtype=BF, device=torch.device(DEV)))
    assert (y.double().cpu() - want).norm() <= 2.0**-9 * 2**0.5 * want.norm()


def test_modes_that_are_refused():
    w4, t = K().pack_weight4(torch.randn(48, 64, device=DEV)), lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=DEV)
    for x, out, more in ((t(17, 64), t(17, 48), dict(mode="residual")), (t(1, 64, dtype=F32), t(1, 48, dtype=F32), dict(norm_w=t(64, dtype=F32))), (t(1, 64), t(1, 24), dict(mode="silu")),
                         (t(1, 64), t(1, 48, dtype=F32), dict(mode="residual")), (t(1, 64), t(1, 48), dict(mode="relu")), (t(1, 64), t(1, 48), dict(norm_w=t(64))),
                         (t(1, 64), t(1, 48), dict(norm_w=t(63, dtype=F32)))):
        with pytest.raises(K().KernelError):
            K().linear4(x, w4, out, **more)


def test_a_rows_bits_do_not_depend_on_the_other_rows_among_eight():
    n, k = 250, 2560
    w4, x = K().pack_weight4(_weights(n, k, BF).to(DEV)), torch.randn(8, k, device=DEV).to(BF)
    one, all_ = torch.empty(1, n, device=DEV), torch.empty(8, n, device=DEV)
    K().linear4(x, w4, all_)
    for i in range(8):
        K().linear4(x[i:i + 1], w4, one)
        assert torch.equal(one[0], all_[i])


def test_rows_that_lie_further_apart_and_row_ranges():
    n, k = 96, 128
    w = _weights(n, k, BF)
    w4 = K().pack_weight4(w.to(DEV), 32)
    x = torch.randn(5, 3 * k, device=DEV).to(BF)
    want, y = torch.empty(5, n, dtype=BF, device=DEV), torch.empty(5, n, dtype=BF, device=DEV)
    K().linear4(x[:, k:2 * k].contiguous(), w4, want)
    K().linear4(x[:, k:2 * k], w4, y)
    assert torch.equal(y, want)
    part = torch.empty(5, 37, dtype=BF, device=DEV)
    K().linear4(x[:, k:2 * k], w4[32:69], part)
    assert torch.equal(part, want[:, 32:69])


def test_not_a_number_stays_in_its_group_and_its_row():
    w, x = _weights(40, 128, BF), torch.randn(6, 128).to(BF)
    w[3, 70], w[21, 5], x[2, 9], x[4, 100] = float("nan"), float("inf"), float("nan"), float("inf")
    w4 = K().pack_weight4(w.to(DEV), 64)
    out = torch.empty(40, 128, device=DEV)
    K().weight4_expand(w4, out)
    bad = torch.zeros(40, 128, dtype=torch.bool)
    bad[3, 64:] = bad[21, :64] = True
    assert torch.equal(out.isnan().cpu(), bad)
    y = torch.empty(6, 40, device=DEV)
    K().linear4(x.to(DEV), w4, y)
    bad = torch.zeros(6, 40, dtype=torch.bool)
    bad[:, 3] = bad[:, 21] = bad[2] = bad[4] = True
    assert torch.equal((~y.isfinite()).cpu(), bad)


# ------------------------------------------------------------------------------------------------ the cache
class Cache:
    """Pages scattered over a pool that held something else: every byte 0xff to begin with, which makes scales NaN."""

    def __init__(self, lens, kv, d, group, page=64, dtype=BF):
        self.lens, self.kv, self.d, self.group, self.page, self.dtype = lens, kv, d, group, page, dtype
        need = [-(-n // page) for n in lens]
        order = torch.randperm(sum(need) + 3).tolist()
        self.table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)     # an entry that nothing may read
        for b, n in enumerate(need):
            for i in range(n):
                self.table[b, i] = order.pop()
        shape = (sum(need) + 3, kv, page * K().kv4_token_bytes(d, group))
        self.k, self.v = (torch.full(shape, 255, dtype=torch.uint8, device=DEV) for _ in range(2))
        self.pt = self.table.to(DEV)
        self.keys = [torch.randn(n, kv, d).mul(torch.exp(0.5 * torch.randn(kv, d))).to(dtype) for n in lens]
        self.values = [torch.randn(n, kv, d).to(dtype) for n in lens]

    def store(self, ids):
        """``ids``: (sequence, position), -1 for padding."""
        pick = lambda what: torch.stack([what[b][p] if b >= 0 else torch.full((self.kv, self.d), 7.0, dtype=self.dtype) for b, p in ids]).to(DEV)
        K().kv4_store(pick(self.keys), pick(self.values), i32([b for b, _ in ids]), i32([p for _, p in ids]), self.k, self.v, self.pt, self.group)

    def fill(self):
        self.store([(b, p) for b, n in enumerate(self.lens) for p in range(n)])


SHAPES = [(1, 16, 16), (2, 32, 32), (3, 48, 16), (2, 64, 64), (2, 80, 16), (1, 96, 32), (8, 128, 64), (2, 128, 128), (5, 192, 64), (2, 256, 16), (1, 256, 128)]


@pytest.mark.parametrize("kv,d,group", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 48, 64, 80, 128])
def test_stored_tokens_come_back_as_their_codes_values(kv, d, group, dtype, page):
    lens = [1, 15, 64, 65, 200]
    c = Cache(lens, kv, d, group, page, dtype)
    c.values[2][:, 0] = 0.5                                       # every number of a head's token the same
    before = c.k.clone()
    # the first tokens in one call, a padding token among them, then sequences go on by one token and by several
    first = [(b, p) for b, n in enumerate(lens) for p in range(n - min(n, b + 1))]
    c.store(first[:7] + [(-1, 3)] + first[7:])
    c.store([(b, p) for b, n in enumerate(lens) for p in range(n - min(n, b + 1), n)])
    held = set(c.table[c.table >= 0].tolist())
    for page_no in range(c.k.shape[0]):
        assert page_no in held or torch.equal(c.k[page_no], before[page_no])      # nothing outside the sequences' pages is written
    new = [min(n, b + 1) for b, n in enumerate(lens)]
    cu, pos = [sum(new[:b]) for b in range(len(lens) + 1)], [p for n, m in zip(lens, new) for p in range(n - m, n)]
    ko, vo = (torch.full((c.k.shape[0], kv, page, d), 9.0, dtype=dtype, device=DEV) for _ in range(2))
    K().kv4_expand(c.k, c.v, c.pt, i32(cu), i32(range(len(lens))), i32(pos), ko, vo, group, max(lens))
    for b, n in enumerate(lens):
        for mine, out in ((c.keys[b], ko), (c.values[b], vo)):
            want = torch.zeros(-(-n // page) * page, kv, d, dtype=dtype)
            want[:n] = P.group_values(mine, group)[0].to(F32).to(dtype)
            got = torch.cat([out[int(c.table[b, i])].transpose(0, 1) for i in range(-(-n // page))])
            assert torch.equal(got.cpu(), want)
    assert (ko[[i for i in range(c.k.shape[0]) if i not in held]] == 9).all()


def test_expansion_leaves_what_no_token_sees_and_sequences_without_tokens():
    c = Cache([300, 200, 100], 2, 64, 64)
    c.fill()
    ko, vo = (torch.full((c.k.shape[0], 2, 64, 64), 9.0, dtype=BF, device=DEV) for _ in range(2))
    # sequence 0 brings two tokens, sequence 1 none, 2 is padding; a window of 40 keys reaches back to 259 - page 4 alone
    K().kv4_expand(c.k, c.v, c.pt, i32([0, 2, 2, 3]), i32([0, 1, -1]), i32([298, 299, 99]), ko, vo, 64, 300, window=40)
    written = [i for i in range(ko.shape[0]) if not (ko[i] == 9).all()]
    assert written == [int(c.table[0, 4])]


def test_tokens_with_an_infinity_or_nan_stand_for_nan_in_their_groups():
    c = Cache([3], 1, 128, 64)
    c.keys[0][1, 0, 70], c.values[0][2, 0, 3] = float("inf"), float("nan")
    c.fill()
    ko, vo = (torch.empty(c.k.shape[0], 1, 64, 128, device=DEV) for _ in range(2))
    K().kv4_expand(c.k, c.v, c.pt, i32([0, 3]), i32([0]), i32([0, 1, 2]), ko, vo, 64, 3)
    bad = torch.zeros(2, 3, 128, dtype=torch.bool)
    bad[0, 1, 64:] = bad[1, 2, :64] = True
    page = int(c.table[0, 0])
    assert torch.equal(torch.stack([ko[page, 0, :3], vo[page, 0, :3]]).isnan().cpu(), bad)


def test_columns_of_a_fused_projection_are_stored_in_place():
    c, d = Cache([70], 2, 64, 64), 64
    qkv = torch.randn(70, 8 * d).to(BF)
    c.keys[0], c.values[0] = qkv[:, 4 * d:6 * d].view(70, 2, d), qkv[:, 6 * d:].view(70, 2, d)
    c.fill()
    want = c.k.clone(), c.v.clone()
    on = qkv.to(DEV)
    c.k.fill_(255), c.v.fill_(255)
    K().kv4_store(on[:, 4 * d:6 * d].view(70, 2, d), on[:, 6 * d:].view(70, 2, d), i32([0] * 70), i32(range(70)), c.k, c.v, c.pt, 64)
    assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])


# ------------------------------------------------------------------------------------------------ attention
def _attend(c, heads, rows, window, max_kv=None, q=None):
    """``rows``: (sequence or -1, position).  Checks against 64 bits and returns the output."""
    scale = P.scale_of(c.d)
    q = torch.randn(len(rows), heads, c.d).to(c.dtype) if q is None else q
    out = torch.full((len(rows), heads * c.d), float("nan"), dtype=c.dtype, device=DEV)
    K().attn4_rows(q.to(DEV), c.k, c.v, c.pt, i32([b for b, _ in rows]), i32([p for _, p in rows]), out, scale, window, c.group, max_kv or max(c.lens))
    held = {}
    for i, (b, p) in enumerate(rows):
        if b < 0:
            assert torch.count_nonzero(out[i]) == 0
            continue
        if b not in held:
            held[b] = (P.group_values(c.keys[b], c.group)[0], *P.group_values(c.values[b], c.group)[::2])
        k, v, z = held[b]
        want, weights, first = P.attention(q[i].double(), k, v, p, scale, window)
        slack = P.attention_slack(q[i].double(), k, v, z, weights, first, scale, c.dtype == BF)
        _near(out[i].view(heads, c.d), want, slack, f"row {i}, sequence {b}, position {p}")
    return out


HEADS = [1, 2, 3, 4, 9, 6, 4, 16, 8, 2, 16]      # query heads per key head, shape by shape


@pytest.mark.parametrize("kv,d,group,of", [(*shape, of) for shape, of in zip(SHAPES, HEADS)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_at_the_edges_of_tiles_and_pages(kv, d, group, of, dtype):
    lens = [1, 15, 16, 17, 63, 64, 65, 130, 333]
    c = Cache(lens, kv, d, group, 64, dtype)
    c.fill()
    rows = [(-1, 500)] + [(b, n - 1) for b, n in enumerate(lens)] + [(8, 100), (-1, 0)]
    _attend(c, kv * of, rows, None)
    _attend(c, kv * of, rows, 20)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 64, 100, 4000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_windows(window, dtype):
    c = Cache([1, 16, 100, 700], 2, 64, 64, 64, dtype)
    c.fill()
    _attend(c, 8, [(0, 0), (1, 15), (2, 99), (3, 699), (3, 640), (3, 63)], window)


@pytest.mark.parametrize("lens,heads,kv", [([5000], 8, 1), ([16383], 64, 8), ([3000, 1], 4, 2), ([700] * 40, 8, 8), ([8192, 1, 4000, 77], 32, 8)])
@pytest.mark.parametrize("page", [16, 64])
def test_long_sequences_in_many_splits(lens, heads, kv, page):
    c = Cache(lens, kv, 128, 64, page)
    c.fill()
    _attend(c, heads, [(b, n - 1) for b, n in enumerate(lens)][:6], None)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_row_shorter_than_its_launch_was_cut_for(dtype):
    """``max_kv`` is a bound: most splits of a short row have no keys."""
    c = Cache([3, 40, 90], 2, 64, 64, 64, dtype)
    c.fill()
    _attend(c, 4, [(0, 2), (1, 39), (2, 89)], None, max_kv=8192)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scores_that_differ_by_hundreds(dtype):
    """Weights far below what 32 bits hold, the largest score first, last and in the middle."""
    c = Cache([257, 257, 257], 1, 64, 64, 64, dtype)
    for b, at in enumerate((0, 256, 100)):
        c.keys[b] *= 3
        c.keys[b][at] = 40 * torch.sign(torch.arange(64) - 31.5).to(dtype)
    c.fill()
    q = (20 * torch.sign(torch.arange(64) - 31.5)).expand(3, 2, 64).to(dtype).clone()
    q[:, 1] *= -1
    _attend(c, 2, [(0, 256), (1, 256), (2, 256)], None, q=q)


def test_a_poisoned_token_poisons_its_readers_only():
    c = Cache([200, 200], 1, 64, 64)
    c.values[0][150, 0, 3] = float("nan")
    c.fill()
    q = torch.randn(4, 2, 64).to(BF).to(DEV)
    out = torch.empty(4, 128, dtype=BF, device=DEV)
    K().attn4_rows(q, c.k, c.v, c.pt, i32([0, 0, 0, 1]), i32([199, 150, 149, 199]), out, 0.125, None, 64, 200)
    assert out.isnan().all(-1).tolist() == [True, True, False, False] and not out[2:].isnan().any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [145, 2100])
def test_a_poisoned_key_alone_in_its_tile_is_not_lost(n, dtype):
    """The last key, alone in its tile and so with its warp (or its split) alone, has a score of NaN: the row's output is NaN."""
    c = Cache([n, n], 1, 64, 64, 64, dtype)
    c.keys[0][n - 1, 0, 3] = float("nan")
    c.fill()
    out = torch.empty(2, 128, dtype=dtype, device=DEV)
    K().attn4_rows(torch.randn(2, 2, 64).to(dtype).to(DEV), c.k, c.v, c.pt, i32([0, 1]), i32([n - 1, n - 1]), out, 0.125, None, 64, n)
    assert out[0].isnan().all() and out[1].isfinite().all()


def test_the_same_bits_every_time_and_on_another_stream():
    c = Cache([2000, 31, 700], 2, 128, 64)
    c.fill()
    rows = [(0, 1999), (1, 30), (2, 699), (-1, 0)]
    q = torch.randn(4, 8, 128).to(BF)
    first = _attend(c, 8, rows, None, q=q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            again = torch.empty_like(first)
            K().attn4_rows(q.to(DEV), c.k, c.v, c.pt, i32([b for b, _ in rows]), i32([p for _, p in rows]), again, P.scale_of(128), None, 64, 2000)
            assert torch.equal(again, first)
    torch.cuda.current_stream().wait_stream(side)
