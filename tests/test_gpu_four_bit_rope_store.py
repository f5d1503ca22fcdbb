"""The engine's way into the 4-bit cache alone: per-head norm and rotation against 64 bits, what the pages then stand for to the last bit, and rows that the
launch before writes while this one is already there."""

import pytest
import torch

import plain_four_bit as P
from test_gpu_four_bit import SHAPES, Cache, i32
from test_gpu_kernels import DEV, K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def _rows(x, w, pos, rot, inv_freq):
    """``x`` ``[tokens, heads, d]`` normed and rotated in 64 bits, and how far a kernel may be.  Angles are 32-bit products, as they are defined.  Every rounding
    to the type moves a number by u of it (2^-8 or 2^-24) at most: two stand in the norm, one in each of cosine and sine, one in each product, one in the sum; beside
    them the 32-bit norm (a sum of d squares and a reciprocal root) and the functions' own errors, (d + 40) 2^-24 in all.  Doubled, for their products."""
    d = x.shape[-1]
    u = 2.0**-8 if x.dtype == BF else 2.0**-24
    a = x.double()
    if w is not None:
        a = a * torch.rsqrt((a**2).mean(-1, keepdim=True) + EPS) * w.double()
    each = 2 * u + (d + 40) * 2.0**-24
    want, slack = a.clone(), 2 * each * a.abs()
    if rot:
        h = rot // 2
        ang = (pos.float()[:, None] * inv_freq).double()[:, None]
        c, s, lo, hi = ang.cos(), ang.sin(), a[..., :h], a[..., h:rot]
        want[..., :h], want[..., h:rot] = lo * c - hi * s, hi * c + lo * s
        most = (lo.abs() * c.abs() + hi.abs() * s.abs(), hi.abs() * c.abs() + lo.abs() * s.abs())
        for at, m, other in ((slice(0, h), most[0], hi), (slice(h, rot), most[1], lo)):
            # (a cosine or sine near 0 is off by 2^-24 of 1, not of itself)
            slack[..., at] = 2 * (each + 3 * u) * m + 2.0**-22 * (a[..., at].abs() + other.abs())
    return want, slack


@pytest.mark.parametrize("kv,d,group", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page,normed,part,table", [(64, True, 1, False), (16, False, 1, True), (80, True, 2, True), (64, True, 0, False)])
def test_rows_are_normed_rotated_and_stored(kv, d, group, dtype, page, normed, part, table):
    """Key heads hold what the first query heads hold, so queries show what keys became; the pages stand for exactly that, coded."""
    lens, of = [1, 15, 64, 65, 200], 2
    heads, rot = kv * of, d // part // 2 * 2 if part else 0
    c = Cache(lens, kv, d, group, page, dtype)
    ids = [(b, p) for b, n in enumerate(lens) for p in range(n)]
    ids = ids[:7] + [(-1, 3)] + ids[7:]
    n = len(ids)
    qkv = (torch.randn(n, heads + 2 * kv, d) * torch.exp(0.5 * torch.randn(heads + 2 * kv, d))).to(dtype)
    qkv[:, heads:heads + kv] = qkv[:, :kv]
    w = [(1 + 0.2 * torch.randn(d)) if normed else None for _ in range(2)]
    on = [t.to(DEV) if t is not None else None for t in w]
    inv_freq = 1.0 / (10000.0 ** (torch.arange(0, rot, 2).float() / max(rot, 1)))
    slot, pos = i32([b for b, _ in ids]), i32([p for _, p in ids])
    x, freq = qkv.view(n, -1).to(DEV), inv_freq.to(DEV) if rot else None
    cs = K().rope_table(pos, freq, n, dtype) if table and rot else None
    q = [torch.full((n, heads, d), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
    before = c.k.clone()
    for i in (1, 0):   # the second call's keys have the norm weight of the first one's queries
        K().kv4_rope_store(x, on[i], on[1 - i], freq, slot, pos, q[i], c.k, c.v, c.pt, heads, kv, d, rot, EPS, group, cs_table=cs, pdl=True)
    have = torch.tensor([b >= 0 for b, _ in ids])
    assert torch.count_nonzero(q[0][~have.to(DEV)]) == 0
    for i in range(2):
        want, slack = _rows(qkv[:, :heads][have], w[i], pos.cpu()[have], rot, inv_freq)
        far = (q[i].cpu()[have].double() - want).abs() - slack
        assert far.max() <= 0, f"off by {float(far.max()):.3g} more than may be"
    held = set(c.table[c.table >= 0].tolist())
    for number in range(c.k.shape[0]):
        assert number in held or torch.equal(c.k[number], before[number])
    ko, vo = (torch.full((c.k.shape[0], kv, page, d), 9.0, dtype=F32, device=DEV) for _ in range(2))
    K().kv4_expand(c.k, c.v, c.pt, i32(range(len(lens) + 1)), i32(range(len(lens))), i32([m - 1 for m in lens]), ko, vo, group, max(lens))
    for b, m in enumerate(lens):
        rows = torch.tensor([i for i, (s, _) in enumerate(ids) if s == b])
        for made, out in ((q[1].cpu()[rows, :kv], ko), (qkv[rows, heads + kv:], vo)):
            got = torch.cat([out[int(c.table[b, i])].transpose(0, 1) for i in range(-(-m // page))])[:m]
            assert torch.equal(got.cpu(), P.group_values(made, group)[0].to(F32)), (b, out is vo)


@pytest.mark.parametrize("rows", [1, 4, 33])
@pytest.mark.parametrize("kv,of,d,group", [(8, 4, 128, 64), (2, 16, 256, 128)])
def test_rows_that_the_launch_before_writes(rows, kv, of, d, group):
    """Product, store and attention behind one another, thirty times over the same buffers, all launches overlapping: the bits of the same launches with the device idle in
    between."""
    heads, k = kv * of, 256
    width = (heads + 2 * kv) * d
    w4 = K().pack_weight4((torch.randn(width, k) / 16).to(BF).to(DEV))
    norm, freq = (1 + 0.2 * torch.randn(d)).to(DEV), 1.0 / (10000.0 ** (torch.arange(0, d, 2).float() / d)).to(DEV)
    xs = torch.randn(30, rows, k, device=DEV).to(BF)
    got = {}
    for pdl in (True, False):
        c = Cache([30] * rows, kv, d, group)
        slot, pos = i32(range(rows)), [i32([t] * rows) for t in range(30)]
        qkv, q, o = (torch.empty(rows, m, dtype=BF, device=DEV) for m in (width, heads * d, heads * d))
        outs = torch.empty(30, rows, heads * d, dtype=BF, device=DEV)
        torch.manual_seed(1)
        c.pt.copy_(torch.randperm(c.k.shape[0])[:rows, None])
        torch.cuda.synchronize()
        for t in range(30):
            K().linear4(xs[t], w4, qkv, pdl=pdl)
            K().kv4_rope_store(qkv, norm, norm, freq, slot, pos[t], q.view(rows, heads, d), c.k, c.v, c.pt, heads, kv, d, d, EPS, group, pdl=pdl)
            K().attn4_rows(q.view(rows, heads, d), c.k, c.v, c.pt, slot, pos[t], o, P.scale_of(d), None, group, 30, pdl=pdl)
            if not pdl:
                torch.cuda.synchronize()
            outs[t].copy_(o)
        got[pdl] = outs, c.k, c.v
    K().check_error_flags()
    assert all(torch.equal(a, b) for a, b in zip(got[True], got[False])) and got[True][0].isfinite().all()
