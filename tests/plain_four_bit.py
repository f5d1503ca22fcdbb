"""Numbers held in 4 bits, written down plainly on the CPU: codes by the 32-bit steps that define them, everything behind them in 64 bits.
Shares no code with the product."""

import math

import torch


def group_values(x, group):
    """(values, s, z) of ``x`` ``[..., size]`` in 64 bits: what its 4-bit form stands for, and every number's group's s and z."""
    f = lambda t: t.float().double()                       # one 32-bit rounding (of a 64-bit result: the correctly rounded one)
    a = x.double().reshape(*x.shape[:-1], -1, group)
    lo, hi = a.min(-1, keepdim=True).values, a.max(-1, keepdim=True).values
    s, z = (f(f(hi - lo) / 15)).bfloat16().double(), (f(hi + lo) / 2).bfloat16().double()
    c = torch.round(f(f(f(a - z) / s) + 7.5)).clamp(0, 15)
    c = torch.where(s == 0, torch.full_like(c, 8.0), c)
    whole = lambda t: t.expand_as(a).reshape(x.shape)
    return (z + (c - 7.5) * s).reshape(x.shape), whole(s), whole(z)


def attention(q, k, v, pos, scale, window=None):
    """``q`` ``[heads, d]`` at position ``pos`` over ``k``, ``v`` ``[tokens, kv heads, d]``, all in 64 bits: (output, weights ``[heads, keys]``,
    first key)."""
    of = q.shape[0] // k.shape[1]
    first = max(0, pos + 1 - window) if window else 0
    kk, vv = k[first:pos + 1].repeat_interleave(of, 1), v[first:pos + 1].repeat_interleave(of, 1)
    p = torch.softmax(torch.einsum("hd,jhd->hj", q, kk) * scale, -1)
    return torch.einsum("hj,jhd->hd", p, vv), p, first


def attention_slack(q, k, v, z, p, first, scale, bf16):
    """How far a kernel's output may be from ``attention``'s, element by element.

    32-bit: a score is a sum of d products, each rounding 2^-24 of it: off by at most (d + 4) 2^-24 sum |q k| scale; the weights by twice that, and
    the exponential, the products and the sums over the keys by (keys + 16) 2^-24 more; all of it times sum p |v|.  bfloat16 on the tensor cores: sums
    over 16 + code are up to 31 s where the number is up to 7.5 s, so 8 times that for a score, beside 2^-9 of p s (c - 7.5) for a weight rounded
    with its scale, 2^-9 of the output, both doubled."""
    of = q.shape[0] // k.shape[1]
    n = p.shape[1]
    kk, vv, zz = (t[first:first + n].repeat_interleave(of, 1) for t in (k, v, z))
    d = q.shape[1]
    score = (d + 4) * 2.0**-24 * scale * torch.einsum("hd,jhd->hj", q.abs(), kk.abs()).amax(-1, keepdim=True)
    each = 2 * score * (8 if bf16 else 1) + (n + 16) * 2.0**-24
    slack = each * torch.einsum("hj,jhd->hd", p, vv.abs() + zz.abs())
    if bf16:
        slack = slack + 2.0**-8 * torch.einsum("hj,jhd->hd", p, (vv - zz).abs()) + 2.0**-8 * torch.einsum("hj,jhd->hd", p, vv).abs()
    return slack


def linear(x, w_values):
    return x.double() @ w_values.T


def linear_slack(x, values, s, group, out):
    """32-bit sums of k terms, group by group; on the tensor cores over 16 + code, corrected by 23.5 times the group's sum: (group / 16 + 2) steps of a
    group and 2^-23 of 54.5 s |x| each (doubled for what a step loses inside), then one step a group of what the groups' sums come to; 2^-24 a term
    where the products are one after another.  A bfloat16 result: 2^-8 of it (twice its rounding)."""
    k = x.shape[1]
    a = x.double().abs()
    slack = 2 * (group / 16 + 2) * 2.0**-23 * 54.5 * (a @ s.T) + (k / group + 80) * 2.0**-24 * (a @ values.abs().T)
    return slack + (2.0**-8 * linear(x, values).abs() if out == torch.bfloat16 else 0)


def scale_of(d):
    return 1.0 / math.sqrt(d)
