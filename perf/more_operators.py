"""The operators that serve a decoder from microscaled 4-bit floating point: rounding to it, its values, products of two operands that are both held in it.

A number is one of 0, 1/2, 1, 3/2, 2, 3, 4 and 6, or minus that, times the scale of its group (of consecutive numbers of a row); a last group may be short.
Every step below is a 32-bit one, |.| are the magnitudes of finite numbers, and roundings are to the nearest, ties to the even code:

    "mx": groups of 32.  s = 2^max(floor(log2 max|group|) - 2, -127),             c = fp4(x / s),              value c s
    "nv": groups of 16.  g = max(max|row| / 2688, 2^-112), u = 1 / (6 g),
                         s = e4m3(max|group| u),  r = 1 / (s g) (0 where s = 0),  c = fp4(x r),                value (c s) g

Magnitudes above 6 become 6.  A group with an infinity or a NaN stands for NaN.
"""

import math

import torch

own = False

DEVICE = "cuda"
GROUP = {"mx": 32, "nv": 16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # products.  One sequence's fused query, key and value projection (the 4B shape): latency counts
        dict(name="product 1 row qkv", op="product", kind="nv", m=1, n=6144, k=2560, dtype="bfloat16", out="bfloat16", silu=False),
        # the output head of one sequence, 32-bit logits: the most weight bytes that a step reads in one product
        dict(name="product 1 row head", op="product", kind="nv", m=1, n=151936, k=2560, dtype="bfloat16", out="float32", silu=False),
        # gate and up projections of eight sequences
        dict(name="product 8 rows gate up", op="product", kind="mx", m=8, n=19456, k=2560, dtype="bfloat16", out="bfloat16", silu=False),
        # down projection of a batch of 48, from the fused gate and up projections
        dict(name="product 48 rows silu down", op="product", kind="nv", m=48, n=2560, k=9728, dtype="bfloat16", out="bfloat16", silu=True),
        # a ragged prompt through the 8B shape's gate and up projections
        dict(name="product 777 rows gate up", op="product", kind="nv", m=777, n=24576, k=4096, dtype="bfloat16", out="bfloat16", silu=False),
        # a prompt of 2,048 tokens through the 32B shape's down projection
        dict(name="product 2048 rows down", op="product", kind="mx", m=2048, n=5120, k=25600, dtype="bfloat16", out="bfloat16", silu=False),
        # the 32-bit path of a tiny model: widths that fill neither groups nor tiles
        dict(name="product 5 rows f32", op="product", kind="nv", m=5, n=389, k=83, dtype="float32", out="float32", silu=False),
        # rounding.  One token's activations
        dict(name="round 1 row", op="round", kind="nv", m=1, k=2560, apart=0, dtype="bfloat16"),
        # a prompt's activations in front of the down projection
        dict(name="round 2000 rows", op="round", kind="mx", m=2000, k=9728, apart=0, dtype="bfloat16"),
        # 32-bit rows of an odd width, taken out of wider ones
        dict(name="round 333 odd rows f32", op="round", kind="nv", m=333, k=1001, apart=7, dtype="float32"),
        # values.  A layer's gate and up projections, for a product that wants them as they are
        dict(name="values 19456 x 2560", op="values", kind="mx", m=19456, k=2560, dtype="bfloat16"),
        # a few rows of an odd width, 32 bits
        dict(name="values 77 odd rows f32", op="values", kind="nv", m=77, k=4111, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: whole groups as most models have them, or any."""
    k = _log_int(rng, lo, hi)
    return k if rng.random() < 0.3 else max(64, k // 64 * 64)


def draw(rng):
    op = rng.choice(["product", "product", "round", "values"])
    kind = rng.choice(["mx", "nv"])
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    if op == "product":
        k, m = _width(rng, 16, 25600), _log_int(rng, 1, 2048)
        n = _log_int(rng, 64, max(65, min(151936, 5 * 10**11 // (2 * m * k), 388 * 10**6 // k)))
        out = "float32" if dtype == "float32" or rng.random() < 0.2 else "bfloat16"
        return dict(op=op, kind=kind, m=m, n=n, k=k, dtype=dtype, out=out, silu=out == "bfloat16" and rng.random() < 0.2)
    k = _width(rng, 16, 25600)
    m = _log_int(rng, 1, 5 * 10**7 // k if op == "values" else 2 * 10**7 // k)
    if op == "values":
        return dict(op=op, kind=kind, m=m, k=k, dtype=dtype)
    return dict(op=op, kind=kind, m=m, k=k, apart=rng.choice([0, 0, 1, 8]), dtype=dtype)


def _item(dtype):
    return 4 if dtype == "float32" else 2


def _held_bytes(rows, k, kind):
    """Bytes of a matrix in 4 bits: its codes, a byte for each group, and for "nv" four for each row."""
    return rows * (math.ceil(k / 2) + math.ceil(k / GROUP[kind]) + (4 if kind == "nv" else 0))


def work(case):
    e, m, k = _item(case["dtype"]), case["m"], case["k"]
    if case["op"] == "product":
        n = case["n"]
        return {"bytes": _held_bytes(n, k, case["kind"]) + m * k * e * (2 if case["silu"] else 1) + m * n * _item(case["out"]), "flops": 2 * m * n * k}
    if case["op"] == "values":   # the held form in, values out
        return {"bytes": _held_bytes(m, k, case["kind"]) + m * k * e, "flops": 2 * m * k}
    return {"bytes": 2 * m * k * e + 2 * _held_bytes(m, k, case["kind"]), "flops": 6 * m * k}   # numbers in, the held form out and in, values out


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(name):
    return {"float32": torch.float32, "bfloat16": torch.bfloat16}[name]


def _rows(case, rows, k, g):
    """Activations with a few large channels."""
    x = torch.randn(rows, k, generator=g, device=DEVICE)
    return (x * torch.exp(0.5 * torch.randn(1, k, generator=g, device=DEVICE))).to(_dtype(case["dtype"]))


def _weights(case, rows, g):
    """Weights as a checkpoint has them (rows of unequal size)."""
    w = torch.randn(rows, case["k"], generator=g, device=DEVICE) * 0.02
    return (w * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEVICE))).to(_dtype(case["dtype"]))


def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    if case["op"] == "product":
        return {"w": _weights(case, case["n"], g), "x": _rows(case, case["m"], case["k"] * (2 if case["silu"] else 1), g)}
    if case["op"] == "values":
        return {"w": _weights(case, case["m"], g)}
    return {"x": _rows(case, case["m"], case["k"] + case["apart"], g)[:, :case["k"]]}


def prepare(case, seed):
    made = _inputs(case, seed)
    state = {"case": case}
    if "x" in made:
        state["x"] = made["x"]
    if own:
        from dryft_b200.ops import kernels as K
        from dryft_b200.parts.base import Runtime

        if "w" in made:
            state["w"] = K.fp4_quantise(made["w"], case["kind"])
        if case["op"] == "product":
            state["rt"] = Runtime(dtype=_dtype(case["dtype"]), device=torch.device(DEVICE, torch.cuda.current_device()))
        return state
    if "w" in made:
        state["w"] = _quantise(made["w"], case["kind"])
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x, kind):
    """The held form: codes, two a byte, the groups' scales, the rows' factors (None for "mx")."""
    k, group = x.shape[-1], GROUP[kind]
    x = torch.nn.functional.pad(x.float(), (0, -k % group)).unflatten(-1, (-1, group))
    finite = x.isfinite()
    size = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    bad = ~finite.all(-1, keepdim=True)
    if kind == "mx":
        g = None
        # 2^floor(log2 size) is the number without its fraction's bits
        top = (size.view(torch.int32) & 0x7F800000).view(torch.float32)
        s = (top * 0.25).clamp(min=2.0**-127)
        y = x / s
    else:
        g = (size.amax(-2, keepdim=True) / torch.full_like(size[:, :1], 2688.0)).clamp(min=2.0**-112)
        u = torch.ones_like(g) / (6.0 * g)
        s = (size * u).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        r = torch.where(s > 0, torch.ones_like(s) / (s * g), torch.zeros_like(s))
        y = x * r
    a = y.abs()
    c = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()) | ((y < 0).byte() << 3)
    c = c.flatten(-2)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    return c[..., 0::2] | (c[..., 1::2] << 4), s.squeeze(-1), None if g is None else g.squeeze(-1), k


def _values(held, kind):
    """What it stands for, in 32 bits."""
    codes, s, g, k = held
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()].unflatten(-1, (-1, GROUP[kind])) * s[..., None]
    v = v.flatten(-2)[..., :k]
    return v if g is None else v * g


def _silu(gu, k):
    """The product of silu(gate), rounded to the activations' type, and what stands beside it, rounded to it too."""
    gate, up = gu[:, :k].float(), gu[:, k:].float()
    return ((gate / (1.0 + torch.exp(-gate))).to(gu.dtype).float() * up).to(gu.dtype)


def run(state):
    case = state["case"]
    kind, dtype = case["kind"], _dtype(case["dtype"])
    if own:
        return _run_own(state)
    if case["op"] == "values":
        return _values(state["w"], kind).to(dtype)
    x = state["x"]
    if case["op"] == "round":
        return _values(_quantise(x, kind), kind).to(dtype)
    if case["silu"]:
        x = _silu(x, case["k"])
    return (_values(_quantise(x, kind), kind) @ _values(state["w"], kind).T).to(_dtype(case["out"]))


# ------------------------------------------------------------------------------------------------ the framework's operators
def _run_own(state):
    from dryft_b200.ops import kernels as K
    from dryft_b200.parts.linear import linear

    case = state["case"]
    if case["op"] == "values":
        return K.fp4_expand(state["w"], out_dtype=_dtype(case["dtype"]))
    if case["op"] == "round":
        return K.fp4_expand(K.fp4_quantise(state["x"], case["kind"]), out_dtype=state["x"].dtype)
    if case["silu"]:
        return K.linear_fp4(state["x"], state["w"], silu=True, out_dtype=_dtype(case["out"]))
    return linear(state["x"], state["w"], state["rt"], out_dtype=_dtype(case["out"]))


# ------------------------------------------------------------------------------------------------ 64 bits
def _nearest(a, bits, least, most):
    """The nearest number of ``bits`` bits behind the leading one, exponents from ``least`` up, magnitude up to ``most``; ties to even.  In 64 bits."""
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (e - 1).clamp(min=least) - bits)
    return torch.round(a / step).mul(step).clamp(-most, most)


def _exact_values(x, kind):
    """The values that the 4-bit form of ``x`` stands for, in 64 bits.  Scales and codes are defined by 32-bit steps: each is worked out in
    64 bits and rounded to 32, which is the correctly rounded 32-bit result."""
    r = lambda t: t.to(torch.float32).double()  # noqa: E731
    rows, k = x.shape
    group = GROUP[kind]
    a = torch.zeros(rows, math.ceil(k / group) * group, dtype=torch.float64, device=x.device)
    a[:, :k] = x
    a = a.reshape(rows, -1, group)
    size = torch.nan_to_num(a.abs(), nan=0.0, posinf=0.0).amax(-1, keepdim=True)
    if kind == "mx":
        _, e = torch.frexp(size)
        s = torch.where(size > 0, torch.ldexp(torch.ones_like(size), (e - 3).clamp(min=-127)), torch.full_like(size, 2.0**-127))
        c, g = _nearest(a / s, 1, 0, 6.0), 1.0
    else:
        g = r(size.amax(1, keepdim=True) / 2688).clamp(min=2.0**-112)
        s = _nearest(r(size * r(1 / r(6 * g))), 3, -6, 448.0)
        c = _nearest(r(a * torch.where(s > 0, r(1 / r(s * g)), torch.zeros_like(s))), 1, 0, 6.0)
    v = torch.where(a.isfinite().all(-1, keepdim=True), c * s * g, torch.full_like(a, math.nan))
    return v.reshape(rows, -1)[:, :k]


def exact(case, seed):
    made = _inputs(case, seed)
    if case["op"] != "product":
        t = made["x"] if case["op"] == "round" else made["w"]
        step = max(1, 2**26 // case["k"])
        return torch.cat([_exact_values(t[i:i + step], case["kind"]) for i in range(0, t.shape[0], step)])
    x, k = made["x"], case["k"]
    if case["silu"]:
        gate = x[:, :k].double()
        x = ((gate * torch.sigmoid(gate)).to(x.dtype).double() * x[:, k:].double()).to(x.dtype)
    x, step = _exact_values(x, case["kind"]), max(1, 2**26 // k)
    return torch.cat([torch.einsum("mk,nk->mn", x, _exact_values(made["w"][i:i + step], case["kind"])) for i in range(0, case["n"], step)], 1)
