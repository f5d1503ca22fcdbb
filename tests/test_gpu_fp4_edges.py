"""Microscaled 4-bit floating point on the GPU at the edges of what its calls allow: gates whose exponential nearly overflows, rows of any size against rows of any other, stages
that end anywhere in a ring, calls that fail, what captured calls and repeated ones choose, and what an engine holds."""

import pytest
import torch

import helpers as H
import plain_fp4 as P
import plain_qwen3
from dryft_b200.ops import kernels as K
from test_gpu_fp4 import near, rows_of

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
KINDS = ("mx", "nv")


def test_silu_of_every_gate():
    """All bfloat16 numbers: within one rounding to bfloat16 (2^-8, or half the smallest number) and the 32-bit function's own error (2^-15, see below) of the definition down to -88.5;
    zero below, where the 32-bit power is infinite; NaN for NaN and for minus infinity."""
    g = torch.arange(65536, device="cuda").to(torch.int32).to(torch.int16).view(BF)
    got = torch.empty(1, 65536, dtype=BF, device="cuda")
    K.silu_mul(torch.cat([g, torch.ones_like(g)])[None], got)
    x, got = g.double().cpu(), got[0].double().cpu()
    want = x * torch.sigmoid(x)
    assert torch.equal(got.isnan(), want.isnan()) and bool((got[x < -88.75] == 0)[x[x < -88.75] > -float("inf")].all())
    near_ = (x >= -88.75) & x.isfinite()
    assert int(near_.sum()) > 48000 and bool(((got - want).abs() <= (2.0**-8 + 2.0**-15) * want.abs() + 2.0**-134)[near_].all())
    assert float(got[x == float("inf")]) == float("inf")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [2, 40])
def test_gates_whose_exponential_is_nearly_too_large(kind, m):
    """1 + exp(-g) between 2^126 and the largest 32-bit number: silu(g) is a bfloat16 number like any other, and counts where what it is multiplied by is large.  Two roundings to
    bfloat16 (2^-8 each, at most), an exponential of 2 + 1.173 |g| ulp at most (106: 2^-16.2) and a division of two."""
    k, n = 256, 200
    gate = torch.arange(-88.5, -85.75, 0.5, device="cuda").repeat(m * k)[:m * k].view(m, k)
    up = torch.randn(m, k, device="cuda") * 2.0**118
    x = torch.cat([gate, up], 1).to(BF)
    assert float(x[:, :k].float().min()) == -88.5
    want = (x[:, :k].double() * torch.sigmoid(x[:, :k].double()) * x[:, k:].double())
    act = torch.empty(m, k, dtype=BF, device="cuda")
    K.silu_mul(x, act)
    assert bool(((act.double() - want).abs() <= (2 * 2.0**-8 + 2.0**-15) * want.abs()).all())
    w = rows_of(n, k, BF)
    q = K.fp4_quantise(w, kind)
    got = K.linear_fp4(x, q, silu=True)
    assert torch.equal(got, K.linear_fp4(act, q))
    near(got, act, w, kind, k)
    # rows of an odd width, which silu_mul takes number by number: at most two of them have a neighbour's code somewhere (as in the test of silu in front)
    odd = torch.cat([x[:, :k - 1], x[:, k:2 * k - 1]], 1)
    act = torch.empty(m, k - 1, dtype=BF, device="cuda")
    K.silu_mul(odd, act)
    q = K.fp4_quantise(w[:, :k - 1], kind)
    got, want = K.linear_fp4(odd, q, silu=True), K.linear_fp4(act, q)
    assert int((got != want).any(1).sum()) <= 2 and bool(((got.float() - want.float()).norm(dim=1) <= 0.5 * want.float().norm(dim=1)).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [16, 100, 300])
def test_stages_that_end_anywhere_in_a_ring(monkeypatch, kind, m):
    """Fewer inputs than a ring of stages holds, as many, and more; one tile and several to a block."""
    n = 700
    for k in (100, 600, 1100, 1300, 1700, 2100, 2900):
        x, w = rows_of(m, k, BF), rows_of(n, k, BF)
        q, h = K.fp4_quantise(w, kind), K.fp4_quantise(x, kind)
        want, terms = P.product(x, w, kind)
        room = (k / 64 + 10) * 2.0**-21 * terms + 2.0**-22 * want.abs()
        plans = [(next(b for b in (16, 32, 64, 128) if m <= b or b == 128), blocks, 1) for blocks in (1, 2, 5)]
        plans += [(nb, blocks, 0) for nb in (128, 192, 256) for blocks in (2, 4) if m > 16]
        for plan in plans:
            monkeypatch.setattr(K, "linear_fp4_plan", lambda *a: plan)
            for operand in (h, x):
                y = K.linear_fp4(operand, q, out_dtype=F32)
                assert bool(((y.double().cpu() - want).abs() <= room).all()), (k, plan)
    K.check_error_flags()


class Launchers:
    """The two launchers of linear_fp4, with what they were asked and, where wanted, an answer of their own."""

    def __init__(self, monkeypatch, rc=None):
        lib = K.fp4_lib()
        self.asked, self.rc, self.real = [], rc, (lib.dryft_linear_fp4, lib.dryft_linear_fp4_rows)
        monkeypatch.setattr(K, "_fp4_calls", (self.of_held, self.of_rows))

    def of_held(self, *a):
        self.asked.append(("held", int(a[13])))
        return self.real[0](*a) if self.rc is None else self.rc

    def of_rows(self, *a):
        self.asked.append(("within" if not a[15] else "apart", int(a[17])))
        return self.real[1](*a) if self.rc is None else self.rc


@pytest.mark.parametrize("kind", KINDS)
def test_the_first_product_of_a_weight_overlaps_nothing(monkeypatch, kind):
    """Asked to overlap the launch before them, products ask for a weight before that has ended: not so the first one of a weight, whose launch before may be what wrote it."""
    v, x = rows_of(300, 512, BF), rows_of(1, 512, BF)
    held, seen = K.fp4_quantise(x, kind), Launchers(monkeypatch)
    for operand in (held, x):
        q = K.fp4_quantise(v, kind)
        results = [K.linear_fp4(operand, q, pdl=True) for _ in range(3)]
        assert [p for _, p in seen.asked] == [0, 1, 1] and {f for f, _ in seen.asked} == {"held" if operand is held else "within"}
        assert all(torch.equal(r, results[0]) for r in results)
        seen.asked.clear()
    # rows that a launch of their own rounds: that one waits for all before itself, and the product is its dependent
    q = K.fp4_quantise(v, kind)
    wide = rows_of(60, 512, BF)
    K.linear_fp4(wide, q, pdl=True), K.linear_fp4(wide, q), K.linear_fp4(wide, q, pdl=False), K.linear_fp4(x, q), K.linear_fp4(x, q, pdl=False)
    assert seen.asked == [("apart", 3), ("apart", 2), ("apart", 0), ("within", 0), ("within", 0)]


@pytest.mark.parametrize("kind", KINDS)
def test_a_product_that_failed_is_not_a_weights_first_one(monkeypatch, kind):
    v, x, wide = rows_of(300, 512, BF), rows_of(1, 512, BF), rows_of(60, 512, BF)
    for operand in (x, wide, K.fp4_quantise(x, kind)):
        q = K.fp4_quantise(v, kind)
        failing = Launchers(monkeypatch, K.UNSUPPORTED)
        with pytest.raises(K.KernelError):
            K.linear_fp4(operand, q, pdl=True)
        assert len(failing.asked) == 1 and not q.read
        seen = Launchers(monkeypatch)
        K.linear_fp4(operand, q, pdl=True)
        assert seen.asked[0][1] == (3 if operand is wide else 0) and q.read
    # no memory for the rounded rows
    q = K.fp4_quantise(v, kind)
    monkeypatch.setattr(K, "_fp4_shape", lambda *a: (1 << 20, 1 << 20, 1 << 20))
    with pytest.raises(RuntimeError):
        K.linear_fp4(wide, q, pdl=True)
    assert not q.read


def test_a_weights_first_product_on_every_stream_overlaps_nothing(monkeypatch):
    """A product that ran on another stream, behind an event there, says nothing about the launch before this one: it may still be the weight's rounding.  Captured products go by whether
    any has run: a weight's rounding is not in front of them unless it is captured too, and then none has."""
    v, x = rows_of(300, 512, BF), rows_of(1, 512, BF)
    for operand in (x, K.fp4_quantise(x, "nv")):
        q, other = K.fp4_quantise(v, "nv"), torch.cuda.Stream()
        seen = Launchers(monkeypatch)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            results = [K.linear_fp4(operand, q, pdl=True) for _ in range(2)]
        results += [K.linear_fp4(operand, q[:], pdl=True) for _ in range(2)]
        assert [p for _, p in seen.asked] == [0, 1, 0, 1]
        torch.cuda.synchronize()
        assert all(torch.equal(r, results[0]) for r in results)
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = K.linear_fp4(K.fp4_quantise(x, "nv"), q, pdl=True)
        g.replay()
        torch.cuda.synchronize()
        assert seen.asked[-1] == ("held", 1) and torch.equal(y, results[0])


def test_a_row_range_is_its_matrixs_memory(monkeypatch):
    """What was written with the whole matrix: a product with a range of its rows is a first one only where none of that matrix was before it."""
    v, x = rows_of(300, 512, BF), rows_of(1, 512, BF)
    q = K.fp4_quantise(v, "nv")
    seen = Launchers(monkeypatch)
    K.linear_fp4(x, q[128:], pdl=True), K.linear_fp4(x, q[:200], pdl=True), K.linear_fp4(x, q, pdl=True), K.linear_fp4(x, q[128:][:100], pdl=True)
    assert [p for _, p in seen.asked] == [0, 1, 1, 1]


def test_a_replay_leaves_the_error_flag_as_it_is(monkeypatch):
    """Where the first product of a process is captured, its flag is not the graph's: what a wait that gave up has left there stays until somebody reads it."""
    v, x = rows_of(300, 512, BF), rows_of(3, 512, BF)
    K.linear_fp4(x, K.fp4_quantise(v, "nv"))     # (loads the kernels)
    monkeypatch.setattr(K, "_error_flags", {})
    q, s, g = K.fp4_quantise(v, "nv"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        y = K.linear_fp4(x, q)
    flag = K.error_flag(x.device)
    flag.fill_(305)
    g.replay()
    torch.cuda.synchronize()
    assert flag.tolist() == [305] and torch.equal(y, K.linear_fp4(x, q))


@pytest.mark.parametrize("kind", KINDS)
def test_a_layer_that_reads_anothers_cache(monkeypatch, kind):
    """Its queries are a product with a range of its matrix's rows, which is taken once, not at every step; every product against the definition on the inputs that it had."""
    from dryft_b200.config import register_architecture, unregister_architecture
    from dryft_b200.config.spec import LayerSpec, ModelSpec, PartSpec, RunStep
    from dryft_b200.engine.api import Engine

    class Shared:
        def __init__(self, raw):
            self.raw = dict(raw)

        def to_dict(self):
            return dict(self.raw)

        def model_spec(self):
            norm = PartSpec("rmsnorm", {"size": 64, "eps": 1e-6})
            attn = PartSpec("attention", {"hidden_size": 64, "num_heads": 5, "num_kv_heads": 5, "head_dim": 32, "scale": 32 ** -0.5, "window": None,
                                          "qk_norm": PartSpec("rmsnorm", {"size": 32, "eps": 1e-6}), "position": PartSpec("rope", {"rotary_dim": 32, "theta": 1e4})})
            ffn = PartSpec("swiglu", {"hidden_size": 64, "intermediate_size": 96})
            layers = tuple(LayerSpec("prenorm", attn, ffn, norm, norm, f"l{i}.attn.", f"l{i}.ffn.", f"l{i}.n1.", f"l{i}.n2.") for i in range(2))
            return ModelSpec("SharedForCausalLM", 211, 64, 512, PartSpec("embedding", {"vocab_size": 211, "hidden_size": 64}), layers, (RunStep(0), RunStep(1, cache_from=0)), norm,
                             PartSpec("lm_head", {"vocab_size": 211, "hidden_size": 64, "tied": True}), embedding_prefix="emb.", final_norm_prefix="fn.", head_prefix="head.")

    register_architecture("SharedForCausalLM", Shared)
    try:
        eng = Engine.from_config({"architectures": ["SharedForCausalLM"], "hidden_size": 64, "vocab_size": 211}, seed=5, std=0.15, dtype="bfloat16", max_batch=1, max_seq_len=64,
                                 weight_bits=4, weight_format=kind, cuda_graphs=False)
        kept, calls, made, look = K.linear_fp4, [], [], K.Fp4.__post_init__

        def linear_fp4(x, w, *a, **kw):
            y = kept(x, w, *a, **kw)
            calls.append((x.clone(), w, kw.get("silu", False), y.clone()))
            return y

        monkeypatch.setattr(K, "linear_fp4", linear_fp4)
        monkeypatch.setattr(K.Fp4, "__post_init__", lambda self: (made.append(self), look(self))[1])
        with torch.inference_mode():
            slots = eng.cache.open_sequences(1)
            eng.stepper.step(slots, [[1, 2, 3, 4, 5]], [[4]])
            eng.stepper.step(slots, [[6]], [[0]])
        assert not made
        assert [c[1].n for c in calls] == 2 * [480, 64, 192, 64, 160, 64, 192, 64, 211]
        for x, w, silu, y in calls:
            x = P.silu_mul(x.cpu()) if silu else x
            xv, wv = P.values(x, kind), K.fp4_expand(w, out_dtype=F32).double().cpu()
            want, terms = xv @ wv.T, xv.abs() @ wv.abs().T
            room = (torch.finfo(y.dtype).eps / 2 + 2.0**-22) * want.abs() + (w.k / 64 + 2) * 2.0**-21 * terms
            if silu:   # (as in the engine's own test: codes' borders)
                room = room + xv.norm(dim=1, keepdim=True) * wv.norm(dim=1)[None] / 30
            assert bool(((y.double().cpu() - want).abs() <= room).all())
    finally:
        unregister_architecture("SharedForCausalLM")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("silu", [False, True])
def test_where_captured_calls_round(monkeypatch, kind, silu):
    """With silu a captured call goes by the limits of captured ones wherever its launches may overlap, not only where it may overlap the launch before it; without silu only there.
    Launches that run in turn go by the eager limits.  The bits are the same."""
    n, k = 640, 2560
    q = K.fp4_quantise(rows_of(n, k, BF), kind)
    xs = [rows_of(m, 2 * k if silu else k, BF) for m in (1, 2, 3, 4, 6, 8, 11, 16)]
    seen, forms = Launchers(monkeypatch), {}
    want = [K.linear_fp4(x, q, silu=silu) for x in xs]
    eager = [f for f, _ in seen.asked]
    seen.asked.clear()
    for pdl in (True, None, False):
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            got = [K.linear_fp4(x, q, silu=silu, pdl=pdl) for x in xs]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        forms[pdl] = [f for f, _ in seen.asked]
        seen.asked.clear()
    assert forms[True] != eager or (kind == "mx" and not silu)       # (of these sizes)
    assert forms[None] == (forms[True] if silu else eager) and forms[False] == eager
    K.check_error_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,plan", [(1, None), (4, None), (40, None), (140, (128, 6, 1)), (140, (128, 12, 2)), (140, (128, 4, 0))])
def test_large_rows_against_small_ones(monkeypatch, kind, m, plan):
    """Rows of every size as weights against rows of every size as activations: where a sum of the terms' magnitudes is far from both ends of 32 bits, so is the result."""
    k, n = 512, 300
    if plan:
        monkeypatch.setattr(K, "linear_fp4_plan", lambda *a: plan)
    sizes = [1e-37, 1e-34, 1e-30, 1e-20, 1e-6, 1.0, 1e6, 1e20, 1e30, 1e34, 4e37]
    w = (torch.randn(n, k, device="cuda") * torch.tensor(sizes, device="cuda").repeat(n // 11 + 1)[:n, None]).to(BF)
    q = K.fp4_quantise(w, kind)
    for i in range(0, 11, m if m < 11 else 11):
        x = (torch.randn(m, k, device="cuda") * torch.tensor(sizes[i:] + sizes[:i], device="cuda").repeat(m // 11 + 1)[:m, None]).to(BF)
        got = K.linear_fp4(x, q, out_dtype=F32)
        want, terms = P.product(x, w, kind)
        fits = terms < 2.0**126                       # (of the rest no 32-bit sum need be a number)
        assert float(fits.double().mean()) > 0.2
        # (as in the test of rare rows; numbers below the smallest normal one may be taken for zeros)
        room = 2.0**-21 * want.abs() + (k / 64 + 2) * 2.0**-21 * terms + (k / 64 + 1) * 2.0**-126
        off = (got.double().cpu() - want).abs()
        assert bool((off <= room)[fits].all()), ((~(off <= room)) & fits).nonzero()[:8].tolist()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", ["b", "d"])
def test_an_engine_holds_what_the_definition_says(model_dirs, monkeypatch, name, dtype, kind):
    """Codes, scales and factors of every matrix: the definition's values rounded to 32 bits once, which is what (c s) g comes to."""
    from dryft_b200.engine.api import Engine

    eng = Engine(model_dirs[name], dtype=dtype, max_batch=1, max_seq_len=64, weight_bits=4, weight_format=kind, cuda_graphs=False)
    t, cfg, used, kept = plain_qwen3.read_model_dir(model_dirs[name])[1], H.config_dict(name), [], K.linear_fp4

    def linear_fp4(x, w, *a, **kw):
        used.append(w)
        return kept(x, w, *a, **kw)

    monkeypatch.setattr(K, "linear_fp4", linear_fp4)
    with torch.inference_mode():
        eng.stepper.step(eng.cache.open_sequences(1), [[1, 2, 3]], [[2]])
    want = []
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        for parts in (["self_attn.q", "self_attn.k", "self_attn.v"], ["self_attn.o"], ["mlp.gate", "mlp.up"], ["mlp.down"]):
            want.append(torch.cat([t[p + part + "_proj.weight"] for part in parts]))
    want.append(t.get("lm_head.weight", t["model.embed_tokens.weight"]))
    assert len(used) == len(want)
    for w, v in zip(used, want):
        assert torch.equal(K.fp4_expand(w, out_dtype=F32).cpu(), P.values(v.to(dtype), kind).to(F32))
