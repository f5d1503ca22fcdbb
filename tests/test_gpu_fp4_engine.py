"""The engine with its matrices in microscaled 4-bit floating point: every product of prompts and of single tokens against the definition on the inputs that it had; with and
without graphs and overlapped launches; through the command line; and what it refuses."""

import json

import pytest
import torch

import helpers as H
import plain_fp4 as F
import plain_qwen3 as P
from dryft_b200.ops import kernels as K

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
KINDS = ("mx", "nv")


def matrices(model_dir, cfg):
    """The matrices that a step multiplies by, in the order of its run: name -> [outputs, inputs] as the checkpoint has them."""
    t = P.read_model_dir(model_dir)[1]
    out = []
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        out.append(torch.cat([t[p + f"self_attn.{n}_proj.weight"] for n in "qkv"]))
        out.append(t[p + "self_attn.o_proj.weight"])
        out.append(torch.cat([t[p + "mlp.gate_proj.weight"], t[p + "mlp.up_proj.weight"]]))
        out.append(t[p + "mlp.down_proj.weight"])
    return out + [t.get("lm_head.weight", t["model.embed_tokens.weight"])]


class Recorded:
    """What every product of a step was given and gave."""

    def __init__(self, monkeypatch):
        self.calls, self.kept = [], K.linear_fp4

        def linear_fp4(x, w, *a, **kw):
            y = self.kept(x, w, *a, **kw)
            self.calls.append((x.clone(), w, kw.get("silu", False), y.clone()))
            return y

        monkeypatch.setattr(K, "linear_fp4", linear_fp4)

    def check(self, held, kind, dtype, layers):
        """The products of one step, each against the definition's on the inputs that it had: a step's own errors, and the border between two codes that a number lies on, are no
        part of that.  (Whole models cannot be compared: a number whose neighbour is taken moves its row by a hundredth, and every number behind it.)"""
        assert len(self.calls) == len(held) == 4 * layers + 1
        for i, ((x, w, silu, y), values) in enumerate(zip(self.calls, held)):
            assert silu == (i < 4 * layers and i % 4 == 3)
            x = x.cpu()
            if silu:
                x = F.silu_mul(x)
            assert torch.equal(K.fp4_expand(w, out_dtype=F32).cpu(), values.to(F32)) or kind == "nv"
            assert y.dtype == (F32 if i == 4 * layers else dtype)
            xv = F.values(x, kind)
            want, terms = xv @ values.T, xv.abs() @ values.abs().T
            # (as in the products' own test.  silu: its 32-bit function is 2^-20 off at the most, which takes one in 2^11 bfloat16 results to a neighbour, 2^-8 away, and one in ten of
            # those over a border between two codes, half a step of one of the row's largest numbers each: a thirtieth of the row's length covers eight at once)
            room = (torch.finfo(y.dtype).eps / 2 + 2.0**-22) * want.abs() + (w.k / 64 + 2) * 2.0**-21 * terms
            off = (y.double().cpu() - want).abs()
            if silu:
                lengths = xv.norm(dim=1, keepdim=True) * values.norm(dim=1)[None]
                assert bool((off <= room + lengths / 30).all()) and float((off <= room).double().mean()) > 0.9
            else:
                assert bool((off <= room).all()), f"product {i}: {float((off / room).max())} of what may be"
        self.calls.clear()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", ["a", "b", "c", "d"])
def test_products_of_prompts_and_of_single_tokens(model_dirs, monkeypatch, name, dtype, kind):
    from dryft_b200.engine.api import Engine

    eng = Engine(model_dirs[name], dtype=dtype, max_batch=4, max_seq_len=512, max_tokens=4 * 512, weight_bits=4, weight_format=kind, cuda_graphs=False)
    cfg = H.config_dict(name)
    held = [F.values(w.to(dtype), kind) for w in matrices(model_dirs[name], cfg)]
    seen = Recorded(monkeypatch)
    check = lambda: seen.check(held, kind, dtype, cfg["num_hidden_layers"])  # noqa: E731
    step = lambda slots, toks, want: eng.stepper.step(slots, toks, want)  # noqa: E731
    with torch.inference_mode():
        prompts = H.prompts_for(name, [100, 37, 170], seed=5)
        slots = eng.cache.open_sequences(3)
        step(slots, [p[:20] for p in prompts], [[19], [0, 1], [5]])
        check()
        step(slots, [prompts[0][20:90], prompts[1][20:30], prompts[2][20:160]], [[69], [9], list(range(139))])
        check()
        for i in range(2):
            step(slots, [[p[n + i]] for p, n in zip(prompts, (90, 30, 160))], [[0], [0], [0]])
            check()
        step(slots[:1], [[prompts[0][95]]], [[0]])
        check()
        eng.cache.close_sequences(slots)
    eng.cache.check()


@pytest.mark.parametrize("kind", KINDS)
def test_graphs_and_overlapped_launches_change_nothing(model_dirs, kind):
    """The same tokens and the same bits of logits with graphs or none, launches overlapped or not."""
    from dryft_b200.engine.api import Engine

    def run(**kw):
        eng = Engine(model_dirs["d"], max_batch=8, max_seq_len=256, weight_bits=4, weight_format=kind, **kw)
        prompts = H.prompts_for("d", [9, 40, 3, 77, 20], seed=2)
        tokens = eng.generate_many(prompts, 12)
        with torch.inference_mode():
            slots = eng.cache.open_sequences(5)
            eng.stepper.step(slots, prompts, [[], [], [], [], []])
            logits = [eng.stepper.step(slots, [[t] for t in range(7, 12)], [[0]] * 5).clone() for _ in range(4)]
        return tokens, torch.stack(logits)

    tokens, logits = run()
    for kw in (dict(cuda_graphs=False), dict(pdl=False), dict(cache_bits=16, cuda_graphs=False, pdl=False)):
        t, lg = run(**kw)
        assert t == tokens and torch.equal(lg, logits)


def test_with_a_cache_in_four_bits_and_from_the_command_line(model_dirs, capsys):
    from dryft_b200.cli import main
    from dryft_b200.engine.api import Engine

    eng = Engine(model_dirs["d"], max_batch=4, max_seq_len=128, weight_bits=4, weight_format="nv", cache_bits=4)
    prompts = [[1, 2, 3], [4, 5]]
    want = eng.generate_many(prompts, 8)
    whole = Engine(model_dirs["d"], max_batch=4, max_seq_len=128)
    matrices = sum(w.numel() for w in P.read_model_dir(model_dirs["d"])[1].values() if w.dim() == 2)
    table = 300 * 256
    assert whole.model.weight_bytes() - eng.model.weight_bytes() > 1.2 * (matrices - table)   # (16 bits - 4.5 bits - a row's factor - rows and inputs up to whole blocks)
    assert main(["generate", "--model", model_dirs["d"], "--max-batch", "4", "--max-seq-len", "128", "--weight-bits", "4", "--weight-format", "nv", "--cache-bits", "4",
                 "--prompt-ids", "1,2,3", "--prompt-ids", "4,5", "--max-new-tokens", "8"]) == 0
    assert [json.loads(line)["tokens"] for line in capsys.readouterr().out.splitlines()] == want


def test_refusals(model_dirs):
    from dryft_b200.config import preset
    from dryft_b200.engine.api import Engine

    for kw, word in ((dict(weight_bits=4, weight_format="fp8"), "fp8"), (dict(weight_format="nv"), "weight_bits=4"), (dict(cache_bits=4, weight_format="mx"), "weight_bits=4")):
        with pytest.raises(ValueError) as e:
            Engine(model_dirs["a"], max_batch=1, max_seq_len=64, **kw)
        assert word in str(e.value)
    with pytest.raises(ValueError) as e:
        Engine.from_config(preset("tevovik-tiny"), max_batch=1, max_seq_len=64, weight_bits=4, weight_format="nv")
    assert "not served" in str(e.value)
