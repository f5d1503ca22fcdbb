"""The engine with its matrices and its cache in 4 bits: against the plain implementation fed the values that the codes stand for, however the tokens are
cut into steps; through the entry point and the command line; and what it refuses."""

import json

import pytest
import torch

import helpers as H
import plain_four_bit as F
import plain_qwen3 as P

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _group(size):
    return max(g for g in (16, 32, 64) if size % g == 0)


class Plain(P.PlainQwen3):
    """The plain model with its matrices replaced by what their 4-bit form stands for, in the model's own precision: its bfloat16 evaluation has bfloat16
    weights (as the products of many rows have; those of few rows do not round them).  ``logits(ids, held)``: attention reads the keys and values ``held``
    (one pair of [tokens, kv heads, d] a layer) instead of the layer's own, which ``made`` has afterwards."""

    def __init__(self, cfg, tensors, dtype, weights):
        tensors = dict(tensors)
        if cfg["tie_word_embeddings"]:
            cfg = dict(cfg, tie_word_embeddings=False)
            tensors["lm_head.weight"] = tensors["model.embed_tokens.weight"]
        super().__init__(cfg, tensors, dtype)
        if weights:
            for name, t in self.t.items():
                if t.dim() == 2 and "embed" not in name:
                    self.t[name] = F.group_values(t, _group(t.shape[1]))[0].to(F32).to(dtype)

    def logits(self, ids, held=None):
        kept, self.made = P.causal_attention, []

        def attention(q, k, v, *a):
            self.made.append((k, v))
            k, v = held[len(self.made) - 1] if held else (k, v)
            return kept(q, k, v, *a)

        P.causal_attention = attention
        try:
            return super().logits(ids)
        finally:
            P.causal_attention = kept


def _models(model_dirs, name, weights):
    cfg, tensors = P.read_model_dir(model_dirs[name])
    return {dt: Plain(cfg, tensors, dt, weights) for dt in (F32, BF)}


def _held(eng, slot, n):
    """What the engine's cache stands for: the keys and values of a sequence's first ``n`` tokens, layer by layer."""
    from dryft_b200.ops import kernels as K

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    out = []
    for i in range(len(eng.spec.schedule)):
        e = eng.cache.entry(i)
        if e.scratch is None:
            return None
        k, v = (torch.zeros_like(t, dtype=F32) for t in e.scratch)
        K.kv4_expand(e.k, e.v, e.page_table, i32([0, 1]), i32([slot]), i32([n - 1]), k, v, eng.model.blocks[eng.spec.schedule[i].layer].mixer.bits_group, n)
        pages = e.page_table[slot, :(n + 63) // 64].long()
        out.append(tuple(t[pages].transpose(1, 2).flatten(0, 1)[:n].cpu() for t in (k, v)))
    return out


def _check(eng, slot, got, plain, tokens, rows, dtype, what):
    """Logits are the plain model's that reads the same keys and values; and (32 bits) what the cache holds is as near to the plain model's own keys and
    values as codes can be: half a step, 1/30 of the group's range, beside what rounding s and z to bfloat16 moves (2^-8 of 7.5 s and of z).  A number
    of the engine's may differ from the plain model's in its last bits, and then fall on the other side of a rounding: the bound holds on either side."""
    n = len(tokens)
    held = _held(eng, slot, n)
    want, p32 = plain[dtype].logits(tokens, held)[rows], plain[F32].logits(tokens, held)[rows]
    tol = H.FP32_TOL if dtype == F32 else H.bf16_tol(want, p32)
    e = H.rel_err(got.float().cpu(), want)
    assert e <= tol, f"{what}: logits off by {e:.3g} (allowed {tol:.3g})"
    if dtype == F32 and held and plain[F32].windows[-1] is None:
        for layer, (made, mine) in enumerate(zip(plain[F32].made, held)):
            for x, y in zip(made, mine):
                _, s, z = F.group_values(x, _group(x.shape[-1]))
                far = (x.double() - y.double()).abs() - (0.5 * s + 2.0**-8 * (7.5 * s + z.abs()) + 1e-4 * x.abs().max())
                assert far.max() <= 0, f"{what}: layer {layer} holds a number off by {float(far.max()):.3g} more than half a step"


@pytest.mark.parametrize("bits", [(4, 16), (16, 4), (4, 4)])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", ["a", "b", "c", "d"])
def test_logits_whole_in_pieces_and_token_by_token(model_dirs, name, dtype, bits):
    from dryft_b200.engine.api import Engine

    eng = Engine(model_dirs[name], dtype=dtype, max_batch=4, max_seq_len=512, max_tokens=4 * 512, weight_bits=bits[0], cache_bits=bits[1])
    plain = _models(model_dirs, name, bits[0] == 4)
    step = lambda slots, toks, want: eng.stepper.step(slots, toks, want)
    with torch.inference_mode():
        for n in (1, 17, 64, 150):
            toks = H.prompts_for(name, [n], seed=n)[0]
            (slot,) = eng.cache.open_sequences(1)
            _check(eng, slot, step([slot], [toks], [list(range(n))]), plain, toks, list(range(n)), dtype, f"{name} whole, {n} tokens")
            eng.cache.close_sequences([slot])
        # three sequences of unequal lengths side by side, in pieces, then token by token
        prompts = H.prompts_for(name, [100, 37, 70], seed=5)
        slots = eng.cache.open_sequences(3)
        step(slots, [p[:20] for p in prompts], [[], [], []])
        got = step(slots, [prompts[0][20:90], prompts[1][20:30], prompts[2][20:60]], [[69], [9], [39]])
        for b, (p, n) in enumerate(zip(prompts, (90, 30, 60))):
            _check(eng, slots[b], got[b:b + 1], plain, p[:n], [n - 1], dtype, f"{name} in pieces, sequence {b}")
        for i in range(7):
            got = step(slots, [[prompts[0][90 + i]], [prompts[1][30 + i]], [prompts[2][60 + i]]], [[0], [0], [0]])
            for b, (p, n) in enumerate(zip(prompts, (90, 30, 60))):
                _check(eng, slots[b], got[b:b + 1], plain, p[:n + i + 1], [n + i], dtype, f"{name} token by token, sequence {b}")
        eng.cache.close_sequences(slots)
    eng.cache.check()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_prompts_replayed_from_a_graph(model_dirs, dtype):
    """The third step of a shape is a replay: lengths are data there, longer ones than the captured step had too."""
    from dryft_b200.engine.api import Engine

    eng = Engine(model_dirs["d"], dtype=dtype, max_batch=2, max_seq_len=512, max_tokens=1024, weight_bits=4, cache_bits=4)
    plain = _models(model_dirs, "d", True)
    toks = H.prompts_for("d", [512], seed=1)[0]
    with torch.inference_mode():
        for start in (0, 0, 0, 256):
            (slot,) = eng.cache.open_sequences(1)
            if start:
                eng.stepper.step([slot], [toks[:start]], [[]])
            got = eng.stepper.step([slot], [toks[start:start + 256]], [[255]])
            _check(eng, slot, got, plain, toks[:start + 256], [start + 255], dtype, f"from {start}")
            eng.cache.close_sequences([slot])
    assert eng.stepper._prompt_graphs


def test_generation_through_the_entry_point_and_the_command_line(model_dirs, capsys):
    """Greedy tokens in 32 bits are the plain model's; graphs or none, the same ones; the command prints them."""
    from dryft_b200.cli import main
    from dryft_b200.engine.api import Engine

    prompts = H.prompts_for("d", [9, 70, 23], seed=3)
    cfg, tensors = P.read_model_dir(model_dirs["d"])
    want = P.plain_generate(Plain(cfg, tensors, F32, True), prompts, 10)
    for graphs in (True, False):
        eng = Engine(model_dirs["d"], dtype="float32", max_batch=4, max_seq_len=128, weight_bits=4, cuda_graphs=graphs)
        assert eng.generate_many(prompts, 10) == want
    eng = Engine(model_dirs["d"], max_batch=4, max_seq_len=128, weight_bits=4, cache_bits=4)
    tokens = eng.generate_many(prompts, 10)
    assert eng.generate_many(prompts, 10) == tokens
    whole = Engine(model_dirs["d"], max_batch=4, max_seq_len=128)
    assert eng.model.weight_bytes() < whole.model.weight_bytes() and eng.cache.bytes() < whole.cache.bytes()
    assert main(["generate", "--model", model_dirs["d"], "--max-batch", "4", "--max-seq-len", "128", "--weight-bits", "4", "--cache-bits", "4",
                 "--max-new-tokens", "10"] + [a for p in prompts for a in ("--prompt-ids", ",".join(map(str, p)))]) == 0
    assert [json.loads(line)["tokens"] for line in capsys.readouterr().out.splitlines()] == tokens


def test_what_is_refused(model_dirs):
    from dryft_b200.config import preset
    from dryft_b200.engine.api import Engine

    for kw, word in ((dict(weight_bits=8), "8 bits"), (dict(cache_bits=2), "2 bits"), (dict(weight_bits=4, bits_group=48), "48")):
        with pytest.raises(ValueError, match=word):
            Engine(model_dirs["a"], max_batch=2, max_seq_len=64, **kw)
    for kw in (dict(weight_bits=4), dict(cache_bits=4)):
        with pytest.raises(ValueError, match="not served"):
            Engine.from_config(preset("tevovik-tiny"), max_batch=2, max_seq_len=64, **kw)


@pytest.mark.parametrize("n_seqs", [1, 3, 8, 24])
def test_decode_at_production_widths_is_the_same_with_and_without_launch_overlap(n_seqs):
    """Two layers 2,560 wide: a decode step whose launches overlap gives bit for bit the logits of the same launches one after the other, with norms, sums and
    activations in the products (up to four rows) and as launches, on the kernels for few rows and for many; and, with the weights alone in 4 bits, stays within
    bfloat16 rounding of the path of separate kernels."""
    from dryft_b200.config import preset
    from dryft_b200.engine.api import Engine

    raw = dict(preset("qwen3-4b"))
    raw.update(num_hidden_layers=2, vocab_size=8192, max_position_embeddings=2048)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 8192, (n,), generator=g).tolist() for n in ((70, 3, 129, 64, 200, 17, 31, 90, 5, 250, 33, 128) * 2)[:n_seqs]]

    def decode_logits(dtype="bfloat16", **opts):
        eng = Engine.from_config(raw, seed=4, std=0.03, max_batch=32, max_seq_len=1024, max_tokens=16 * 1024, dtype=dtype, weight_bits=4, **opts)
        outs = []
        with torch.inference_mode():
            s = eng.cache.open_sequences(len(prompts))
            lg = eng.stepper.step(s, prompts, [[len(p) - 1] for p in prompts])
            idx = torch.tensor(s, device="cuda")
            for _ in range(5):
                eng.cache.last_token[idx] = (torch.arange(len(prompts), device="cuda") * 37 + len(outs) * 11).int() % 8192
                lg = eng.stepper.decode_from_state(s)[: len(prompts)].float()
                outs.append(lg.cpu())
            eng.cache.close_sequences(s)
        del eng
        torch.cuda.empty_cache()
        return torch.stack(outs)

    overlapped = decode_logits(cache_bits=4)
    assert torch.equal(overlapped, decode_logits(cache_bits=4, cuda_graphs=False)) and torch.equal(overlapped, decode_logits(cache_bits=4, pdl=False))
    fused, separate, exact = decode_logits(), decode_logits(fuse_decode=False), decode_logits("float32")
    tol = H.bf16_tol(separate, exact)
    assert H.rel_err(fused, separate) <= tol and H.rel_err(fused, exact) <= tol
