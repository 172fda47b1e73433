"""A model whose cache is kept in 8 bits: the store, decode and prompt attention together, through the engine, against the plain model
with the same rounding of keys and values."""

import json
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.helpers import CONFIGS, model_folder, plain_weights, requests_for
from tests.plain import cache8 as plain8
from tests.plain import model as plain

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def plain_logits8(tag, tokens, mode, monkeypatch, keep8=True):
    """The plain model's logits with keys and values as the 8-bit cache gives them back."""
    attend = plain.causal_gqa_attention
    with monkeypatch.context() as patch:
        if keep8:
            patch.setattr(plain, "causal_gqa_attention", lambda q, k, v: attend(q, plain8.quantised(k), plain8.quantised(v)))
        if mode == "lowp":
            patch.setattr(plain, "LOWP", torch.bfloat16)
        return plain.forward(torch.tensor(tokens), plain_weights(tag), CONFIGS[tag], torch.float64 if mode == "f64" else torch.float32).double().cpu()


def engine8(tag, dtype, max_tokens, **options):
    from gtar_kimik3_public_b200.engine import Engine
    from gtar_kimik3_public_b200.generate import load

    engine = Engine(load(model_folder(tag), dtype, "cuda:0", cache_dtype="float8_e4m3fn"), max_tokens, **options)
    for group in engine.cache.kv_groups:  # every place poisoned
        group.k.view(torch.uint8).fill_(0x7F)
        group.v.view(torch.uint8).fill_(0x7F)
        group.k_exp.fill_(255)
        group.v_exp.fill_(255)
    return engine


def replay(engine, requests, prompt_cuts):
    """Each request's tokens in pieces, all requests in the same steps, then the rest one by one; logits of every token."""
    from gtar_kimik3_public_b200.engine import StepEntry

    at, rows = [0] * len(requests), [[] for _ in requests]
    pieces = [list(cuts) + [1] * (len(r) - sum(cuts)) for r, cuts in zip(requests, prompt_cuts)]
    for step in range(max(len(p) for p in pieces)):
        live = [i for i, p in enumerate(pieces) if step < len(p)]
        entries = [StepEntry(i, requests[i][at[i]:at[i] + pieces[i][step]], list(range(pieces[i][step]))) for i in live]
        logits = engine.step(entries)
        row = 0
        for i in live:
            n = pieces[i][step]
            rows[i].append(logits[row:row + n].double().cpu())
            at[i], row = at[i] + n, row + n
    engine.check()
    engine.end_all()
    return [torch.cat(r) for r in rows]


LENGTHS, CUTS = [70, 100, 12], [(63,), (40, 3, 50), (1, 8)]


@pytest.mark.parametrize("tag,dtype", [("tiny_a", "float32"), ("tiny_c", "float32"), ("tiny_b", "bfloat16"), ("tiny_c", "bfloat16")])
@pytest.mark.parametrize("graphs", [True, False])
def test_engine_steps(tag, dtype, graphs, monkeypatch):
    requests = requests_for(tag, LENGTHS, seed=3)
    got = replay(engine8(tag, dtype, 64 * 8, max_seqs=4, use_graphs=graphs), requests, CUTS)
    for tokens, logits in zip(requests, got):
        oracle = plain_logits8(tag, tokens, "f64", monkeypatch)
        err = (logits - oracle).abs().max().item()
        if dtype == "float32":
            # 1e-4 as for the 16-bit cache, and room for a few keys or values that lie between two 8-bit numbers and go the other way: four of some
            # ten thousand roundings move the logits by a thirtieth of what all of them do
            moved = (oracle - plain_logits8(tag, tokens, "f64", monkeypatch, keep8=False)).abs().max().item()
            assert err < 1e-4 + 0.1 * moved
        else:
            standard = (plain_logits8(tag, tokens, "lowp", monkeypatch) - oracle).abs().max().item()
            assert err <= 2 * standard + 1e-4, f"{err:.3e} against {standard:.3e}"


def test_float32_steps_do_not_depend_on_the_cut():
    requests = requests_for("tiny_b", LENGTHS, seed=4)
    engine = engine8("tiny_b", "float32", 64 * 8, max_seqs=4)
    whole = replay(engine, requests, [(n,) for n in LENGTHS])
    for cuts in (CUTS, [(), (64,), (5,)]):
        assert all(torch.equal(a, b) for a, b in zip(whole, replay(engine, requests, cuts)))


def test_generation_and_command_line(tmp_path, monkeypatch):
    from gtar_kimik3_public_b200 import generate as api

    tag = "tiny_c"
    prompts = requests_for(tag, [5, 66, 1], seed=21)
    model = api.load(model_folder(tag), "bfloat16", cache_dtype="float8_e4m3fn")
    got = api.generate(model, prompts, max_new_tokens=12, temperature=0.0)
    for prompt, tokens in zip(prompts, got):
        oracle = plain_logits8(tag, prompt + tokens, "f64", monkeypatch)
        standard = (plain_logits8(tag, prompt + tokens, "lowp", monkeypatch) - oracle).abs().max().item()
        for i, token in enumerate(tokens):
            row = oracle[len(prompt) - 1 + i]
            assert row[token] >= row.max() - 2 * (2 * standard + 1e-4)
    command = [sys.executable, "-m", "gtar_kimik3_public_b200.scripts.generate", "--model", str(model_folder(tag)), "--cache-dtype", "float8_e4m3fn",
               "--prompt-ids", ",".join(map(str, prompts[0])), "--max-new-tokens", "12", "--temperature", "0"]
    shown = subprocess.run(command, capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert shown.returncode == 0, shown.stderr
    assert shown.stdout.splitlines()[0] == ",".join(map(str, got[0]))


def test_trace_run(tmp_path, monkeypatch):
    tag = "tiny_c"
    tokens = requests_for(tag, [80], seed=31)[0]
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": tokens[:70], "want": [69]}]}]
    steps += [{"step": i + 1, "entries": [{"id": "a", "tokens": [tokens[70 + i]], "want": [0]}]} for i in range(10)]
    command = [sys.executable, str(ROOT / "bin" / "trace_run"), "--model", str(model_folder(tag)), "--dtype", "bfloat16", "--cache-dtype", "float8_e4m3fn",
               "--out", str(tmp_path), "--max-tokens", "128"]
    done = subprocess.run(command, input="".join(json.dumps(s) + "\n" for s in steps), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    oracle = plain_logits8(tag, tokens, "f64", monkeypatch)[69:]
    standard = (plain_logits8(tag, tokens, "lowp", monkeypatch)[69:] - oracle).abs().max().item()
    got = torch.stack([torch.from_numpy(np.fromfile(tmp_path / f"{i}.f32", dtype="<f4")) for i in range(11)])
    assert (got.double() - oracle).abs().max().item() <= 2 * standard + 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_an_attention_layer_with_a_window(dtype, d, monkeypatch):
    """Pages go back to the pool as the window leaves them and are used again by another sequence; prompts, pieces and single tokens."""
    from dataclasses import replace

    from gtar_kimik3_public_b200.cache import Cache, CacheLayout
    from gtar_kimik3_public_b200.engine.step import SequenceStep, plan_step
    from gtar_kimik3_public_b200.parts import build_part
    from tests.test_gpu_kernels import DEV, rand
    from tests.test_gpu_parts import load_part

    hidden, n_q, n_kv, window, eps, theta, n = 96, 4, 2, 70, 1e-5, 1e4, 260
    rope = build_part("position", "rope", dim=d, base=theta)
    mixer = build_part("mixer", "gqa_attention", hidden_size=hidden, n_q_heads=n_q, n_kv_heads=n_kv, head_dim=d, qk_norm_eps=eps, position=rope, window=window)
    w = {"q_proj.weight": rand(n_q * d, hidden, seed=1, scale=0.1), "k_proj.weight": rand(n_kv * d, hidden, seed=2, scale=0.1),
         "v_proj.weight": rand(n_kv * d, hidden, seed=3, scale=0.1), "o_proj.weight": rand(hidden, n_q * d, seed=4, scale=0.1),
         "q_norm.weight": 1 + 0.1 * rand(d, seed=5), "k_norm.weight": 1 + 0.1 * rand(d, seed=6)}
    w = {k: v.to(torch.bfloat16).double() if "proj" in k else v.float().double() for k, v in w.items()}
    load_part(mixer, w, dtype)
    rope.prepare(n, torch.device(DEV))
    request = replace(mixer.cache_request(), dtype=torch.float8_e4m3fn)
    cache = Cache(CacheLayout([request]), 64 * 9, dtype, DEV, max_seqs=2)
    group, = cache.kv_groups
    for t in (group.k, group.v):
        t.view(torch.uint8).fill_(0x7F)
    group.k_exp.fill_(255)
    group.v_exp.fill_(255)
    xs = [rand(n, hidden, seed=7 + i).to(dtype) for i in range(2)]
    slots, at, rows = [cache.open(), cache.open()], [0, 0], [[], []]
    pieces = [[100, 3, 64] + [1] * 93, [1] * 90 + [33, 70] + [1] * 67]
    for step in range(max(map(len, pieces))):
        live = [i for i in range(2) if step < len(pieces[i])]
        sequences = [SequenceStep(slots[i], cache.grow(slots[i], pieces[i][step]), [0] * pieces[i][step], []) for i in live]
        cache.sync()
        ctx = plan_step(sequences, dtype, torch.device(DEV), 1)
        x = torch.cat([xs[i][at[i]:at[i] + pieces[i][step]] for i in live]).to(DEV)
        out, row = mixer.forward(x, ctx, cache.view(0)).double().cpu(), 0
        for i in live:
            m = pieces[i][step]
            rows[i].append(out[row:row + m])
            at[i], row = at[i] + m, row + m
    cache.check_invariants()
    assert len(group.owned[slots[0]]) <= 3  # what the window has left went back
    cfg = {"num_attention_heads": n_q, "num_key_value_heads": n_kv, "head_dim": d, "rms_norm_eps": eps, "rope_theta": theta}
    attend = plain.causal_gqa_attention

    def wanted(x, keep8, lowp):
        with monkeypatch.context() as patch:
            as_kept = plain8.quantised if keep8 else (lambda t: t)
            patch.setattr(plain, "causal_gqa_attention", lambda q, k, v: attend(q, as_kept(k), as_kept(v), window))
            if lowp:
                patch.setattr(plain, "LOWP", torch.bfloat16)
                return plain.attention_mixer(x.float(), {k: v.float() for k, v in w.items()}, "", cfg).double()
            return plain.attention_mixer(x.double(), w, "", cfg)

    for i in range(2):
        got, oracle = torch.cat(rows[i]), wanted(xs[i], True, False)
        assert got.shape[0] == sum(pieces[i]) and torch.isfinite(got).all()
        oracle = oracle[: got.shape[0]]
        err = (got - oracle).abs().max().item()
        if dtype == torch.float32:  # as for whole models: a few roundings that lie between two numbers
            moved = (oracle - wanted(xs[i], False, False)[: got.shape[0]]).abs().max().item()
            assert err < 1e-4 + 0.1 * moved
        else:
            standard = (wanted(xs[i], True, True)[: got.shape[0]] - oracle).abs().max().item()
            assert err <= 2 * standard + 1e-4
