"""Steps of several tokens over an 8-bit cache through the engine: the same bits whether a step is met for the first time, run for its capture or replayed, and
whatever lengths the cache could hold."""

import pytest
import torch

from gtar_kimik3_public_b200.registry import config_from_dict
from tests.helpers import requests_for
from tests.tiny_configs import TINY_LONG

pytestmark = pytest.mark.gpu

CONFIGS = {"heads of 64": TINY_LONG,
           "heads of 128": {**TINY_LONG, "num_attention_heads": 32, "num_key_value_heads": 8, "head_dim": 128, "num_hidden_layers": 1}}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from gtar_kimik3_public_b200.weights import write_random_model

    out = {}
    for name, config in CONFIGS.items():
        out[name] = tmp_path_factory.mktemp("model")
        write_random_model(out[name], config_from_dict(config), 0, std=0.08)
    return out


# tokens of a step that come behind tokens of an earlier one, a request each
SHAPES = {"a prompt of 64": ([0], [64]), "a prompt of 128": ([0], [128]), "a prompt of 700": ([0], [700]), "sixteen times sixteen": ([60 + 9 * i for i in range(16)], [16] * 16),
          "a few guesses": ([400, 30, 9], [4, 4, 3])}


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("shape", list(SHAPES))
def test_a_step_gives_the_same_bits_whenever_it_comes(name, shape, folders):
    from gtar_kimik3_public_b200.engine import Engine, StepEntry
    from gtar_kimik3_public_b200.generate import load

    past, new = SHAPES[shape]
    requests = requests_for("tiny_long", [p + n for p, n in zip(past, new)], seed=5)
    model = load(folders[name], "bfloat16", "cuda:0", cache_dtype="float8_e4m3fn")
    got = []
    for room in (64 * 80, 64 * 202):  # sequences of 5,120 tokens and of 12,928
        engine = Engine(model, room, max_seqs=16)
        assert engine.cache.max_seq_len == room
        for _ in range(4):
            for i, (r, p) in enumerate(zip(requests, past)):
                if p:  # each by itself, in a step of its own shape
                    engine.step([StepEntry(i, r[:p])])
            got.append(engine.step([StepEntry(i, r[p:], list(range(len(r) - p))) for i, (r, p) in enumerate(zip(requests, past))]).clone())
            engine.check()
            engine.end_all()
    assert all(torch.equal(g, got[0]) for g in got), [(g - got[0]).abs().max().item() for g in got]
