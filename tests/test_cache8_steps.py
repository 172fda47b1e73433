"""Steps of several tokens over an 8-bit cache, on the host: the bound on lengths that a captured step is made for, and that what is chosen by a step's true
lengths is what is chosen by the bound that stands for them."""

from types import SimpleNamespace

import pytest
import torch

from gtar_kimik3_public_b200.cache import Cache, CacheLayout
from gtar_kimik3_public_b200.engine.graphs import StepGraphs
from gtar_kimik3_public_b200.engine.step import SequenceStep, pack_step
from gtar_kimik3_public_b200.ops.functional import length_class, prompt8_length
from gtar_kimik3_public_b200.parts.base import KVRequest, RowsRequest, StateRequest

E4 = torch.float8_e4m3fn


def cache_of(*requests, longest=40960):
    return Cache(CacheLayout(list(requests)), longest, torch.bfloat16, "cpu", max_seqs=4, max_seq_len=longest)


def graphs_over(cache):
    graphs = object.__new__(StepGraphs)
    graphs.cache, graphs.events = cache, []
    return graphs


def prompt(past, n):
    return pack_step([SequenceStep(0, past, [1] * n, [n - 1])], 10)


def test_which_caches_keep_8_bits():
    assert cache_of(KVRequest(2, 64, dtype=E4)).keeps_8_bits and cache_of(StateRequest((3,)), KVRequest(2, 64, window=100, dtype=E4)).keeps_8_bits
    assert not cache_of(KVRequest(2, 64)).keeps_8_bits and not cache_of(RowsRequest(64), StateRequest((3,))).keeps_8_bits


def test_length_classes():
    """1, 1.5, 2, 3, 4, ... times the least."""
    assert [length_class(n, 256) for n in (0, 1, 256, 257, 384, 385, 512, 513, 768, 1025)] == [
        (0, 256), (0, 256), (0, 256), (256, 384), (256, 384), (384, 512), (384, 512), (512, 768), (512, 768), (1024, 1536)]
    for n in list(range(1, 5000, 7)) + [40000, 1 << 20, 2**31 - 1]:
        below, bound = length_class(n, 256)
        assert below < n <= bound and bound <= max(256, 2 * n) and length_class(bound, 256) == (below, bound)


@pytest.mark.parametrize("past,n,bound", [(0, 2, 256), (0, 128, 256), (0, 300, 384), (1000, 64, 1536), (0, 2048, 2048), (39000, 1000, 40960)])
def test_captured_prompts_are_made_for_lengths_like_theirs(past, n, bound):
    packed = prompt(past, n)
    small, plain = graphs_over(cache_of(KVRequest(2, 64, dtype=E4))), graphs_over(cache_of(KVRequest(2, 64)))
    assert small.launch_bounds(packed) == (bound, 0) and small.key_of(packed) == (n, 1, 1, n, bound)
    assert plain.launch_bounds(packed) == (40960, 0) and plain.key_of(packed) == (n, 1, 1, n, 0)  # as ever
    assert packed.max_kv_len <= small.launch_bounds(packed)[0] <= 40960


def test_single_tokens_are_bounded_as_ever():
    single = pack_step([SequenceStep(0, 1500, [1], [0]), SequenceStep(1, 3, [1], [0])], 10)
    for cache in (cache_of(KVRequest(2, 64, dtype=E4)), cache_of(KVRequest(2, 64))):
        graphs = graphs_over(cache)
        assert graphs.launch_bounds(single) == graphs.length_bounds(single) == (1536, 1280) and graphs.key_of(single) == (2, 2, 2, 1, 1536)


@pytest.mark.parametrize("longest", [512, 4096, 12928, 40960])
def test_a_step_takes_the_same_kernel_whenever_it_comes(longest):
    """By its own lengths, as when it is first met, or by the bound, as when it is captured."""
    graphs = graphs_over(cache_of(KVRequest(8, 128, dtype=E4), longest=longest))
    for new, past in [(64, 0), (128, 0), (300, 0), (2048, 0), (16, 300), (4, 2000), (32, 100), (512, 2000), (3, 12000)]:
        if past + new > longest:
            continue
        packed = SimpleNamespace(all_single=False, max_kv_len=past + new, max_q_len=new)
        own, bounded = (prompt8_length(length, new) for length in (past + new, graphs.launch_bounds(packed)[0]))
        assert own == bounded >= new
    for window in (16, 700, 2**31 - 1):
        assert prompt8_length(3000, 40, window) == min(prompt8_length(3000, 40), window + 40)
