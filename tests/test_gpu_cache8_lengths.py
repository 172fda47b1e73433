"""Several tokens a sequence over 8-bit pages where a sequence's numbers cannot be: fewer positions than tokens, none, a length below zero or beyond the
bound.  Reported; tokens in front of the first position see no key and are zeros, the others and the step's other sequences are what they are."""

import pytest
import torch

from tests.test_gpu_cache8 import DEV, F, SEVERAL, check_attention, held, ints, rand, sequences

pytestmark = pytest.mark.gpu


@pytest.fixture
def way(request, monkeypatch):
    """Through the kernel for few rows, through clean pages, or through the kernel for any size."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: request.param == "few")
    return torch.float32 if request.param == "any" else torch.bfloat16


@pytest.fixture
def dealt(request):
    """How the tcgen05 prefill kernels deal out their tiles: (blocks that stay, one tile a block, keys a step)."""
    from gtar_kimik3_public_b200.ops.library import library

    stay, one, keys = request.param
    before = (library().gk_set_attention_prefill_stay(stay), library().gk_set_attention_prefill_one_tile(one), library().gk_set_attention_prefill_keys(keys))
    yield
    library().gk_set_attention_prefill_stay(before[0])
    library().gk_set_attention_prefill_one_tile(before[1])
    library().gk_set_attention_prefill_keys(before[2])


def check_lengths(dtype, d, window, sink, new, lens, wrong, given, bound):
    """Sequence ``wrong`` is given the length ``given``; the longest length is said to be ``bound``."""
    n_q, n_kv = 4, 2
    kv, slots, table = sequences(lens, n_kv, d)
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    q = rand(cu[-1], n_q, d, seed=5).to(dtype)
    said = list(lens)
    said[wrong] = given
    f = F()
    good = f.attention_prefill8(q.to(DEV), kv, ints(*cu), ints(*lens), slots, max(new), max(lens), d**-0.5, window, sink)
    f.check_kernel_errors(DEV)
    out = torch.full(q.shape, 5.0, dtype=dtype, device=DEV)
    f.attention_prefill8(q.to(DEV), kv, ints(*cu), ints(*said), slots, max(new), bound, d**-0.5, window, sink, out)
    with pytest.raises(f.KernelError, match="length"):
        f.check_kernel_errors(DEV)
    for i in range(len(new)):
        here = slice(cu[i], cu[i + 1])
        if i != wrong:
            assert torch.equal(out[here], good[here]), f"sequence {i}"
            continue
        length = max(0, min(given, -(-bound // 64) * 64))
        blind = max(0, new[i] - length)
        assert (out[here][:blind] == 0).all(), "tokens in front of position 0"
        if blind < new[i]:
            k, v = held(kv, table, int(slots[i]), lens[i])
            check_attention(out[here][blind:], q[here][blind:], k[:length], v[:length], length - (new[i] - blind), window, sink, SEVERAL[dtype], "the rest")


# new tokens, true lengths, which is wrong, what it is said to be, the bound on lengths
WRONG = [([70, 1, 40], [200, 64, 40], 0, 0, 200),      # no positions, 70 tokens
         ([70, 1, 40], [200, 64, 40], 0, -7, 200),     # less than none
         ([70, 1, 40], [200, 64, 40], 0, 33, 200),     # tokens in front of position 0 and behind it in one tile
         ([300, 5], [300, 90], 0, 100, 300),           # whole tiles in front of position 0
         ([5, 300], [90, 300], 1, 1, 300),
         ([300, 5], [300, 60], 0, 300, 64)]            # a bound that is too small


@pytest.mark.parametrize("way", ["clean"], indirect=True)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sink", [(0, False), (40, True)])
@pytest.mark.parametrize("new,lens,wrong,given,bound", WRONG)
def test_fewer_positions_than_tokens(way, d, window, sink, new, lens, wrong, given, bound):
    check_lengths(way, d, window, sink, new, lens, wrong, given, bound)


@pytest.mark.parametrize("way", ["clean"], indirect=True)
@pytest.mark.parametrize("dealt", [(1, 1, 128), (0, 1, 128), (0, 0, 128), (0, 0, 64)], indirect=True)
@pytest.mark.parametrize("new,lens,wrong,given,bound", WRONG)
def test_fewer_positions_than_tokens_in_every_prefill_kernel(way, dealt, new, lens, wrong, given, bound):
    check_lengths(way, 128, 0, False, new, lens, wrong, given, bound)


@pytest.mark.parametrize("way", ["few", "any"], indirect=True)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sink", [(0, False), (40, True)])
@pytest.mark.parametrize("new,lens,wrong,given,bound", WRONG[:-1])  # (a bound is no more than a hint to these kernels)
def test_fewer_positions_than_tokens_without_clean_pages(way, d, window, sink, new, lens, wrong, given, bound):
    check_lengths(way, d, window, sink, new, lens, wrong, given, bound)


@pytest.mark.parametrize("way", ["few", "clean", "any"], indirect=True)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cut", [(2, 0), (0, 40)])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 40])
@pytest.mark.parametrize("new,lens,wrong,given,bound", WRONG[:-1])
def test_the_largest_windows_in_front_of_position_0(way, d, cut, window, new, lens, wrong, given, bound, monkeypatch):
    """A position below zero less the largest window would leave 32 bits: as if there were no window."""
    monkeypatch.setattr(F(), "rows8_cut", lambda *sizes: cut)
    check_lengths(way, d, window, False, new, lens, wrong, given, bound)


@pytest.mark.parametrize("way", ["clean"], indirect=True)
@pytest.mark.parametrize("dealt", [(1, 1, 128), (0, 1, 128), (0, 0, 128), (0, 0, 64)], indirect=True)
@pytest.mark.parametrize("new,lens,wrong,given,bound", WRONG)
def test_the_largest_window_in_every_prefill_kernel(way, dealt, new, lens, wrong, given, bound):
    check_lengths(way, 128, 2**31 - 1, False, new, lens, wrong, given, bound)


@pytest.mark.parametrize("way", ["few", "clean"], indirect=True)
@pytest.mark.parametrize("d", [64, 128])
def test_more_tokens_than_max_q_len(way, d):
    """Reported whichever kernel takes them; the step's other sequences are what they are."""
    kv, slots, _ = sequences([300, 90], 2, d)
    q = rand(275, 4, d, seed=5).to(way).to(DEV)
    args = (kv, ints(0, 270, 275), ints(300, 90), slots)
    good = F().attention_prefill8(q, *args, 270, 300, d**-0.5)
    F().check_kernel_errors(DEV)
    for most in (0, 2, 100, 269):
        got = F().attention_prefill8(q, *args, most, 300, d**-0.5)
        with pytest.raises(F().KernelError, match="length"):
            F().check_kernel_errors(DEV)
        if most >= 5:
            assert torch.equal(got[270:], good[270:])


@pytest.mark.parametrize("way", ["clean"], indirect=True)
@pytest.mark.parametrize("d", [64, 128])
def test_a_window_over_more_tokens_than_max_q_len(way, d):
    """What the launch covers of such a sequence, its last tile, sees clean pages: the window goes back from the sequence's own first token."""
    n_q, n_kv, new, n, window = 4, 2, 200, 271, 10
    kv, slots, table = sequences([n], n_kv, d)
    q = rand(new, n_q, d, seed=5).to(way)
    # the memory that the call will take for its pages holds NaN
    poison = torch.full((2, -(-n // 64), n_kv, 64, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    del poison
    out = torch.full(q.shape, 5.0, dtype=way, device=DEV)
    F().attention_prefill8(q.to(DEV), kv, ints(0, new), ints(n), slots, 2, n, d**-0.5, window, False, out)
    with pytest.raises(F().KernelError, match="length"):
        F().check_kernel_errors(DEV)
    k, v = held(kv, table, int(slots[0]), n)
    check_attention(out[-8:], q[-8:], k, v, n - 8, window, False, SEVERAL[way], "the last tokens")


@pytest.mark.parametrize("way", ["few", "clean", "any"], indirect=True)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("past,pages", [(73, 1), (74, 1), (137, 2)])
def test_pages_that_the_window_has_left_are_not_looked_at(way, d, past, pages):
    """Up to the page whose last position is the one right in front of the window: no page number stands for them any more."""
    window, new, n_q, n_kv = 10, 5, 4, 2
    kv, slots, table = sequences([past + new, 30], n_kv, d)
    kv.block_table[slots[0].long(), :pages] = -1
    q = rand(new + 2, n_q, d, seed=5).to(way)
    got = F().attention_prefill8(q.to(DEV), kv, ints(0, new, new + 2), ints(past + new, 30), slots, new, past + new, d**-0.5, window)
    F().check_kernel_errors(DEV)
    for i, (at, m, n) in enumerate([(0, new, past + new), (new, 2, 30)]):
        k, v = held(kv, table, int(slots[i]), n)
        check_attention(got[at:at + m], q[at:at + m], k, v, n - m, window, False, SEVERAL[way], f"sequence {i}")
