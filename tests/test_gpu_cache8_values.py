"""Values of very unlike sizes that do not share their columns: what a column holds is what its own numbers make it, however large another column's are."""

import pytest
import torch

from tests.test_gpu_cache8 import DEV, F, SEVERAL, SINGLE, check_attention, empty_pages, fill, held, ints, rand

pytestmark = pytest.mark.gpu


def lone(n, n_kv, d, power, at, seed=2):
    """Ordinary rows, but for one that holds 2^power in a column and zeros, and one of 2^-power beside it."""
    v = rand(n, n_kv, d, seed=seed)
    v[at] = 0
    v[at, :, 5] = 2.0**power
    v[at + 1] *= 2.0**-min(power, 40)
    v[:at, :, 5] = 0
    v[at + 1:, :, 5] = 0
    return v


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n_q,n_kv", [(4, 2), (16, 1)])
@pytest.mark.parametrize("cut", [(1, 0), (4, 0), (0, 40)])
@pytest.mark.parametrize("power", [12, 24, 100])
@pytest.mark.parametrize("n,at", [(300, 3), (300, 290), (1500, 700)])
def test_decode(d, n_q, n_kv, cut, power, n, at):
    kv, slots, table = empty_pages(1, n, n_kv, d)
    fill(kv, table, int(slots[0]), rand(n, n_kv, d, seed=1), lone(n, n_kv, d, power, at))
    q = rand(1, n_q, d, seed=5).to(torch.bfloat16)
    got = F().attention_decode8(q.to(DEV), kv, ints(n), slots, n, d**-0.5, cut=cut)
    k, v = held(kv, table, int(slots[0]), n)
    check_attention(got, q, k, v, n - 1, 0, False, SINGLE[torch.bfloat16], "one token")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("power", [12, 24, 100])
@pytest.mark.parametrize("at", [3, 296])
def test_several_tokens(d, few, window, power, at, monkeypatch):
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: few)
    n, m, n_q, n_kv = 300, 7, 8, 2
    kv, slots, table = empty_pages(1, n, n_kv, d)
    fill(kv, table, int(slots[0]), rand(n, n_kv, d, seed=1), lone(n, n_kv, d, power, at))
    q = rand(m, n_q, d, seed=5).to(torch.bfloat16)
    got = F().attention_prefill8(q.to(DEV), kv, ints(0, m), ints(n), slots, m, n, d**-0.5, window)
    k, v = held(kv, table, int(slots[0]), n)
    check_attention(got, q, k, v, n - m, window, False, SEVERAL[torch.bfloat16], "several tokens")
