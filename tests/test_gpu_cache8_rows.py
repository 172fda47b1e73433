"""Rows on their way into the 8-bit cache that are not ordinary ones, in every kernel that writes: few tokens, many, any head size, and the decode kernel that
writes its own token.  Each key is the formula in 64 bits rounded once."""

import pytest
import torch

from tests.plain import cache8 as plain8
from tests.plain import model as plain
from tests.test_gpu_cache8 import DEV, F, SINGLE, check_attention, empty_pages, fill, held, ints, rand

pytestmark = pytest.mark.gpu

WAYS = ["few", "many", "decode"]


def written(way, qkv, n_q, n_kv, d, eps, weight, cos, sin, positions):
    """Keys and values ``[n, n_kv, d]`` as the cache holds them after the rows of ``qkv`` were written, one a sequence at ``positions``: by the write of few
    tokens, by that of many (the same rows as often as it takes), or by the decode kernel."""
    n = qkv.shape[0]
    kv, slots, table = empty_pages(n, max(positions) + 1, n_kv, d)
    table_args = [None if t is None else t.to(DEV) for t in (weight, weight, cos, sin)]
    how = (*table_args[:2], eps, *table_args[2:])
    if way == "decode":
        for t in (kv.k, kv.v):  # places before the new one: zeros under some power
            t.view(torch.uint8).zero_()
        kv.k_exp.fill_(127)
        kv.v_exp.fill_(127)
        F().attention_decode8_fused(qkv.to(DEV), n_q, n_kv, d, *how, kv, ints(*[p + 1 for p in positions]), slots, max(positions), max(positions) + 1, 0.1)
    else:
        times = 1 if way == "few" else -(-(7 << 20) // (n * (n_q + 2 * n_kv) * d))
        tokens = [i for _ in range(times) for i in range(n)]  # (the same row to the same place: whichever comes last)
        F().qk_norm_rope_write8(qkv[tokens].to(DEV), n_q, n_kv, d, *how, ints(*[positions[i] for i in tokens]), ints(*tokens), slots, kv, max(positions))
    F().check_kernel_errors(DEV)
    rows = [held(kv, table, int(slots[i]), p + 1) for i, p in enumerate(positions)]
    return [torch.stack([r[j][-1] for r in rows]) for j in (0, 1)]


def formula(x, weight, eps, cos, sin, positions):
    """RMSNorm and rotation of keys ``[n, n_kv, d]`` in 64 bits."""
    x = x.double()
    if weight is not None:
        x = plain.rms_norm(x, weight.double(), eps)
    if cos is not None:
        c, s = (torch.cat([t, t], -1).double()[positions] for t in (cos, sin))
        x = plain.apply_rotary(x, c, s)
    return x


def tables(positions, d):
    cos, sin = plain.rotary_tables(torch.arange(positions), d, 1e4)
    return cos[:, : d // 2].float().contiguous(), sin[:, : d // 2].float().contiguous()


def equal(got, want, what):
    want = plain8.quantised(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)), what


@pytest.mark.parametrize("way,d", [(w, d) for w in WAYS for d in (64, 128)] + [("few", 32), ("few", 80)])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_normed_rows_of_any_size(way, d, eps):
    """Rows of 2^-110 to 2^126: their squares leave 32 bits on both sides, their norm does not."""
    powers = [-110, -70, -64, -30, 0, 40, 62, 63, 64, 80, 100, 126]
    n, n_q, n_kv = len(powers), 2, 2
    keys = rand(n, n_kv, d, seed=1).clamp(-1.9, 1.9) * torch.tensor([2.0**p for p in powers], dtype=torch.float64).view(-1, 1, 1)
    keys[5, 0, 1:] = 0  # one number alone
    keys[7, 1, : d - 1] *= 2.0**-60  # and one far above the others
    qkv = torch.cat([rand(n, n_q, d, seed=2), keys, rand(n, n_kv, d, seed=3)], 1).to(torch.bfloat16)
    weight = (1 + 0.1 * rand(d, seed=4)).float()
    positions = [3 * i for i in range(n)]
    cos, sin = tables(40, d)
    got, values = written(way, qkv.view(n, -1), n_q, n_kv, d, eps, weight, cos, sin, positions)
    equal(got, formula(qkv[:, n_q:n_q + n_kv], weight, eps, cos, sin, positions), "keys")
    equal(values, qkv[:, n_q + n_kv:].double(), "values")


@pytest.mark.parametrize("way,d", [(w, d) for w in WAYS for d in (64, 128)] + [("few", 32)])
def test_rotated_rows_beyond_the_largest_number(way, d):
    """Two numbers near the largest whose rotation mixes them to more than 32 bits hold: the largest number that the cache holds, as the formula's is."""
    n, n_q, n_kv = 6, 2, 1
    keys = torch.full((n, n_kv, d), 3.3e38, dtype=torch.float64)
    keys[1::2, :, : d // 2] *= -1
    qkv = torch.cat([rand(n, n_q, d, seed=2), keys, rand(n, n_kv, d, seed=3)], 1).to(torch.bfloat16)
    positions = [0, 1, 2, 3, 4, 5]
    cos, sin = tables(6, d)
    got, _ = written(way, qkv.view(n, -1), n_q, n_kv, d, 1e-6, None, cos, sin, positions)
    want = formula(qkv[:, n_q:n_q + n_kv], None, 0.0, cos, sin, positions)
    assert (want.abs() > 3.5e38).any()
    equal(got, want, "keys")


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("norm", [True, False])
def test_keys_next_to_borders(way, d, norm):
    """Every number of a key within some tens of 2^-23 of itself of the middle between two 8-bit numbers, on either side, by the choice of the norm's weights
    or of the rotation's table.  What separates the two sides is what 32 bits lose in a dozen roundings."""
    n, n_q, n_kv, half = 48, 1, 1, d // 2
    gen = torch.Generator().manual_seed(11)
    keys = (torch.randn((n, 1, d), generator=gen, dtype=torch.float64)).to(torch.bfloat16)
    keys = torch.where(keys == 0, torch.ones_like(keys), keys)
    middle = (2 * torch.randint(8, 16, (n, d), generator=gen).double() + 1) / 16  # between m/8 and (m + 1)/8
    middle = middle * 2.0 ** torch.randint(-5, 8, (n, d), generator=gen).double()
    middle[:, 0] = 400.0  # every row's power is that of a maximum of 448 at most and more than 224
    off = torch.randint(-40, 41, (n, d), generator=gen).double() * 2.0**-23
    target = middle * (1 + off)
    positions = list(range(n))
    if norm:
        # one row's weights are another's noise: each row is a call of its own
        weight, cos, sin, eps = None, None, None, 1e-6
        got, want = [], []
        for i in range(0, n, 8):
            x = keys[i, 0].double()
            unit = x / torch.sqrt((x * x).mean() + eps)
            weight = (target[i] / unit).float()
            qkv = torch.cat([keys[i], keys[i], keys[i]]).to(torch.bfloat16).view(1, -1)
            got.append(written(way, qkv, n_q, n_kv, d, eps, weight, None, None, [0])[0])
            want.append(formula(keys[i:i + 1], weight, eps, None, None, [0]))
        got, want = torch.cat(got), torch.cat(want)
    else:
        # c and s so that the first number of a pair comes out next to its middle: u c - v s = target
        u, v = keys[:, 0, :half].double(), keys[:, 0, half:].double()
        sin = (0.5 * torch.randn((n, half), generator=gen, dtype=torch.float64)).float()
        cos = ((target[:, :half] + v * sin.double()) / u).float()
        qkv = torch.cat([keys, keys, keys], 1).view(n, -1)
        got, _ = written(way, qkv, n_q, n_kv, d, 1e-6, None, cos.contiguous(), sin.contiguous(), positions)
        want = formula(keys, None, 0.0, cos, sin, positions)
    equal(got, want, "keys")


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (6, 2, 64)])
def test_a_position_outside_the_rotation_s_table(n_q, n_kv, d):
    """The decode kernel leaves such a token's key where it was, writes its value and reports it, as the write by itself does; the others are what they are."""
    lens = [65, 40, 90]
    cos, sin = (t.to(DEV) for t in tables(64, d))
    qkv = rand(3, (n_q + 2 * n_kv) * d, seed=7).to(torch.bfloat16).to(DEV)
    w = (1 + 0.1 * rand(d, seed=20)).float().to(DEV)
    pages = []
    for fused in (True, False):
        kv, slots, table = empty_pages(3, max(lens), n_kv, d)
        if fused:
            F().attention_decode8_fused(qkv, n_q, n_kv, d, w, w, 1e-6, cos, sin, kv, ints(*lens), slots, 63, max(lens), 0.1)
        else:
            F().qk_norm_rope_write8(qkv, n_q, n_kv, d, w, w, 1e-6, cos, sin, ints(*[m - 1 for m in lens]), ints(0, 1, 2), slots, kv, 63)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        pages.append(kv)
        k, _ = held(kv, table, int(slots[0]), 65)
        assert torch.isnan(k[64]).all()  # the poison
    for name in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(getattr(pages[0], name).view(torch.uint8), getattr(pages[1], name).view(torch.uint8)), name


@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("cut", [(1, 0), (4, 0), (0, 40)])
def test_queries_of_the_decode_kernel(n_q, n_kv, d, cut):
    """Scores of some tens from queries that the kernel norms and rotates: they are rounded to halves, 2^-11 of each number, so a score may be off by 2^-11
    of the sum of its products' sizes, and a probability by twice that of itself (once in the sum below it); 32-bit arithmetic in front of it loses 2^-20."""
    lens, eps = [300, 64, 777], 1e-6
    kv, slots, table = empty_pages(3, max(lens), n_kv, d)
    for i, m in enumerate(lens):
        fill(kv, table, int(slots[i]), rand(m - 1, n_kv, d, seed=30 + i, scale=3.0), rand(m - 1, n_kv, d, seed=60 + i))
    qkv = rand(3, (n_q + 2 * n_kv) * d, seed=7).to(torch.bfloat16)
    w = (3 + 0.3 * rand(d, seed=20)).float()
    cos, sin = tables(max(lens), d)
    got = F().attention_decode8_fused(qkv.to(DEV), n_q, n_kv, d, w.to(DEV), w.to(DEV), eps, cos.to(DEV), sin.to(DEV), kv, ints(*lens), slots, max(lens) - 1,
                                      max(lens), d**-0.5, cut=cut)
    F().check_kernel_errors(DEV)
    x = formula(qkv.view(3, -1, d)[:, :n_q], w, eps, cos, sin, [m - 1 for m in lens])
    for i, m in enumerate(lens):
        k, v = held(kv, table, int(slots[i]), m)
        sizes = torch.einsum("hd,jhd->hj", x[i].abs(), k.abs().repeat_interleave(n_q // n_kv, 1)) * d**-0.5
        off = (2.0**-11 + 2.0**-20) * sizes.max().item()
        assert off < 0.2
        check_attention(got[i:i + 1], x[i:i + 1], k, v, m - 1, 0, False, SINGLE[torch.bfloat16] + torch.expm1(torch.tensor(2 * off)).item(), f"sequence of {m}")


@pytest.mark.parametrize("d", [64, 128])
def test_a_layer_whose_norm_weights_begin_anywhere(d):
    """Weights that begin between sixteen bytes: the decode kernel that norms refuses them, and a layer takes the write and the attention instead."""
    from types import SimpleNamespace

    from gtar_kimik3_public_b200.parts import build_part

    n_q, n_kv, lens = 4, 2, [70, 5]
    mixer = build_part("mixer", "gqa_attention", hidden_size=64, n_q_heads=n_q, n_kv_heads=n_kv, head_dim=d, qk_norm_eps=1e-6, position=None)
    both = (1 + 0.1 * rand(2 * d + 3, seed=4)).to(torch.bfloat16).to(DEV)
    mixer.q_norm, mixer.k_norm = both[1:d + 1], both[d + 3:2 * d + 3]
    qkv = rand(2, (n_q + 2 * n_kv) * d, seed=7).to(torch.bfloat16).to(DEV)
    got = []
    for layer in (True, False):
        kv, slots, table = empty_pages(2, max(lens), n_kv, d)
        for i, m in enumerate(lens):
            fill(kv, table, int(slots[i]), rand(m - 1, n_kv, d, seed=30 + i), rand(m - 1, n_kv, d, seed=60 + i))
        at, seq, kv_len = ints(*[m - 1 for m in lens]), ints(0, 1), ints(*lens)
        if layer:
            with pytest.raises(F().KernelError, match="16-byte"):
                F().attention_decode8_fused(qkv, n_q, n_kv, d, mixer.q_norm, mixer.k_norm, 1e-6, None, None, kv, kv_len, slots, 69, 70, d**-0.5)
            ctx = SimpleNamespace(all_single=True, tok_pos=at, tok_seq=seq, kv_len=kv_len, slots=slots, max_position=69, max_kv_len=70, typical_kv_len=0)
            got.append(mixer._attend(qkv, ctx, kv, None, None, True))
        else:
            q = F().qk_norm_rope_write8(qkv, n_q, n_kv, d, mixer.q_norm, mixer.k_norm, 1e-6, None, None, at, seq, slots, kv, 69)
            got.append(F().attention_decode8(q, kv, kv_len, slots, 70, d**-0.5))
    F().check_kernel_errors(DEV)
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_the_decode_kernel_writes_the_same_bytes(d, eps):
    """Rows of zeros, of zeros but for a number, of far and ordinary sizes, of infinities and NaN, with and without signs: as the write by itself."""
    n, n_q, n_kv = 12, 2, 2
    keys = rand(n, n_kv, d, seed=1)
    keys[0] = 0
    keys[1] = -0.0
    keys[2, :, 1:] = 0
    keys[3, :, ::2] = -0.0
    for i, power in enumerate((-100, -65, 62, 64, 100)):
        keys[4 + i] *= 2.0**power
        keys[4 + i, :, ::3] = -0.0
    keys[9, 0, 5], keys[9, 1, 7] = float("inf"), float("nan")
    keys[10, :, 3] = 2.0**70
    keys[11] *= 2.0**-24
    qkv = torch.cat([rand(n, n_q, d, seed=2), keys, rand(n, n_kv, d, seed=3)], 1).to(torch.bfloat16).view(n, -1).to(DEV)
    w = (1 + 0.1 * rand(d, seed=4)).float()
    w[::5] *= -1
    cos, sin = (t.to(DEV) for t in tables(40, d))
    positions, pages = [3 * i for i in range(n)], []
    for fused in (True, False):
        kv, slots, _ = empty_pages(n, 40, n_kv, d)
        how = (w.to(DEV), w.to(DEV), eps, cos, sin)
        if fused:
            F().attention_decode8_fused(qkv, n_q, n_kv, d, *how, kv, ints(*[p + 1 for p in positions]), slots, max(positions), 40, 0.1)
        else:
            F().qk_norm_rope_write8(qkv, n_q, n_kv, d, *how, ints(*positions), ints(*range(n)), slots, kv, max(positions))
        pages.append(kv)
    for name in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(getattr(pages[0], name).view(torch.uint8), getattr(pages[1], name).view(torch.uint8)), name
