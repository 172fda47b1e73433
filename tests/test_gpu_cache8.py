"""The 8-bit key/value cache on the device: the write, the way back, and attention of single tokens and of prompts over it, each against
a plain implementation in 64 bits; refusals; numbers that are none, places that must not be read, page numbers that cannot be."""

import pytest
import torch

from tests.plain import cache8 as plain8
from tests.plain import model as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64


def F():
    from gtar_kimik3_public_b200.ops import functional

    return functional


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def empty_pages(n_seqs, longest, n_kv, d, page=PAGE, spare=3, seed=1):
    """Pages in a scrambled order, every place poisoned: NaN numbers under the largest byte."""
    per = max(1, -(-longest // page))
    n_pages = n_seqs * per + spare
    gen = torch.Generator().manual_seed(seed)
    table = torch.randperm(n_pages, generator=gen)[: n_seqs * per].to(torch.int32).view(n_seqs, per)
    slots = torch.randperm(n_seqs + 2, generator=gen)[:n_seqs].to(torch.int32)
    whole = torch.zeros((n_seqs + 2, per), dtype=torch.int32)
    whole[slots.long()] = table
    k, v = (torch.full((n_pages, n_kv, page, d), 0x7F, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    k_exp, v_exp = (torch.full((n_pages, n_kv, page), 255, dtype=torch.uint8, device=DEV) for _ in range(2))
    return F().PagedKV8(k, v, k_exp, v_exp, whole.to(DEV)), slots.to(DEV), whole


def fill(kv, table, slot, k, v, first=0):
    """Puts the plain quantised rows of a sequence from position ``first`` on into its pages (the bytes by torch's own cast)."""
    page = kv.page_size
    for name, rows in (("k", k), ("v", v)):
        e = plain8.exponent_of(rows)
        x8 = (rows.double() / 2.0 ** e.unsqueeze(-1).double()).float().to(torch.float8_e4m3fn).view(torch.uint8)
        for j in range(first, rows.shape[0]):
            at = int(table[slot, j // page])
            getattr(kv, name).view(torch.uint8)[at, :, j % page] = x8[j].to(DEV)
            getattr(kv, name + "_exp")[at, :, j % page] = (e[j] + 127).to(torch.uint8).to(DEV)


def held(kv, table, slot, length):
    """What the pages stand for, [length, n_kv, d] in 64 bits on the CPU."""
    out = []
    for name in ("k", "v"):
        x = getattr(kv, name).cpu().float().double() * (2.0 ** (getattr(kv, name + "_exp").cpu().double() - 127)).unsqueeze(-1)
        pages = [x[int(table[slot, i])] for i in range(-(-length // kv.page_size))]
        out.append(torch.cat(pages, 1).transpose(0, 1)[:length])
    return out


# ------------------------------------------------------------------ write
HEADS = [(4, 2, 128), (12, 4, 64), (6, 2, 80), (2, 2, 32), (3, 1, 2), (16, 1, 128), (2, 1, 512)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_q,n_kv,d", HEADS)
@pytest.mark.parametrize("norm,rope", [(True, True), (False, False)])
def test_write(dtype, n_q, n_kv, d, norm, rope):
    eps, lens, past = 1e-5, [1, 67, 5], [0, 60, 127]
    kv, slots, table = empty_pages(3, 132, n_kv, d)
    pos = [p + i for n, p in zip(lens, past) for i in range(n)]
    seq = [i for i, n in enumerate(lens) for _ in range(n)]
    qkv = rand(len(pos), (n_q + 2 * n_kv) * d, seed=2).to(dtype)
    wq, wk = (1 + 0.1 * rand(d, seed=20)).float(), (1 + 0.1 * rand(d, seed=21)).float()
    cos, sin = plain.rotary_tables(torch.arange(132), d, 1e4)
    cos, sin = cos[:, : d // 2].float().contiguous(), sin[:, : d // 2].float().contiguous()
    q = F().qk_norm_rope_write8(qkv.to(DEV), n_q, n_kv, d, wq.to(DEV) if norm else None, wk.to(DEV) if norm else None, eps,
                                cos.to(DEV) if rope else None, sin.to(DEV) if rope else None, ints(*pos), ints(*seq), slots, kv, max(pos))
    x = qkv.double().view(-1, n_q + 2 * n_kv, d)

    def finished(y, w):
        y = plain.rms_norm(y, w.double(), eps) if norm else y
        c, s = (torch.cat([t[pos], t[pos]], -1).double() for t in (cos, sin))
        return plain.apply_rotary(y, c, s) if rope else y

    want_q, want_k, want_v = finished(x[:, :n_q], wq), finished(x[:, n_q:n_q + n_kv], wk), x[:, n_q + n_kv:]
    # 32-bit arithmetic on the way (a dozen roundings of 2^-24 of the pair that the rotation mixes; the sum of squares shares its own), then one
    # rounding of half a step
    noise = 2.0**-20
    reach = want_q.abs().amax(-1, keepdim=True)
    half = torch.finfo(dtype).eps / 2
    assert ((q.double().cpu() - want_q).abs() <= half * want_q.abs() + (noise if norm or rope else 0) * reach).all()
    written = torch.zeros(kv.k.shape[0], PAGE, dtype=torch.bool)
    got = {i: held(kv, table, int(slots[i]), p + n) for i, (n, p) in enumerate(zip(lens, past))}
    for t, (p, i) in enumerate(zip(pos, seq)):
        gk, gv = got[i][0][p], got[i][1][p]
        assert torch.equal(gv, plain8.quantised(want_v[t])), f"v of token {t}"  # no arithmetic before the rounding: the same bits
        e = plain8.exponent_of(want_k[t] * (1 + noise)).unsqueeze(-1).double()  # a maximum next to a power's end may take the power above it
        _, power = torch.frexp((want_k[t] / 2.0**e).abs().clamp_min(2.0**-6))
        step = torch.ldexp(torch.ones_like(want_k[t]), power - 4) * 2.0**e
        off = (gk - want_k[t]).abs()
        assert (off <= (1 + 1e-6) * step / 2 + (noise * want_k[t].abs().amax(-1, keepdim=True) if norm or rope else 0)).all(), f"k of token {t}"
        if not (norm or rope):
            assert torch.equal(gk, plain8.quantised(want_k[t]))
        written[int(table[int(slots[i]), p // PAGE]), p % PAGE] = True
    # nothing else was written
    untouched = ~written[:, None, :].expand(-1, n_kv, -1)
    for name in ("k", "v"):
        assert (getattr(kv, name).view(torch.uint8).cpu()[untouched] == 0x7F).all()
        assert (getattr(kv, name + "_exp").cpu()[untouched] == 255).all()


@pytest.mark.parametrize("n_q,n_kv,d,lens", [(16, 8, 128, [700, 1, 65]), (6, 2, 64, [1500, 800]), (3, 3, 128, [2300]),
                                             (16, 8, 128, [1500, 1, 400]), (6, 2, 64, [8000, 3500]), (3, 3, 128, [6400])])
@pytest.mark.parametrize("norm", [True, False])
def test_write_of_many_tokens(n_q, n_kv, d, lens, norm):
    """Too few rows for the warps that stay, and enough.  Keys are the formula in 64 bits rounded once, all of them; a place outside the pages is left out and
    reported, the others are what they are."""
    past, eps = [5 * i for i in range(len(lens))], 1e-6
    kv, slots, table = empty_pages(len(lens), max(lens) + 20, n_kv, d)
    pos = [p + i for n, p in zip(lens, past) for i in range(n)]
    seq = [i for i, n in enumerate(lens) for _ in range(n)]
    qkv = rand(len(pos), (n_q + 2 * n_kv) * d, seed=2).to(torch.bfloat16)
    assert (len(pos) * (n_q + 2 * n_kv) * d >= 7 << 20) == (sum(lens) > (1900 if n_kv == 8 else 2300))
    wq, wk = (1 + 0.1 * rand(d, seed=20)).to(torch.bfloat16), (1 + 0.1 * rand(d, seed=21)).to(torch.bfloat16)
    cos, sin = plain.rotary_tables(torch.arange(max(pos) + 1), d, 1e4)
    cos, sin = cos[:, : d // 2].float().contiguous(), sin[:, : d // 2].float().contiguous()
    wrong = len(pos) // 2
    seq_given = list(seq)
    seq_given[wrong] = len(lens)
    args = (wq.to(DEV), wk.to(DEV), eps, cos.to(DEV), sin.to(DEV)) if norm else (None, None, eps, None, None)
    q = F().qk_norm_rope_write8(qkv.to(DEV), n_q, n_kv, d, *args, ints(*pos), ints(*seq_given), slots, kv, max(pos))
    with pytest.raises(Exception, match="page number"):
        F().check_kernel_errors(DEV)
    x = qkv.double().view(-1, n_q + 2 * n_kv, d)

    def finished(y, w):
        if not norm:
            return y
        c, s = (torch.cat([t[pos], t[pos]], -1).double() for t in (cos, sin))
        return plain.apply_rotary(plain.rms_norm(y, w.double(), eps), c, s)

    want_q, want_k, want_v = finished(x[:, :n_q], wq), finished(x[:, n_q:n_q + n_kv], wk), x[:, n_q + n_kv:]
    reach = want_q.abs().amax(-1, keepdim=True)
    assert ((q.double().cpu() - want_q).abs() <= 2.0**-8 * want_q.abs() + (2.0**-20 if norm else 0) * reach).all()
    want_k, want_v = plain8.quantised(want_k), plain8.quantised(want_v)
    got = [held(kv, table, int(slots[i]), p + n) for i, (n, p) in enumerate(zip(lens, past))]
    got_k, got_v = (torch.cat([g[j][p:] for g, p in zip(got, past)]) for j in (0, 1))
    keep = torch.arange(len(pos)) != wrong
    assert torch.equal(got_v[keep], want_v[keep]) and torch.equal(got_k[keep], want_k[keep])
    assert torch.isnan(got_k[wrong]).all()  # the poison


@pytest.mark.parametrize("d", [32, 64, 128])
def test_write_rows_at_the_edges(d):
    """Zeros, a maximum of 448 times a power and right above it, ties between two numbers, numbers below the smallest step, the largest and
    smallest numbers, infinities and NaN."""
    big = 3.3895313892515355e38  # bfloat16's largest
    rows = torch.zeros(12, d, dtype=torch.float64)
    rows[1, 0], rows[1, 1] = 448.0, 1.0625  # halfway between 1 and 1.125
    rows[2, 0], rows[2, 1], rows[2, 2] = -450.0, 2.125, 2.375  # one power up
    rows[3, 0], rows[3, 1], rows[3, 2], rows[3, 3] = 448.0, 2.0**-10, 3 * 2.0**-10, 2.0**-11  # half a smallest step, one and a half, a quarter
    rows[4, 0], rows[4, 1] = big, -big
    rows[5, :] = 2.0**-120
    rows[6, 0], rows[6, 1], rows[6, 2] = float("inf"), 1.0, 3.0
    rows[7, 0], rows[7, 1] = float("nan"), -448.0 * 2.0**-5
    rows[8, :] = float("-inf")
    rows[9, 3] = -(448.0 * 2.0**-64)
    rows[10, 5] = 448.0 * 2.0**-66
    rows[11, :] = torch.linspace(-1, 1, d, dtype=torch.float64)
    rows = rows.to(torch.bfloat16)
    n = rows.shape[0]
    kv, slots, table = empty_pages(1, n, 1, d)
    qkv = torch.cat([torch.zeros_like(rows), rows, rows.flip(0)], 1)
    F().qk_norm_rope_write8(qkv.to(DEV), 1, 1, d, None, None, 1.0, None, None, ints(*range(n)), ints(*[0] * n), slots, kv, n - 1)
    k, v = held(kv, table, int(slots[0]), n)
    for got, want in ((k, rows), (v, rows.flip(0))):
        want = plain8.quantised(want.double())
        assert torch.equal(torch.isnan(got[:, 0]), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got[:, 0]), torch.nan_to_num(want))


def test_write_read_only_and_queries_alone():
    kv, slots, _ = empty_pages(1, 10, 2, 64)
    qkv = rand(10, (4 + 4) * 64).to(torch.bfloat16)
    q = F().qk_norm_rope_write8(qkv.to(DEV), 4, 2, 64, None, None, 1.0, None, None, ints(*range(10)), ints(*[0] * 10), slots, kv, 9, write_kv=False)
    assert torch.equal(q.cpu().view(10, -1), qkv[:, : 4 * 64])
    assert (kv.k.view(torch.uint8) == 0x7F).all() and (kv.v_exp == 255).all()


# ------------------------------------------------------------------ read back
@pytest.mark.parametrize("n_kv,d,page", [(2, 128, 64), (1, 64, 64), (3, 10, 32), (8, 80, 96)])
@pytest.mark.parametrize("last", [0, 1, 70])
def test_read_back(n_kv, d, page, last):
    lens = [1, 64, 0, 65, 200]
    kv, slots, table = empty_pages(5, 200, n_kv, d, page)
    for i, n in enumerate(lens):
        fill(kv, table, int(slots[i]), rand(n, n_kv, d, seed=i), rand(n, n_kv, d, seed=9 + i, scale=3.0))
    out = F().PagedKV(*(torch.full(kv.k.shape, 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)), kv.block_table)
    back = F().read_pages8(kv, ints(*lens), slots, 200, out, last)
    assert back is out
    named = torch.zeros(kv.k.shape[0], dtype=torch.bool)
    for i, n in enumerate(lens):
        slot = int(slots[i])
        want = held(kv, table, slot, n) if n else None
        for index in range(-(-n // page)):
            if last and (index + 1) * page <= n - last:
                continue
            at = int(table[slot, index])
            named[at] = True
            rows = min(page, n - index * page)
            for got, x in ((out.k[at], want[0]), (out.v[at], want[1])):
                got = got.double().cpu().transpose(0, 1)
                assert torch.equal(got[:rows], x[index * page:index * page + rows])  # exact: eight bits times a power of two
                assert (got[rows:] == 0).all()
    assert (out.k.cpu()[~named] == 7.0).all() and (out.v.cpu()[~named] == 7.0).all()


# ------------------------------------------------------------------ attention
def check_attention(got, q, k, v, past, window, sink, rounding, what):
    """A result is rounded once to its type, half a step; each probability may be off by ``rounding`` of itself, so that their sum with the values'
    sizes bounds what comes of it."""
    got, dtype = got.double().cpu(), got.dtype
    want, weight = (plain8.attention(q, k, x, past, window, sink) for x in (v, v.abs()))
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - torch.finfo(dtype).eps / 2 * want.abs() - rounding * weight
    assert (off <= 0).all(), f"{what}: {off.max():.3e} beyond"


# 32-bit scores of size up to 32 and 32-bit sums: 2^-24 of 32 in the exponent a few times over.  In a bfloat16 step of single tokens probabilities are
# rounded to halves (2^-11), in one of several tokens to bfloat16 at the least (2^-8).
SINGLE = {torch.float32: 2.0**-16, torch.bfloat16: 2.0**-11 + 2.0**-14}
SEVERAL = {torch.float32: 2.0**-16, torch.bfloat16: 2.0**-8 + 2.0**-12}


def sequences(lens, n_kv, d, page=PAGE, key_scale=1.0, window=0, new=None):
    """Filled pages for sequences of these lengths; with a window the places before it stay poisoned."""
    kv, slots, table = empty_pages(len(lens), max(1, max(lens)), n_kv, d, page)
    for i, n in enumerate(lens):
        k = rand(n, n_kv, d, seed=30 + i, scale=key_scale)
        v = rand(n, n_kv, d, seed=60 + i) * torch.exp(rand(n, n_kv, 1, seed=90 + i))
        m = 1 if new is None else new[i]
        fill(kv, table, int(slots[i]), k, v, max(0, n - m + 1 - window) if window else 0)
    return kv, slots, table


GROUPS = [(1, 1, 128), (4, 2, 128), (16, 4, 128), (8, 1, 128), (12, 1, 128), (16, 1, 64), (6, 2, 64), (17, 1, 64), (6, 2, 80), (3, 3, 16)]


@pytest.mark.parametrize("dtype,cut", [(torch.bfloat16, None), (torch.bfloat16, (1, 0)), (torch.bfloat16, (3, 0)), (torch.bfloat16, (8, 0)),
                                       (torch.bfloat16, (0, 1)), (torch.bfloat16, (0, 40)), (torch.float32, None)])
@pytest.mark.parametrize("n_q,n_kv,d", GROUPS)
@pytest.mark.parametrize("window,sink", [(0, False), (70, True)])
def test_decode(dtype, cut, n_q, n_kv, d, window, sink):
    lens = [1, 64, 65, 300, 777, 0, 16]
    kv, slots, table = sequences(lens, n_kv, d, window=window)
    q = rand(len(lens), n_q, d, seed=5).to(dtype)
    got = F().attention_decode8(q.to(DEV), kv, ints(*lens), slots, 777, d**-0.5, window, sink, cut=cut)
    assert (got[5] == 0).all()  # a sequence without tokens
    for i, n in enumerate(lens):
        if n:
            k, v = held(kv, table, int(slots[i]), n)
            check_attention(got[i:i + 1], q[i:i + 1], k, v, n - 1, window, sink, SINGLE[dtype], f"sequence of {n}")
    F().check_kernel_errors(DEV)


@pytest.mark.parametrize("page", [32, 96])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_other_pages(page, dtype):
    n_q, n_kv, d, lens = 4, 2, 128, [100, 32, 97]
    kv, slots, table = sequences(lens, n_kv, d, page)
    q = rand(9, n_q, d, seed=5).to(dtype)
    one = F().attention_decode8(q[:3].contiguous().to(DEV), kv, ints(*lens), slots, 100, d**-0.5)
    several = F().attention_prefill8(q.to(DEV), kv, ints(0, 3, 6, 9), ints(*lens), slots, 3, 100, d**-0.5)
    for i, m in enumerate(lens):
        k, v = held(kv, table, int(slots[i]), m)
        check_attention(one[i:i + 1], q[i:i + 1], k, v, m - 1, 0, False, SINGLE[dtype], f"sequence of {m}")
        check_attention(several[3 * i:3 * i + 3], q[3 * i:3 * i + 3], k, v, m - 3, 0, False, SEVERAL[dtype], f"sequence of {m}")


@pytest.mark.parametrize("n_q,n_kv,d", [(16, 8, 128), (8, 1, 128), (12, 1, 128), (16, 1, 64), (6, 2, 64), (1, 1, 64)])
@pytest.mark.parametrize("cut", [None, (1, 0), (4, 0), (0, 1), (0, 40)])
@pytest.mark.parametrize("window,norm,weights", [(0, True, torch.float32), (70, True, torch.bfloat16), (0, False, torch.float32)])
def test_decode_from_the_projection(n_q, n_kv, d, cut, window, norm, weights):
    """Norm, rotation, write and attention in one kernel: the cache gets the bytes that the write gives, the places around them stay, and the
    outputs are those of attention over them."""
    lens, eps = [1, 64, 65, 300, 777, 97, 32, 33], 1e-5
    n = len(lens)
    kv, slots, table = empty_pages(n, max(lens), n_kv, d)
    for i, m in enumerate(lens):  # all but the new token
        k, v = rand(m - 1, n_kv, d, seed=30 + i), rand(m - 1, n_kv, d, seed=60 + i)
        fill(kv, table, int(slots[i]), k, v, max(0, m - window) if window else 0)
    copy = F().PagedKV8(kv.k.view(torch.uint8).clone().view(torch.float8_e4m3fn), kv.v.view(torch.uint8).clone().view(torch.float8_e4m3fn),
                        kv.k_exp.clone(), kv.v_exp.clone(), kv.block_table)
    qkv = rand(n, (n_q + 2 * n_kv) * d, seed=7).to(torch.bfloat16)
    qkv[3, n_q * d:] = 0
    wq, wk = (1 + 0.1 * rand(d, seed=20)).to(weights).to(DEV), (1 + 0.1 * rand(d, seed=21)).to(weights).to(DEV)
    cos, sin = plain.rotary_tables(torch.arange(max(lens)), d, 1e4)
    cos, sin = cos[:, : d // 2].float().contiguous().to(DEV), sin[:, : d // 2].float().contiguous().to(DEV)
    how = (wq, wk, eps, cos, sin) if norm else (None, None, eps, None, None)
    pos = ints(*[m - 1 for m in lens])
    F().qk_norm_rope_write8(qkv.to(DEV), n_q, n_kv, d, *how, pos, ints(*range(n)), slots, copy, max(lens) - 1)
    got = F().attention_decode8_fused(qkv.to(DEV), n_q, n_kv, d, *how, kv, ints(*lens), slots, max(lens) - 1, 777, d**-0.5, window, cut=cut)
    F().check_kernel_errors(DEV)
    for a, b in ((kv.k, copy.k), (kv.v, copy.v), (kv.k_exp, copy.k_exp), (kv.v_exp, copy.v_exp)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    x = qkv.double().view(n, n_q + 2 * n_kv, d)[:, :n_q]
    if norm:
        c, s = (torch.cat([t, t], -1).double().cpu()[[m - 1 for m in lens]] for t in (cos, sin))
        x = plain.apply_rotary(plain.rms_norm(x, wq.double().cpu(), eps), c, s)
    for i, m in enumerate(lens):
        k, v = held(kv, table, int(slots[i]), m)
        # queries in 32 bits: 2^-20 of scores of up to some twenty
        check_attention(got[i:i + 1], x[i:i + 1], k, v, m - 1, window, False, SINGLE[torch.bfloat16] + 2.0**-15, f"sequence of {m}")
    # a layer that attends over what another has written
    again = F().attention_decode8_fused(qkv.to(DEV), n_q, n_kv, d, *how, kv, ints(*lens), slots, max(lens) - 1, 777, d**-0.5, window, write_kv=False, cut=cut)
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype,few", [(torch.bfloat16, None), (torch.bfloat16, True), (torch.bfloat16, False), (torch.float32, None)])
@pytest.mark.parametrize("n_q,n_kv,d", GROUPS)
@pytest.mark.parametrize("window,sink", [(0, False), (70, True)])
@pytest.mark.parametrize("new,lens", [([4, 1, 7, 3], [4, 200, 71, 66]), ([150, 1, 65, 0, 90], [150, 130, 300, 64, 90])])
def test_prefill(dtype, few, n_q, n_kv, d, window, sink, new, lens, monkeypatch):
    if few is not None:  # through the kernel for few rows, or through clean pages, whichever the rule would take
        monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: few)
    kv, slots, table = sequences(lens, n_kv, d, window=window, new=new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = rand(cu[-1] + 2, n_q, d, seed=5).to(dtype)  # two rows behind the last sequence
    out = torch.full(q.shape, 5.0, dtype=dtype, device=DEV)
    got = F().attention_prefill8(q.to(DEV), kv, ints(*cu), ints(*lens), slots, max(new), max(lens), d**-0.5, window, sink, out)
    assert got is out and (got[cu[-1]:] == 5.0).all()
    for i, (m, n) in enumerate(zip(new, lens)):
        if m:
            k, v = held(kv, table, int(slots[i]), n)
            check_attention(got[cu[i]:cu[i + 1]], q[cu[i]:cu[i + 1]], k, v, n - m, window, sink, SEVERAL[dtype], f"sequence {i}")
    F().check_kernel_errors(DEV)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m", [1, 3, 140])
def test_values_of_very_different_sizes(d, m):
    """Rows of values from 2^-60 to 2^100 and rows of zeros in one sequence; scores that grow along it, so that the maximum moves."""
    n, n_q, n_kv = 300, 4, 2
    kv, slots, table = empty_pages(1, n, n_kv, d)
    power = torch.randint(-60, 3, (n, n_kv, 1), generator=torch.Generator().manual_seed(3)).double()
    power[n // 3] = 100.0
    k, v = rand(n, n_kv, d, seed=1), rand(n, n_kv, d, seed=2) * 2.0**power
    v[n // 2:n // 2 + 9] = 0
    q = rand(m, n_q, d, seed=5)
    for j in range(n):  # a drift of up to 40 in the score towards the end, most of it away from the row of 2^100
        k[j] += q[-1, ::2] * (j / n) * 40 * d**0.5 / (q[-1, ::2] ** 2).sum(-1, keepdim=True)
    fill(kv, table, int(slots[0]), k, v)
    q = q.to(torch.bfloat16)
    k, v = held(kv, table, int(slots[0]), n)
    if m == 1:
        got = F().attention_decode8(q.to(DEV), kv, ints(n), slots, n, d**-0.5)
    else:
        got = F().attention_prefill8(q.to(DEV), kv, ints(0, m), ints(n), slots, m, n, d**-0.5)
    check_attention(got, q, k, v, n - m, 0, False, (SINGLE if m == 1 else SEVERAL)[torch.bfloat16], "values")


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (6, 2, 64), (6, 2, 80)])
def test_numbers_that_are_none(n_q, n_kv, d):
    """A key that is NaN makes the outputs of its kv head NaN where it is visible and nothing else."""
    lens = [100, 90]
    kv, slots, table = sequences(lens, n_kv, d)
    kv.k.view(torch.uint8)[int(table[int(slots[0]), 0]), 0, 30, 1] = 0x7F
    q = rand(2, n_q, d, seed=5).to(torch.bfloat16).to(DEV)
    got = F().attention_decode8(q, kv, ints(*lens), slots, 100, d**-0.5)
    group = n_q // n_kv
    assert torch.isnan(got[0, :group]).all() and torch.isfinite(got[0, group:]).all() and torch.isfinite(got[1]).all()
    behind = F().attention_decode8(q, kv, ints(30, 90), slots, 100, d**-0.5)  # the key lies behind the sequence's end
    assert torch.isfinite(behind).all()
    inside = F().attention_decode8(q, kv, ints(*lens), slots, 100, d**-0.5, window=60)  # and in front of the window
    assert torch.isfinite(inside).all()


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (6, 2, 64), (6, 2, 80)])
@pytest.mark.parametrize("m", [5, 90])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("few", [True, False])
def test_values_that_are_none_reach_only_who_sees_them(n_q, n_kv, d, m, window, few, monkeypatch):
    """A value that holds a NaN: tokens in front of it, tokens whose window has left it and other heads do not meet it."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: few)
    n, group = 150, n_q // n_kv
    kv, slots, table = sequences([n, 80], n_kv, d)
    at = n - m + 2  # the step's third token
    for name in ("k", "v"):
        kv_bytes = getattr(kv, name).view(torch.uint8)
        if name == "v":
            kv_bytes[int(table[int(slots[0]), at // PAGE]), 1, at % PAGE, 7] = 0xFF
    q = rand(m + 3, n_q, d, seed=5).to(torch.bfloat16).to(DEV)
    got = F().attention_prefill8(q, kv, ints(0, m, m + 3), ints(n, 80), slots, m, n, d**-0.5, window)
    see = torch.tensor([t >= 2 and (not window or n - m + t < at + window) for t in range(m)])
    assert torch.isfinite(got[m:]).all() and torch.isfinite(got[:m, :group]).all()
    assert torch.isfinite(got[:m, group:2 * group][~see]).all()
    assert torch.isnan(got[:m, group:2 * group][see][:, :, 7]).all()


def test_prefill_where_pages_keep_their_numbers(monkeypatch):
    """Bounds on lengths so large that renumbered pages would be more than there are: the prefill kernels see the same pages under other numbers."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: False)
    n_q, n_kv, d, new, lens = 4, 2, 128, [70, 1, 40], [200, 64, 40]
    kv, slots, table = sequences(lens, n_kv, d, new=new)
    wide = torch.cat([kv.block_table, torch.zeros((kv.block_table.shape[0], 60), dtype=torch.int32, device=DEV)], 1).contiguous()
    wide = F().PagedKV8(kv.k, kv.v, kv.k_exp, kv.v_exp, wide)
    q = rand(111, n_q, d, seed=5).to(torch.bfloat16)
    args = (ints(0, 70, 71, 111), ints(*lens), slots, 70)
    got = F().attention_prefill8(q.to(DEV), wide, *args, 64 * 60, d**-0.5)
    assert torch.equal(got, F().attention_prefill8(q.to(DEV), kv, *args, 200, d**-0.5))
    F().check_kernel_errors(DEV)


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (6, 2, 64)])
def test_prefill_where_sequences_share_pages(n_q, n_kv, d, monkeypatch):
    """The same slot at two lengths that end inside one page, and another sequence that begins with its first page: under their own numbers the pages serve
    all of them."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: False)
    new, lens = [70, 1, 40, 5], [200, 180, 130, 170]
    kv, slots, table = sequences([200, 200, 200, 200], n_kv, d)
    whole = kv.block_table.clone()
    whole[slots[2], 0] = whole[slots[0], 0]
    slots = torch.stack([slots[0], slots[0], slots[2], slots[0]])
    narrow = F().PagedKV8(kv.k, kv.v, kv.k_exp, kv.v_exp, whole)
    wide = F().PagedKV8(kv.k, kv.v, kv.k_exp, kv.v_exp, torch.cat([whole, torch.zeros((whole.shape[0], 60), dtype=torch.int32, device=DEV)], 1).contiguous())
    q = rand(116, n_q, d, seed=5).to(torch.bfloat16).to(DEV)
    args = (ints(0, 70, 71, 111, 116), ints(*lens), slots, 70)
    want = F().attention_prefill8(q, narrow, *args, 200, d**-0.5)
    for _ in range(5):
        assert torch.equal(F().attention_prefill8(q, wide, *args, 64 * 60, d**-0.5), want)
    F().check_kernel_errors(DEV)


def test_a_window_longer_than_any_sequence(monkeypatch):
    """As if there were none, up to the largest number that a window can be."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: False)
    kv, slots, _ = sequences([200, 64], 2, 128)
    q = rand(71, 4, 128, seed=5).to(torch.bfloat16).to(DEV)
    args = (ints(0, 70, 71), ints(200, 64), slots, 70, 200, 0.1)
    want = F().attention_prefill8(q, kv, *args)
    for window in (200, 2**31 - 71, 2**31 - 1):
        assert torch.equal(F().attention_prefill8(q, kv, *args, window), want)


@pytest.mark.parametrize("few", [True, False])
def test_page_numbers_slots_and_lengths_that_cannot_be(few, monkeypatch):
    """They are skipped and reported; the step's other sequences are what they are."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: few)
    n_q, n_kv, d = 4, 2, 128
    lens = [100, 90, 70]
    kv, slots, table = sequences(lens, n_kv, d)
    q = rand(3, n_q, d, seed=5).to(torch.bfloat16).to(DEV)
    args = (kv, ints(*lens), slots, 100, d**-0.5)
    good = F().attention_decode8(q, *args)
    F().check_kernel_errors(DEV)
    several = rand(120, n_q, d, seed=6).to(torch.bfloat16).to(DEV)
    prompts = [(m, ints(0, m, 2 * m, 3 * m), F().attention_prefill8(several[: 3 * m], kv, ints(0, m, 2 * m, 3 * m), ints(*lens), slots, m, 100, d**-0.5))
               for m in (3, 40)]  # through both kernels
    keep = kv.block_table.clone()
    for wrong in (-1, kv.k.shape[0], 2**31 - 1):
        kv.block_table[int(slots[1]), 1] = wrong
        got = F().attention_decode8(q, *args)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        assert torch.equal(got[[0, 2]], good[[0, 2]])
        for m, cu, want in prompts:
            got = F().attention_prefill8(several[: 3 * m], kv, cu, ints(*lens), slots, m, 100, d**-0.5)
            with pytest.raises(Exception, match="page number"):
                F().check_kernel_errors(DEV)
            assert torch.equal(got[:m], want[:m]) and torch.equal(got[2 * m:], want[2 * m:])
        F().read_pages8(kv, ints(*lens), slots, 100)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        kv.block_table.copy_(keep)
    for wrong_slots, wrong_lens in (([int(slots[0]), 99, int(slots[2])], lens), (slots.tolist(), [100, 10**6, 70]), (slots.tolist(), [100, -5, 70])):
        got = F().attention_decode8(q, kv, ints(*wrong_lens), ints(*wrong_slots), 100, d**-0.5)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        assert torch.equal(got[[0, 2]], good[[0, 2]])
    qkv = rand(2, (n_q + 2 * n_kv) * d).to(torch.bfloat16).to(DEV)
    before = kv.k.view(torch.uint8).clone()
    for pos, seq in (([128, 128], [0, 0]), ([-1, -1], [0, 0]), ([5, 5], [3, -1])):
        F().qk_norm_rope_write8(qkv, n_q, n_kv, d, None, None, 1.0, None, None, ints(*pos), ints(*seq), slots, kv, 128)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        assert torch.equal(kv.k.view(torch.uint8), before)


def test_starts_that_cannot_be_behind_clean_pages(monkeypatch):
    """Starts beyond the queries and starts that fall: put within the queries and in order, and reported."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: False)
    kv, slots, table = sequences([100, 90], 2, 128)
    q = rand(80, 4, 128, seed=5).to(torch.bfloat16).to(DEV)
    good = F().attention_prefill8(q, kv, ints(0, 40, 80), ints(100, 90), slots, 40, 100, 0.1)
    F().check_kernel_errors(DEV)
    for cu in ([0, 40, 9000], [0, 40, 20]):
        out = torch.full(q.shape, 5.0, dtype=q.dtype, device=DEV)
        F().attention_prefill8(q, kv, ints(*cu), ints(100, 90), slots, 40, 100, 0.1, out=out)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        assert torch.equal(out[:40], good[:40]) and (torch.equal(out[40:], good[40:]) if cu[2] > 80 else (out[40:] == 5.0).all())


def test_tokens_that_there_are_none_of(monkeypatch):
    """Starts beyond the queries, starts that fall, and more tokens than ``max_q_len``: left out and reported by the kernel for few rows."""
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: True)
    kv, slots, table = sequences([100, 90], 2, 128)
    q = rand(8, 4, 128, seed=5).to(torch.bfloat16).to(DEV)
    good = F().attention_prefill8(q, kv, ints(0, 4, 8), ints(100, 90), slots, 4, 100, 0.1)
    F().check_kernel_errors(DEV)
    for cu, most, kept in (([0, 4, 900], 4, 8), ([0, 4, 2], 4, 4), ([-3, 4, 8], 4, None), ([0, 4, 8], 2, None)):
        out = torch.full(q.shape, 5.0, dtype=q.dtype, device=DEV)
        F().attention_prefill8(q, kv, ints(*cu), ints(100, 90), slots, most, 100, 0.1, out=out)
        with pytest.raises(Exception, match="page number"):
            F().check_kernel_errors(DEV)
        if kept is not None:
            assert torch.equal(out[:4], good[:4]) and (kept == 8 or (out[4:] == 5.0).all())


def test_a_length_that_cannot_be_writes_nothing():
    kv, slots, table = sequences([100, 90], 2, 128)
    before = [t.view(torch.uint8).clone() for t in (kv.k, kv.v, kv.k_exp, kv.v_exp)]
    qkv = rand(2, 8 * 128).to(torch.bfloat16).to(DEV)
    for wrong in (10**6, 0, -4):
        F().attention_decode8_fused(qkv, 4, 2, 128, None, None, 1.0, None, None, kv, ints(wrong, wrong), slots, 99, 100, 0.1)
        if wrong:
            with pytest.raises(Exception, match="page number"):
                F().check_kernel_errors(DEV)
        assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, (kv.k, kv.v, kv.k_exp, kv.v_exp)))


def test_which_kernels_start_early(monkeypatch):
    """Prefill attention over pages made clean reads what the kernel in front writes, before it waits: it never starts early.  The kernel that joins
    pieces touches nothing before it waits."""
    from tests.test_early_launches import _early_edges

    kv, slots, table = sequences([300, 200], 2, 128)
    q = rand(120, 4, 128, seed=5).to(torch.bfloat16).to(DEV)
    lens, cu = ints(300, 200), ints(0, 60, 120)
    monkeypatch.setattr(F(), "rows8_wins", lambda *sizes: False)
    prompts = lambda: F().attention_prefill8(q, kv, cu, lens, slots, 60, 300, 0.1)  # noqa: E731
    pieces = lambda: F().attention_decode8(q[:2], kv, lens, slots, 300, 0.1, cut=(0, 40))  # noqa: E731
    want = prompts().clone(), pieces().clone()
    before = F().set_pdl(True)
    try:
        edges = [_early_edges(run) for run in (prompts, pieces)]
    finally:
        F().set_pdl(before)
    assert edges == [(1, 0), (1, 1)]
    assert torch.equal(prompts(), want[0]) and torch.equal(pieces(), want[1])


def test_refusals():
    f = F()
    kv, slots, _ = empty_pages(2, 100, 2, 64)
    n, lens = 2, ints(10, 20)
    q = torch.zeros((n, 4, 64), dtype=torch.bfloat16, device=DEV)

    def refused(match, call):
        with pytest.raises(f.KernelError, match=match):
            call()

    refused("contiguous", lambda: f.attention_decode8(q.transpose(0, 1), kv, lens, slots, 100, 0.1))
    refused("do not fit", lambda: f.attention_decode8(q[:, :3].contiguous(), kv, lens, slots, 100, 0.1))
    refused("do not fit", lambda: f.attention_decode8(torch.zeros((n, 4, 32), dtype=torch.bfloat16, device=DEV), kv, lens, slots, 100, 0.1))
    refused("float32 or bfloat16", lambda: f.attention_decode8(q.half(), kv, lens, slots, 100, 0.1))
    refused("entries", lambda: f.attention_decode8(q, kv, lens[:1], slots, 100, 0.1))
    refused("int32", lambda: f.attention_decode8(q, kv, lens.long(), slots, 100, 0.1))
    refused("window", lambda: f.attention_decode8(q, kv, lens, slots, 100, 0.1, -1))
    refused("window", lambda: f.attention_prefill8(q, kv, ints(0, 1, 2), lens, slots, 1, 100, 0.1, -1))
    refused("on cpu", lambda: f.attention_decode8(q, kv, lens.cpu(), slots, 100, 0.1))
    refused("like q", lambda: f.attention_decode8(q, kv, lens, slots, 100, 0.1, out=q.float()))
    refused("entries", lambda: f.attention_prefill8(q, kv, ints(0, 2), lens, slots, 1, 100, 0.1))
    refused("bfloat16", lambda: f.read_pages8(kv, lens, slots, 100, f.PagedKV(kv.k, kv.v, kv.block_table)))
    qkv = torch.zeros((n, 8 * 64), dtype=torch.bfloat16, device=DEV)
    w, table = torch.ones(64, device=DEV), torch.zeros((5, 32), device=DEV)
    write = lambda **a: f.qk_norm_rope_write8(**{**dict(qkv=qkv, n_q=4, n_kv=2, head_dim=64, q_weight=w, k_weight=w, eps=1e-6, cos=None, sin=None,  # noqa: E731
                                                        tok_pos=lens, tok_seq=ints(0, 1), slots=slots, kv=kv, max_position=20), **a})
    refused("wide", lambda: write(n_q=6))
    refused("fit", lambda: write(n_q=6, n_kv=1))
    refused("both or neither", lambda: write(k_weight=None))
    refused("head_dim entries", lambda: write(q_weight=w[:32].contiguous(), k_weight=w[:32].contiguous()))
    refused("go together", lambda: write(cos=table))
    refused("beyond the rotary table", lambda: write(cos=table, sin=table))
    refused("q_out", lambda: write(q_out=q[:1]))
    refused("entries", lambda: write(tok_pos=ints(0, 1, 2)))
    e4, byte = torch.float8_e4m3fn, torch.uint8
    pages = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device=DEV)  # noqa: E731
    good = dict(k=pages((2, 1, 64, 64), e4), v=pages((2, 1, 64, 64), e4), k_exp=pages((2, 1, 64), byte), v_exp=pages((2, 1, 64), byte),
                block_table=pages((1, 2), torch.int32))
    f.PagedKV8(**good)
    for match, wrong in (("float8", dict(k=pages((2, 1, 64, 64), torch.bfloat16))), ("alike", dict(v=pages((2, 1, 64, 32), e4))),
                         ("exponents", dict(k_exp=pages((2, 1, 32), byte))), ("uint8", dict(v_exp=pages((2, 1, 64), torch.int32))),
                         ("int32", dict(block_table=pages((1, 2), torch.int64)))):
        refused(match, lambda: f.PagedKV8(**{**good, **wrong}))
    refused("page size", lambda: f.PagedKV8(pages((2, 1, 40, 64), e4), pages((2, 1, 40, 64), e4), pages((2, 1, 40), byte), pages((2, 1, 40), byte),
                                            good["block_table"]))


def test_empty_steps():
    kv, slots, _ = empty_pages(2, 100, 2, 64)
    none = ints()
    q = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    assert F().attention_decode8(q, kv, none, none, 0, 0.1).shape == (0, 4, 64)
    assert F().attention_prefill8(q, kv, ints(0, 0), ints(5), slots[:1], 0, 5, 0.1).shape == (0, 4, 64)
    F().read_pages8(kv, none, none, 0)
    F().qk_norm_rope_write8(torch.zeros((0, 8 * 64), dtype=torch.bfloat16, device=DEV), 4, 2, 64, None, None, 1.0, None, None, none, none, slots, kv, 0)
