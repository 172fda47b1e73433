"""What the 8-bit key/value cache is timed at: the store, the way back, and the two attentions that read it.

The cache keeps keys and values in pages of 64 positions ``[page, kv head, position, head size]`` as e4m3 numbers, with one
power of two a (position, kv head) beside them: ``x = x8 * 2^(b - 127)`` with ``b`` a byte, the smallest power for which the row's
largest number stays within 448.  Sizes are those of the benchmark's configurations (16 or 32 query heads on 8 kv heads of 128) and of
the small ones (heads of 64).  ``own`` says which side ``run`` takes: the operators written out in torch, or the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
EPS = 1e-6
ROPE_BASE = 1e6
TOP = 448.0  # the largest e4m3 number
LOW, HIGH = -64, 119  # powers of two that a row may be scaled by


def listed():
    return [
        # the keys and values of eight requests' next tokens, early in their answers
        {"name": "store_step", "op": "store", "n_q": 16, "n_kv": 8, "d": 128, "new": "1,1,1,1,1,1,1,1", "past": "3,9,17,30,41,50,62,63", "window": 0},
        # odd pieces of three prompts, small heads: one begins in the middle of a page, one behind a full one
        {"name": "store_pieces", "op": "store", "n_q": 12, "n_kv": 4, "d": 64, "new": "37,300,513", "past": "0,64,1000", "window": 0},
        # three long prompts that start together
        {"name": "store_prompts", "op": "store", "n_q": 32, "n_kv": 8, "d": 128, "new": "2048,4096,1777", "past": "0,0,0", "window": 0},
        # one conversation read back
        {"name": "read_one", "op": "read", "n_q": 16, "n_kv": 8, "d": 128, "new": "1", "past": "1110", "window": 0},
        # a batch of unequal conversations read back
        {"name": "read_many", "op": "read", "n_q": 32, "n_kv": 8, "d": 128, "new": "1,1,1,1,1,1,1,1", "past": "4095,99,8190,2776,639,16000,7777,63",
         "window": 0},
        # one person's conversation, one token: latency
        {"name": "decode_one", "op": "decode", "n_q": 16, "n_kv": 8, "d": 128, "new": "1", "past": "700", "window": 0},
        # eight unequal conversations
        {"name": "decode_8", "op": "decode", "n_q": 32, "n_kv": 8, "d": 128, "new": "1,1,1,1,1,1,1,1", "past": "255,700,1201,1777,2303,2900,3517,4095",
         "window": 0},
        # a full batch of conversations of 1,024 to 8,192 tokens
        {"name": "decode_64", "op": "decode", "n_q": 32, "n_kv": 8, "d": 128, "new": "1*64", "past": "1023:8191", "window": 0},
        # one very long document
        {"name": "decode_long", "op": "decode", "n_q": 32, "n_kv": 8, "d": 128, "new": "1", "past": "131071", "window": 0},
        # a few guessed tokens of each of sixteen conversations looked at in one step
        {"name": "prompt_guesses", "op": "prompt", "n_q": 32, "n_kv": 8, "d": 128, "new": "4*16", "past": "600:3000", "window": 0},
        # the benchmark's prompt
        {"name": "prompt_2048", "op": "prompt", "n_q": 16, "n_kv": 8, "d": 128, "new": "2048", "past": "0", "window": 0},
        # unequal prompts, one of them a piece behind 4,000 tokens
        {"name": "prompts_unequal", "op": "prompt", "n_q": 32, "n_kv": 8, "d": 128, "new": "129,514,1027,2049,3333", "past": "4000,0,130,0,0", "window": 0},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    n_q, n_kv, d = rng.choice([(16, 8, 128), (32, 8, 128), (32, 8, 128), (12, 4, 64), (8, 8, 128), (14, 2, 64), (16, 1, 128), (6, 2, 64)])
    op = rng.choice(["store", "read", "decode", "decode", "prompt", "prompt"])
    window = 0
    if op == "decode":
        n = _spread(rng, 1, 64)
        top = _spread(rng, 64, 131072 // max(1, n * n_kv // 16))
        new, past = [1] * n, [_spread(rng, 1, top) - 1 for _ in range(n)]
        window = rng.choice([0, 0, 0, _spread(rng, 16, top)])
    elif op == "read":
        n = _spread(rng, 1, 16)
        new, past = [1] * n, [_spread(rng, 1, 20000 // n) for _ in range(n)]
    elif op == "store":
        n = _spread(rng, 1, 32)
        new, past = [_spread(rng, 1, max(2, 7000 // n)) for _ in range(n)], [rng.choice([0, _spread(rng, 1, 500)]) for _ in range(n)]
    elif rng.random() < 0.5:  # few tokens each
        n = _spread(rng, 1, 24)
        new, past = [rng.randint(1, 12) for _ in range(n)], [_spread(rng, 1, 4000) for _ in range(n)]
        new[0] = max(2, new[0])
        window = rng.choice([0, 0, 0, _spread(rng, 16, 4000)])
    else:
        n = _spread(rng, 1, 6)
        new = [_spread(rng, 2, 3200 // n) for _ in range(n)]
        past = [rng.choice([0, 0, _spread(rng, 1, 2500)]) for _ in range(n)]
        window = rng.choice([0, 0, 0, _spread(rng, 16, 3000)])
    return {"op": op, "n_q": n_q, "n_kv": n_kv, "d": d, "new": ",".join(map(str, new)), "past": ",".join(map(str, past)), "window": window}


def _lengths(case):
    """The step's new tokens and cached ones, sequence by sequence."""
    text = case["new"]
    new = [int(text.split("*")[0])] * int(text.split("*")[1]) if "*" in text else [int(x) for x in text.split(",")]
    text = case["past"]
    if ":" in text:  # so many lengths spread evenly between the two, in an order that is none
        low, high = (int(x) for x in text.split(":"))
        n = len(new)
        past = [low + (high - low) * ((i * 37) % n) // max(1, n - 1) for i in range(n)]
    else:
        past = [int(x) for x in text.split(",")]
    return new, past


def work(case):
    new, past = _lengths(case)
    n_q, n_kv, d, window = case["n_q"], case["n_kv"], case["d"], case["window"]
    tokens, kept = sum(new), 2 * n_kv * (d + 1)  # bytes of a position in the cache
    if case["op"] == "store":
        length = sum(p + n for p, n in zip(past, new))
        # the projection in, the rotation's rows once, queries out, the cache's rows in; then every position back in 16 bits
        positions = max(p + n for p, n in zip(past, new))
        return {"bytes": tokens * (2 * (n_q + 2 * n_kv) * d + 2 * n_q * d + kept) + min(tokens, positions) * 4 * d + length * (kept + 4 * n_kv * d),
                "flops": tokens * (n_q + n_kv) * d * 8}
    if case["op"] == "read":
        length = sum(p + n for p, n in zip(past, new))
        return {"bytes": length * (kept + 4 * n_kv * d), "flops": length * 2 * n_kv * d}
    pairs = seen = 0
    for n, p in zip(new, past):
        first = max(0, p + 1 - window) if window else 0
        seen += p + n - first
        pairs += sum(min(p + i + 1, window) for i in range(n)) if window else n * p + n * (n + 1) // 2
    return {"bytes": seen * kept + tokens * n_q * d * 4, "flops": 4 * pairs * n_q * d}


def _quantise(x):
    """e4m3 numbers and the bytes of their powers of two, a row (the last dimension) at a time."""
    top = x.abs().amax(-1)
    part, power = torch.frexp(top)  # top = part * 2^power, 0.5 <= part < 1; 448 = 0.875 * 2^9
    e = (power - 9 + (part > 0.875).to(power.dtype)).clamp(LOW, HIGH)
    e = torch.where(top > 0, e, torch.full_like(e, LOW))
    x8 = torch.ldexp(x, -e.unsqueeze(-1)).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return x8, (e + 127).to(torch.uint8)


def _values(x8, b):
    return torch.ldexp(x8.float(), b.to(torch.int32).unsqueeze(-1) - 127)


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(int(seed))
    new, past = _lengths(case)
    n, n_q, n_kv, d = len(new), case["n_q"], case["n_kv"], case["d"]
    length = [p + m for p, m in zip(past, new)]
    pages = [-(-m // PAGE) for m in length]
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.zeros((n + 2, max(pages)), dtype=torch.int32, device=DEVICE)
    slots = (torch.randperm(n + 2, generator=gen, device=DEVICE)[:n]).to(torch.int32)
    at = 0
    for i, slot in enumerate(slots.tolist()):
        table[slot, :pages[i]] = order[at:at + pages[i]]
        at += pages[i]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    # keys are normed and rotated, so they are alike in size; values differ from token to token
    k, k_exp = _quantise(rand(n_pages, n_kv, PAGE, d))
    v, v_exp = _quantise(rand(n_pages, n_kv, PAGE, d) * torch.exp(0.7 * rand(n_pages, n_kv, PAGE, 1)))
    tokens = sum(new)
    ints = dict(dtype=torch.int32, device=DEVICE)
    state = {
        **case, "k": k, "v": v, "k_exp": k_exp, "v_exp": v_exp, "table": table, "slots": slots,
        "kv_len": torch.tensor(length, **ints), "cu_q": torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), **ints),
        "tok_pos": torch.cat([torch.arange(p, p + m) for p, m in zip(past, new)]).to(**ints),
        "tok_seq": torch.repeat_interleave(torch.arange(n), torch.tensor(new)).to(**ints),
        "max_q_len": max(new), "max_kv_len": max(length), "scale": d ** -0.5,
    }
    if case["op"] == "store":
        state["qkv"] = rand(tokens, (n_q + 2 * n_kv) * d).to(torch.bfloat16)
        state["wq"], state["wk"] = 1 + 0.1 * rand(d), 1 + 0.1 * rand(d)
        angle = torch.arange(max(length), device=DEVICE, dtype=torch.float64).unsqueeze(1) / ROPE_BASE ** (
            torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
        state["cos"], state["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    elif case["op"] != "read":
        state["q"] = rand(tokens, n_q, d).to(torch.bfloat16)
    if case["op"] in ("store", "read"):
        state["k16"] = torch.zeros((n_pages, n_kv, PAGE, d), dtype=torch.bfloat16, device=DEVICE)
        state["v16"] = torch.zeros_like(state["k16"])
    return state


def run(s):
    if own:
        return _own(s)
    if s["op"] == "store":
        q = _plain_store(s)
        k, v = _plain_read(s)
        return {"q": q, "k": k, "v": v}
    if s["op"] == "read":
        k, v = _plain_read(s)
        return {"k": k, "v": v}
    return _plain_attention(s)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from gtar_kimik3_public_b200.ops import functional as F

    kv = s.get("view")
    if kv is None:  # what a cache makes once for a layer
        kv = s["view"] = F.PagedKV8(s["k"], s["v"], s["k_exp"], s["v_exp"], s["table"])
        if "k16" in s:
            s["pages16"] = F.PagedKV(s["k16"], s["v16"], s["table"])
    op = s["op"]
    if op == "decode":
        return F.attention_decode8(s["q"], kv, s["kv_len"], s["slots"], s["max_kv_len"], s["scale"], s["window"])
    if op == "prompt":
        return F.attention_prefill8(s["q"], kv, s["cu_q"], s["kv_len"], s["slots"], s["max_q_len"], s["max_kv_len"], s["scale"], s["window"])
    out = {}
    if op == "store":
        out["q"] = F.qk_norm_rope_write8(s["qkv"], s["n_q"], s["n_kv"], s["d"], s["wq"], s["wk"], EPS, s["cos"], s["sin"], s["tok_pos"], s["tok_seq"],
                                         s["slots"], kv, s["max_kv_len"] - 1)
    F.read_pages8(kv, s["kv_len"], s["slots"], s["max_kv_len"], s["pages16"])
    return {**out, "k": s["k16"], "v": s["v16"]}


# ------------------------------------------------------------------ the operators written out
def _plain_store(s):
    n_q, n_kv, d = s["n_q"], s["n_kv"], s["d"]
    x = s["qkv"].float().view(-1, n_q + 2 * n_kv, d)
    pos = s["tok_pos"].long()
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)

    def normed(x, w):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., : d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    page = s["table"][s["slots"][s["tok_seq"].long()].long(), pos // PAGE].long()
    for name, rows in (("k", normed(x[:, n_q:n_q + n_kv], s["wk"])), ("v", x[:, n_q + n_kv:])):
        x8, b = _quantise(rows)
        s[name].view(torch.uint8)[page, :, pos % PAGE] = x8.view(torch.uint8)
        s[name + "_exp"][page, :, pos % PAGE] = b
    return normed(x[:, :n_q], s["wq"]).to(torch.bfloat16)


def _plain_read(s):
    """Every position of every sequence as bfloat16, in pages of the same numbers; what is behind a sequence's end in its last page is zero."""
    table = s["table"][s["slots"].long()].long()
    first = torch.arange(table.shape[1], device=table.device) * PAGE
    here = first < s["kv_len"].unsqueeze(1)
    page = table[here]
    row = first.expand_as(here)[here].unsqueeze(1) + torch.arange(PAGE, device=table.device)
    valid = (row < s["kv_len"].unsqueeze(1).expand_as(here)[here].unsqueeze(1))[:, None, :, None]
    for name in ("k", "v"):
        x = _values(s[name][page], s[name + "_exp"][page])
        s[name + "16"][page] = torch.where(valid, x, torch.zeros_like(x)).to(torch.bfloat16)
    return s["k16"], s["v16"]


def _plain_attention(s):
    n_q, n_kv, d, window = s["n_q"], s["n_kv"], s["d"], s["window"]
    n, most = s["kv_len"].shape[0], s["max_q_len"]
    keys = torch.arange(s["max_kv_len"], device=DEVICE)
    page = s["table"][s["slots"].long()].long()[:, keys // PAGE]
    row = (keys % PAGE).expand_as(page)
    k, v = (_values(s[name][page, :, row], s[name + "_exp"][page, :, row]) for name in ("k", "v"))  # [n, keys, n_kv, d]
    here = keys < s["kv_len"].unsqueeze(1)
    v = torch.where(here[:, :, None, None], v, torch.zeros_like(v))
    # the step's tokens with a row of places a sequence
    new = s["cu_q"][1:] - s["cu_q"][:-1]
    place = torch.arange(most, device=DEVICE)
    there = place < new.unsqueeze(1)
    q = torch.zeros((n, most, n_q, d), device=DEVICE)
    q[there] = s["q"].float()
    last = (s["kv_len"] - new).unsqueeze(1) + place  # the last key that a place sees
    visible = keys <= last.unsqueeze(2)
    if window:
        visible = visible & (keys > last.unsqueeze(2) - window)
    scores = torch.einsum("ntgcd,nsgd->ngcts", q.view(n, most, n_kv, n_q // n_kv, d), k) * s["scale"]
    scores = scores.masked_fill(~visible[:, None, None], float("-inf"))
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.einsum("ngcts,nsgd->ntgcd", scores, v)
    o = o / scores.sum(-1).permute(0, 3, 1, 2).unsqueeze(-1)
    return o.reshape(n, most, n_q, d)[there].to(torch.bfloat16)


# ------------------------------------------------------------------ in 64 bits, a sequence at a time
def exact(case, seed):
    s = prepare(case, seed)
    new, past = _lengths(case)
    n_q, n_kv, d, window = case["n_q"], case["n_kv"], case["d"], case["window"]
    table, slots = s["table"].tolist(), s["slots"].tolist()

    def rounded(x):
        """The nearest e4m3 number times the row's power of two, ties to even: steps of 2^-3 of the number's own power, of 2^-9 below 2^-6."""
        top = x.abs().max(-1, keepdim=True).values
        e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp_min(1e-300) / TOP)), torch.full_like(top, LOW))
        e = torch.where(top > TOP * 2.0 ** e, e + 1, e)
        e = torch.where((top > 0) & (top <= TOP * 2.0 ** (e - 1)), e - 1, e).clamp(LOW, HIGH)
        y = x / 2.0 ** e
        step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(y / step).mul(step).clamp(-TOP, TOP) * 2.0 ** e

    def kept(i, name):
        ids = torch.tensor(table[slots[i]][: -(-(past[i] + new[i]) // PAGE)], device=DEVICE)
        x = s[name][ids].double() * 2.0 ** (s[name + "_exp"][ids].double() - 127).unsqueeze(-1)
        return ids, x.transpose(1, 2).reshape(-1, n_kv, d)[: past[i] + new[i]]

    outputs, at = [], 0
    pages = {name: torch.zeros(s["k"].shape, dtype=torch.float64, device=DEVICE) for name in ("k", "v")} if case["op"] in ("store", "read") else {}
    for i, (n, p) in enumerate(zip(new, past)):
        (ids, k), (_, v) = kept(i, "k"), kept(i, "v")
        if case["op"] == "store":
            x = s["qkv"][at:at + n].double().view(n, -1, d)
            cos, sin = s["cos"][p:p + n].double().unsqueeze(1), s["sin"][p:p + n].double().unsqueeze(1)
            rows = []
            for part, w in ((x[:, :n_q], s["wq"]), (x[:, n_q:n_q + n_kv], s["wk"])):
                y = part / torch.sqrt((part * part).sum(-1, keepdim=True) / d + EPS) * w.double()
                half = torch.cat([-y[..., d // 2:], y[..., : d // 2]], -1)
                rows.append(y * torch.cat([cos, cos], -1) + half * torch.cat([sin, sin], -1))
            outputs.append(rows[0])
            k[p:], v[p:] = rounded(rows[1]), rounded(x[:, n_q + n_kv:])
        if pages:
            for name, x in (("k", k), ("v", v)):
                whole = torch.zeros((len(ids) * PAGE, n_kv, d), dtype=torch.float64, device=DEVICE)
                whole[: p + n] = x
                pages[name][ids] = whole.view(-1, PAGE, n_kv, d).transpose(1, 2)
        else:
            q = s["q"][at:at + n].double()
            o = torch.empty_like(q)
            for t in range(0, n, 512):  # so many tokens at a time
                m = min(512, n - t)
                where = p + t + torch.arange(m, device=DEVICE).unsqueeze(1)
                key = torch.arange(p + n, device=DEVICE)
                hidden = (key > where) | ((key <= where - window) if window else torch.zeros_like(key, dtype=torch.bool))
                for h in range(n_q):
                    a = q[t:t + m, h] @ k[:, h * n_kv // n_q].T * d ** -0.5
                    a = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
                    o[t:t + m, h] = a @ v[:, h * n_kv // n_q]
            outputs.append(o)
        at += n
    if not pages:
        return torch.cat(outputs)
    return {**({"q": torch.cat(outputs)} if outputs else {}), **pages}
