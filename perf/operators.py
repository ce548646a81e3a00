"""The 8-bit key/value cache's operators as cases that can be timed: what a serving step does with such a cache.

A row is the key (or the value) of one position and one key/value head.  It is kept as hd numbers of type e4m3 times
2^e, e a whole number: the smallest one from -100 on for which the row's largest magnitude is at most 448 * 2^e.  Pools:
codes [pages, kv heads, 64, hd] of keys and of values, exponents as bytes e + 127 [pages, kv heads, 2, 64] (keys, then
values).  The page of a sequence's position p is table[sequence, p // 64].

* ``append``: the step's new queries, keys and values come out of the projection; bias, split-half rotation by the
  position's cosines and sines, queries rounded to bfloat16, keys and values rounded into the cache.
* ``decode``: one new token of every sequence attends to all that its sequence has cached (or to the last ``window``
  positions of it).
* ``prefill``: runs of new tokens, packed back to back, attend causally to what their sequences have cached, their own
  keys among it.

Sequences are given by ``lengths``: a rule that spreads ``seqs`` lengths between ``longest / ragged`` and ``longest``.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
LOWEST = -100            # the least exponent of a row


# ---------------------------------------------------------------------------------------------------------
# cases
def _case(name, op, nh, nkv, hd, seqs, longest, ragged=1, new=1, window=0, bias=False, rot=None):
    """``new``: new tokens of the longest sequence (the others bring their share of it, one at least)."""
    return {"name": name, "op": op, "nh": nh, "nkv": nkv, "hd": hd, "seqs": seqs, "longest": longest, "ragged": ragged, "new": new,
            "window": window, "bias": bias, "rot": hd if rot is None else rot}


def listed():
    return [
        # one sequence's next token, in every layer of every step: nothing but latency
        _case("append one token", "append", 16, 16, 128, 1, 700),
        # a step of a busy server with grouped heads
        _case("append 64 tokens", "append", 28, 4, 128, 64, 8000, ragged=16, bias=True),
        # prompts of unequal length behind what is cached already, half of every head rotated
        _case("append ragged prompts", "append", 16, 4, 80, 7, 2500, ragged=9, new=1031, rot=40),
        # a long prompt in one step
        _case("append 8192 tokens", "append", 16, 16, 128, 1, 8192, new=8192, bias=True),
        # one sequence, a short context
        _case("decode 1 x 777", "decode", 16, 16, 128, 1, 777),
        # a small batch, every head with keys of its own
        _case("decode 8 x 4096", "decode", 16, 16, 128, 8, 4096),
        # a large ragged batch with seven query heads to a key head
        _case("decode 64 x 8192 ragged", "decode", 28, 4, 128, 64, 8192, ragged=8),
        # one sequence with a long context
        _case("decode 1 x 131071", "decode", 28, 4, 128, 1, 131071),
        # layers that see a window of the context only, narrow heads
        _case("decode 24 x window 4096", "decode", 32, 4, 64, 24, 20011, ragged=3, window=4096),
        # a short prompt
        _case("prefill 200", "prefill", 16, 16, 128, 1, 200, new=200),
        # chunks of prompts behind contexts of unequal length
        _case("prefill ragged chunks", "prefill", 28, 4, 128, 5, 6100, ragged=3, new=1500),
        # a long prompt
        _case("prefill 8192", "prefill", 16, 16, 128, 1, 8192, new=8192),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    nkv = rng.choice([1, 2, 4, 5, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 6, 7, 8, 12, 16])
    while nkv * group > 48:
        group = max(1, group // 2)
    hd = rng.choice([64, 128, 128, 128, 80, 96, 104] + ([] if op == "prefill" else [192, 256]))
    nh = nkv * group
    window = rng.choice([0, 0, 0, _spread(rng, 17, 5000)]) if op != "append" else 0
    ragged = rng.choice([1, 1, 2, 5, 11])
    if op == "append":
        seqs = _spread(rng, 1, 96)
        new = 1 if rng.random() < 0.4 else _spread(rng, 2, max(3, int(4.5e7 / (seqs * (nh + 2 * nkv) * hd))))
        longest = new + _spread(rng, 1, 9000)
    elif op == "decode":
        seqs = _spread(rng, 1, 64)
        new, longest = 1, _spread(rng, 40, max(50, min(131072, int(1.0e8 / (seqs * nkv * hd)))))
    else:
        seqs = _spread(rng, 1, 9)
        new = _spread(rng, 2, max(3, int(math.sqrt(6.0e10 / (seqs * nh * hd)))))
        longest = new + (0 if rng.random() < 0.4 else _spread(rng, 1, max(2, min(20000, int(2.0e10 / (seqs * new * nh * hd)), int(2.0e8 / (seqs * nkv * 2 * hd))))))
    case = _case("", op, nh, nkv, hd, seqs, longest, ragged, new, window, rng.random() < 0.5, rng.choice([hd, hd, hd // 2, 0]))
    del case["name"]
    return case


def _sequences(case):
    """(lengths with the new tokens, new tokens) of the case's sequences."""
    n, longest, ragged, new = case["seqs"], case["longest"], case["ragged"], case["new"]
    shares = [1.0 if n == 1 or ragged == 1 else ragged ** (-((i * 7 + 3) % n) / (n - 1)) for i in range(n)]
    shares[0] = 1.0
    news = [max(1, int(new * s)) for s in shares]
    return [max(t, int(longest * s)) for s, t in zip(shares, news)], news


def _seen(case, length, new):
    """Of a sequence with ``new`` new tokens at its end: (pairs of a query and a key that it sees, keys that any of them sees)."""
    w, past = case["window"] or length, length - new
    pairs = sum(min(p + 1, w) for p in range(past, length)) if new <= 20000 else 0
    return pairs, min(length, w + new - 1)


def work(case):
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    lengths, news = _sequences(case)
    n = sum(news)
    if case["op"] == "append":
        width = (nh + 2 * nkv) * hd
        tables = sum(news) * case["rot"] * 4
        return {"bytes": n * width * 4 + tables + (width * 4 if case["bias"] else 0) + n * nh * hd * 2 + n * nkv * (2 * hd + 2),
                "flops": n * (3 * (nh + nkv) * case["rot"] + 2 * nkv * hd)}
    pairs = keys = 0
    for length, new in zip(lengths, news):
        p, k = _seen(case, length, new)
        pairs, keys = pairs + p, keys + k
    return {"bytes": keys * nkv * (2 * hd + 2) + 2 * n * nh * hd * 2, "flops": 4 * nh * hd * pairs}


# ---------------------------------------------------------------------------------------------------------
# what a program has in hand
def _rows_to_codes(x):
    """(codes e4m3, exponent bytes) of the rows (last dimension) of float32 ``x``."""
    amax = x.abs().amax(-1)
    m, top = torch.frexp(amax)                           # amax = m 2^top, m in [0.5, 1): amax <= 0.875 * 2^(9 + e)
    e = torch.where(m <= 0.875, top - 9, top - 8).clamp_min(LOWEST)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def prepare(case, seed):
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    lengths, news = _sequences(case)
    pages = [(length + PAGE - 1) // PAGE for length in lengths]
    total = sum(pages) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, count in enumerate(pages):
        table[i, :count] = order[at:at + count]
        at += count
    # keys with a few strong channels, values of plain size; the pools hold rows already, as in a running server
    strong = 1.0 + 3.0 * (torch.arange(hd, device="cuda") % 29 == 3)
    codes, exps = [], torch.empty((total, nkv, 2, PAGE), dtype=torch.uint8, device="cuda")
    for which in range(2):
        pool = torch.empty((total, nkv, PAGE, hd), dtype=torch.float8_e4m3fn, device="cuda")
        for lo in range(0, total, 512):
            x = randn(min(512, total - lo), nkv, PAGE, hd) * (strong if which == 0 else 0.7)
            pool[lo:lo + 512], exps[lo:lo + 512, :, which] = _rows_to_codes(x)
        codes.append(pool)
    n = sum(news)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for t in news:
        starts.append(starts[-1] + t)
    pasts = [length - t for length, t in zip(lengths, news)]
    tok_seq = torch.repeat_interleave(torch.arange(len(news), device="cuda", dtype=torch.int32), ints(news))
    tok_pos = (torch.arange(n, device="cuda", dtype=torch.int32) - ints(starts)[tok_seq.long()] + ints(pasts)[tok_seq.long()])
    state = {"case": case, "k": codes[0], "v": codes[1], "exps": exps, "table": table, "tok_seq": tok_seq, "tok_pos": tok_pos.to(torch.int32),
             "seq_start": ints(starts), "seq_past": ints(pasts), "max_new": max(news), "longest": max(lengths),
             "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if case["op"] == "append":
        half, width = case["rot"] // 2, (nh + 2 * nkv) * hd
        state["qkv"] = randn(n, width)
        state["qkv"].view(n, nh + 2 * nkv, hd)[:, :nh + nkv] *= strong
        state["bias"] = 0.3 * randn(width) if case["bias"] else None
        freq = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
        angle = torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        state["q"] = torch.empty((n, nh, hd), dtype=torch.bfloat16, device="cuda")
    else:
        state["q"] = (1.2 * randn(n, nh, hd)).to(torch.bfloat16)
        state["out"] = torch.empty_like(state["q"])
        # tiles of 128 new tokens of a sequence, those that see the most keys first
        tiles = sorted(((i, f) for i, t in enumerate(news) for f in range(0, t, 128)),
                       key=lambda sf: -(pasts[sf[0]] + min(sf[1] + 128, news[sf[0]])))
        state["tile_seq"], state["tile_first"] = ints([t[0] for t in tiles]), ints([t[1] for t in tiles])
    return state


# ---------------------------------------------------------------------------------------------------------
# one pass
def _append_plain(s):
    c = s["case"]
    nh, nkv, hd, half = c["nh"], c["nkv"], c["hd"], c["rot"] // 2
    x = s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]
    x = x.view(-1, nh + 2 * nkv, hd)
    pos, seq = s["tok_pos"].long(), s["tok_seq"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = x[:, :nh + nkv]
    a, b = qk[..., :half], qk[..., half:2 * half]
    qk = torch.cat((a * cos - b * sin, b * cos + a * sin, qk[..., 2 * half:]), -1)
    s["q"].copy_(qk[:, :nh])
    page, place = s["table"][seq, pos // PAGE].long(), pos % PAGE
    k, ke = _rows_to_codes(qk[:, nh:])
    v, ve = _rows_to_codes(x[:, nh + nkv:])
    s["k"].view(torch.uint8)[page, :, place] = k.view(torch.uint8)
    s["v"].view(torch.uint8)[page, :, place] = v.view(torch.uint8)
    s["exps"][page, :, 0, place] = ke
    s["exps"][page, :, 1, place] = ve


def _cached(s, pool, which):
    """float32 [sequences, kv heads, positions, hd] of what the pool holds for every sequence."""
    page = s["table"].clamp_min(0).long()
    x = pool[page].float() * torch.ldexp(torch.ones((), device="cuda"), s["exps"][:, :, which][page].int() - 127)[..., None]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :s["longest"]]


def _attend_plain(s):
    c = s["case"]
    nh, nkv, hd, most = c["nh"], c["nkv"], c["hd"], s["max_new"]
    start, past = s["seq_start"].long(), s["seq_past"].long()
    news, n_seqs = start[1:] - start[:-1], past.numel()
    place = torch.arange(most, device="cuda")
    rows = (start[:-1, None] + place).clamp_max(s["q"].shape[0] - 1)
    live = place < news[:, None]
    pos = past[:, None] + place
    q = s["q"].float()[rows].view(n_seqs, most, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n_seqs, nkv, -1, hd)
    k, v = _cached(s, s["k"], 0), _cached(s, s["v"], 1)
    score = (q @ k.transpose(2, 3)).view(n_seqs, nh, most, -1) * hd ** -0.5
    key = torch.arange(k.shape[2], device="cuda")
    hidden = key > pos[..., None]
    if c["window"]:
        hidden |= key <= pos[..., None] - c["window"]
    score.masked_fill_(hidden[:, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    weight = score.exp_()
    total = weight.sum(-1, keepdim=True)
    o = (weight.view(n_seqs, nkv, -1, weight.shape[-1]) @ v).view(n_seqs, nh, most, hd) / total
    s["out"][rows[live]] = o.permute(0, 2, 1, 3)[live].to(torch.bfloat16)


def _own(s):
    from esp_b200.csrc import ops
    from esp_b200.parts.base import Workspace
    c = s["case"]
    shape = (c["nh"], c["nkv"], c["hd"])
    if c["op"] == "append":
        ops.kv8_rope_append(s["qkv"], s["bias"], s["tok_seq"], s["tok_pos"], s["cos"], s["sin"], c["rot"], s["q"], s["k"], s["v"],
                            s["exps"], s["table"], PAGE, *shape, True, s["status"])
    elif c["op"] == "decode":
        if "ws" not in s:                                # scratch that a program keeps from step to step
            s["ws"] = Workspace(s["q"].device)
        ops.attn_decode_kv8(s["q"], s["k"], s["v"], s["exps"], s["out"], s["ws"], s["tok_seq"], s["tok_pos"], s["table"], PAGE,
                            *shape, c["window"], s["status"])
    else:
        ops.attn_prefill_kv8(s["q"], s["k"], s["v"], s["exps"], s["out"], s["tile_seq"], s["tile_first"], s["seq_start"],
                             s["seq_past"], s["table"], PAGE, *shape, c["window"], s["status"])


def run(state):
    if own:
        _own(state)
    elif state["case"]["op"] == "append":
        _append_plain(state)
    else:
        _attend_plain(state)
    if state["case"]["op"] == "append":
        return {"q": state["q"], "k": state["k"], "v": state["v"], "exps": state["exps"].view(torch.float8_e8m0fnu)}
    return {"out": state["out"]}


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
def _exact_row_exponent(row_max):
    """The smallest e >= LOWEST with row_max <= 448 * 2^e, by trying."""
    e = torch.full_like(row_max, float(LOWEST))
    guess = torch.floor(torch.log2(row_max.clamp_min(2.0 ** -120) / 448.0)) - 1
    e = torch.maximum(e, guess)
    for _ in range(3):
        e = torch.where(row_max > 448.0 * torch.exp2(e), e + 1, e)
    return e


def _exact_e4m3(y):
    """The nearest e4m3 numbers (ties to even) to float64 ``y`` of magnitude up to 448, as float64."""
    binade = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(binade - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["op"] == "append":
        half = case["rot"] // 2
        n = s["qkv"].shape[0]
        x = s["qkv"].double().view(n, nh + 2 * nkv, hd)
        if s["bias"] is not None:
            x = x + s["bias"].double().view(nh + 2 * nkv, hd)
        turned = x.clone()
        c, d = s["cos"].double()[s["tok_pos"].long()].unsqueeze(1), s["sin"].double()[s["tok_pos"].long()].unsqueeze(1)
        lo, hi = x[:, :nh + nkv, :half], x[:, :nh + nkv, half:2 * half]
        turned[:, :nh + nkv, :half] = lo * c - hi * d
        turned[:, :nh + nkv, half:2 * half] = hi * c + lo * d
        k, v = s["k"].double(), s["v"].double()
        exps = torch.exp2(s["exps"].double() - 127)
        page = s["table"][s["tok_seq"].long(), (s["tok_pos"] // PAGE).long()].long()
        place = (s["tok_pos"] % PAGE).long()
        for pool, which, rows in ((k, 0, turned[:, nh:nh + nkv]), (v, 1, turned[:, nh + nkv:])):
            e = _exact_row_exponent(rows.abs().amax(-1))
            pool[page, :, place] = _exact_e4m3(rows / torch.exp2(e).unsqueeze(-1))
            exps[page, :, which, place] = torch.exp2(e)
        return {"q": turned[:, :nh], "k": k, "v": v, "exps": exps}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, pasts = s["seq_start"].tolist(), s["seq_past"].tolist()
    for i, past in enumerate(pasts):
        row0, row1 = starts[i], starts[i + 1]
        length = past + row1 - row0
        pages = s["table"][i, :(length + PAGE - 1) // PAGE].long()
        at = torch.arange(past, length, device="cuda").unsqueeze(1)
        j = torch.arange(length, device="cuda").unsqueeze(0)
        sees = (j <= at) & ((at - j < case["window"]) if case["window"] else (j >= 0))
        for g in range(nkv):
            keys, values = ((pool[pages, g].double() * torch.exp2(s["exps"][pages, g, w].double() - 127).unsqueeze(-1)).reshape(-1, hd)[:length]
                            for w, pool in ((0, s["k"]), (1, s["v"])))
            for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                a = s["q"][row0:row1, h].double() @ keys.T / math.sqrt(hd)
                out[row0:row1, h] = torch.softmax(torch.where(sees, a, -math.inf), -1) @ values
    return {"out": out}
