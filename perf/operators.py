"""Measured cases of the paged key-value cache operators and of the windowed prompt attention (``valle_amd.ops``).

Four operators that a decoder with a bounded cache runs one after another:

* ``window_attention``        prompt rows against a sliding window, the first tokens and a text prefix that stay visible
* ``paged_kv_write``          new keys and values into the pages of their sequences
* ``paged_decode_attention``  one new token of each sequence against its pages, adding up the attention weight of every key
* ``kv_evict``                the keys with the least accumulated weight leave, the others move up

``run`` computes them in plain torch operations in 32 bits, or, where ``own`` is true, by the calls a user makes.  Lengths are a
function of the case alone, so that ``work`` knows them; every value comes from the seed.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- cases -----------------------------------------------------------------------------------------------------------------------
def _win(name, dtype, B, lo, hi, H, Hkv, dh, window, sinks, text_lo, text_hi):
    return dict(name=name, op="window", dtype=dtype, B=B, lo=lo, hi=hi, H=H, Hkv=Hkv, dh=dh, window=window, sinks=sinks, text_lo=text_lo,
                text_hi=text_hi)


def _write(name, dtype, B, lo, hi, at_lo, at_hi, Hkv, dh, page):
    return dict(name=name, op="write", dtype=dtype, B=B, lo=lo, hi=hi, at_lo=at_lo, at_hi=at_hi, Hkv=Hkv, dh=dh, page=page)


def _dec(name, dtype, B, lo, hi, H, Hkv, dh, page, window, sinks, text_lo, text_hi, mass):
    return dict(name=name, op="decode", dtype=dtype, B=B, lo=lo, hi=hi, H=H, Hkv=Hkv, dh=dh, page=page, window=window, sinks=sinks,
                text_lo=text_lo, text_hi=text_hi, mass=mass)


def _evict(name, dtype, B, lo, hi, Hkv, dh, page, budget, recent, sinks, text_lo, text_hi):
    return dict(name=name, op="evict", dtype=dtype, B=B, lo=lo, hi=hi, Hkv=Hkv, dh=dh, page=page, budget=budget, recent=recent, sinks=sinks,
                text_lo=text_lo, text_hi=text_hi)


def listed():
    return [
        # two short prompts, a handful of phonemes each: the call's latency
        _win("window_short", "bf16", 2, 12, 37, 16, 16, 64, 16, 2, 5, 9),
        # a batch of utterances of the benchmark's length (text, 3 s prompt, up to 10 s), the text prefix visible throughout
        _win("window_batch", "bf16", 32, 700, 1100, 16, 16, 64, 256, 0, 40, 130),
        # one recording of several minutes, grouped heads of 128
        _win("window_long", "bf16", 1, 12289, 12289, 16, 4, 128, 2048, 4, 0, 0),
        # the token-exact mode with the heads of the d1536 model
        _win("window_fp32", "fp32", 2, 700, 1025, 16, 16, 96, 300, 4, 40, 60),
        # one decode step of six slots: one token each
        _write("write_step", "bf16", 6, 1, 1, 230, 1000, 16, 64, 16),
        # the prompts of 64 utterances at once, behind what each slot holds already
        _write("write_prompts", "bf16", 64, 150, 420, 0, 77, 16, 64, 32),
        # one utterance near the end of its 10 s
        _dec("decode_one", "bf16", 1, 1025, 1025, 16, 16, 64, 16, 0, 0, 0, 0, False),
        # a full batch of utterances, the attention weight of every key added up for a later eviction
        _dec("decode_batch", "bf16", 64, 330, 1100, 16, 16, 64, 32, 0, 0, 0, 0, True),
        # three recordings of a quarter of an hour with grouped heads, the whole cache read: few rows, a long axis
        _dec("decode_long", "bf16", 3, 40000, 60001, 32, 8, 128, 64, 0, 0, 0, 0, False),
        # long recordings in the token-exact mode, only the text prefix and the last seconds visible
        _dec("decode_window", "fp32", 16, 9000, 30011, 16, 16, 96, 64, 1500, 4, 40, 130, False),
        # four slots past their budget
        _evict("evict_slots", "bf16", 4, 900, 1500, 16, 64, 16, 768, 75, 0, 40, 130),
        # long recordings brought back to half their cache
        _evict("evict_long", "bf16", 32, 4500, 9001, 8, 128, 64, 4096, 512, 4, 0, 0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _heads(rng):
    dh = rng.choice([32, 40, 64, 64, 96, 128, 128])
    H = rng.choice([4, 8, 16, 16, 32])
    Hkv = H // rng.choice([g for g in (1, 1, 2, 4, 8, 16) if H % g == 0])
    return H, Hkv, dh


def draw(rng):
    op = rng.choice(["window", "write", "decode", "decode", "evict"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    H, Hkv, dh = _heads(rng)
    page = rng.choice([8, 16, 32, 64, 128])
    hi = _log(rng, 1, 8000)
    lo = max(1, int(hi * rng.uniform(0.2, 1.0)))
    text_hi = rng.choice([0, min(hi, _log(rng, 2, 200))])
    text_lo = text_hi // 2
    sinks = rng.choice([0, 1, 4, 17])
    window = rng.choice([0, _log(rng, 1, 4000)])
    if op == "window":
        most = (9.0e10 if dtype == "bf16" else 2.0e10) / H / dh  # pairs: a plain pass holds the scores of all of them
        hi = min(hi, int(most ** 0.5))
        lo, text_hi = min(lo, hi), min(text_hi, hi)
        text_lo = text_hi // 2
        B = _log(rng, 1, max(1, min(48, int(min(most, 5.0e8 / H) / hi / hi))))
        c = _win("", dtype, B, lo, hi, H, Hkv, dh, window, sinks, text_lo, text_hi)
    elif op == "write":
        B = _log(rng, 1, max(1, min(64, int(1.2e7 / (Hkv * dh * hi)))))
        c = _write("", dtype, B, lo, hi, 0, _log(rng, 1, 500), Hkv, dh, page)
    elif op == "decode":
        hi = _log(rng, 1, 30000)
        lo = max(1, int(hi * rng.uniform(0.2, 1.0)))
        text_hi = min(hi, text_hi)
        B = _log(rng, 1, max(1, min(64, int(1.2e8 / (Hkv * dh * hi)))))
        c = _dec("", dtype, B, lo, hi, H, Hkv, dh, page, window, sinks, text_hi // 2, text_hi, rng.choice([True, False]))
    else:
        hi = _log(rng, 16, 9000)
        lo = max(1, int(hi * rng.uniform(0.2, 1.0)))
        B = _log(rng, 1, max(1, min(48, int(1.5e8 / (Hkv * dh * hi)))))
        budget = max(1, int(hi * rng.uniform(0.2, 0.9)))
        sinks = min(sinks, budget)
        recent = min(budget - sinks, _log(rng, 1, 500))
        c = _evict("", dtype, B, lo, hi, Hkv, dh, page, budget, recent, sinks, min(hi, text_lo), min(hi, text_hi))
    del c["name"]
    return c


def _ragged(B, lo, hi, salt):
    """B lengths from lo to hi, the last one hi: a function of the case alone."""
    got = [lo + ((b + salt) * 2654435761 >> 7) % (hi - lo + 1) for b in range(B)]
    got[-1] = hi
    return got


def _lengths(c):
    return _ragged(c["B"], c["lo"], c["hi"], 1)


def _texts(c):
    return [min(t, n) for t, n in zip(_ragged(c["B"], c["text_lo"], c["text_hi"], 5), _lengths(c))]


# ---- what a program has in hand --------------------------------------------------------------------------------------------------
def _values(g, *shape, dtype, gain=1.0, shift=0.0):
    """Normal values with an offset for each head and channel, as projections of layer-normed rows have."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(gain)
    if shift:
        x += shift * torch.randn(shape[-1], generator=g, device="cuda", dtype=torch.float32)
    return x.to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(g, c, lengths):
    """Pages for these lengths in an order of their own, with a few that no sequence has."""
    page, B = c["page"], c["B"]
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "window":
        lengths = _lengths(c)
        off = [0]
        for n in lengths:
            off.append(off[-1] + n)
        s["q"] = _values(g, off[-1], c["H"], c["dh"], dtype=dtype, gain=1.5)
        s["k"] = _values(g, off[-1], c["Hkv"], c["dh"], dtype=dtype, shift=0.5)
        s["v"] = _values(g, off[-1], c["Hkv"], c["dh"], dtype=dtype, shift=0.5)
        s["seq_off"], s["text_len"] = _int32(off), _int32(_texts(c))
        return s
    if c["op"] == "write":
        lengths = _lengths(c)
        start = _ragged(c["B"], c["at_lo"], c["at_hi"], 3)
        off = [0]
        for n in lengths:
            off.append(off[-1] + n)
        s["table"], total = _pool(g, c, [a + n for a, n in zip(start, lengths)])
        s["k"] = _values(g, off[-1], c["Hkv"], c["dh"], dtype=dtype, shift=0.5)
        s["v"] = _values(g, off[-1], c["Hkv"], c["dh"], dtype=dtype, shift=0.5)
        s["start"], s["seq_off"] = _int32(start), _int32(off)
    else:
        lengths = _lengths(c)
        s["table"], total = _pool(g, c, lengths)
        s["lengths"], s["text_len"] = _int32(lengths), _int32(_texts(c))
        if c["op"] == "decode":
            s["q"] = _values(g, c["B"], c["H"], c["dh"], dtype=dtype, gain=1.5)
    s["k_pages"] = _values(g, total, c["Hkv"], c["page"], c["dh"], dtype=dtype, shift=0.5)
    s["v_pages"] = _values(g, total, c["Hkv"], c["page"], c["dh"], dtype=dtype, shift=0.5)
    # weight that earlier steps added up: a few keys have most of it, and freshly written ones none
    mass = torch.rand(total, c["Hkv"], c["page"], generator=g, device="cuda")
    s["mass"] = torch.where(mass < 0.05, torch.zeros_like(mass), mass.pow(6).mul_(40.0))
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------------------
def _softmax(scores, visible):
    scores = scores.masked_fill_(~visible, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_window(s):
    c, off, text = s["case"], s["seq_off"].long(), s["text_len"]
    G, L = c["H"] // c["Hkv"], c["hi"]
    n = off[1:] - off[:-1]
    at = torch.arange(L, device="cuda")
    valid = at < n[:, None]
    row = torch.where(valid, off[:-1, None] + at, off[:-1, None])
    q = s["q"][row].float().transpose(1, 2).unflatten(1, (c["Hkv"], G))  # (B, Hkv, G, L, dh)
    k = s["k"][row].float().permute(0, 2, 3, 1).unsqueeze(2)              # (B, Hkv, 1, dh, L)
    v = s["v"][row].float().transpose(1, 2).unsqueeze(2)                  # (B, Hkv, 1, L, dh)
    i, j = at[:, None], at[None, :]
    near = (i - j < c["window"]) | (j < c["sinks"]) if c["window"] else torch.ones_like(i == j)
    visible = ((j < text[:, None, None]) | ((j <= i) & near)) & valid[:, None, :]
    p = _softmax((q @ k).mul_(1.0 / math.sqrt(c["dh"])), visible[:, None, None])
    o = (p @ v).flatten(1, 2).transpose(1, 2)  # (B, L, H, dh)
    out = torch.empty_like(s["q"])
    out[row] = torch.where(valid[:, :, None, None], o, o[:, :1]).to(out.dtype)
    return out


def _plain_write(s):
    c = s["case"]
    rows = torch.arange(s["k"].shape[0], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["seq_off"][1:], rows, right=True)
    pos = (s["start"][b] + rows - s["seq_off"][b]).long()
    page, slot = s["table"][b, pos // c["page"]].long(), pos % c["page"]
    s["k_pages"][page, :, slot] = s["k"]
    s["v_pages"][page, :, slot] = s["v"]
    s["mass"][page, :, slot] = 0.0
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "mass": s["mass"]}


def _plain_decode(s):
    c, n = s["case"], s["lengths"].long()[:, None]
    B, Hkv, G = c["B"], c["Hkv"], c["H"] // c["Hkv"]
    if c["window"] and c["window"] < c["hi"]:
        first = max(c["sinks"], c["text_hi"])
        head = s["text_len"].long().clamp(min=c["sinks"])[:, None]
        a, w = torch.arange(first, device="cuda")[None], n - c["window"] + torch.arange(c["window"], device="cuda")[None]
        pos = torch.cat([a.expand(B, -1), w], 1)
        visible = torch.cat([(a < head) & (a < n), (w >= head) & (w >= 0)], 1)
    else:
        pos = torch.arange(c["hi"], device="cuda")[None].expand(B, -1)
        visible = pos < n
    pos = torch.where(visible, pos, n - 1)
    page, slot = s["table"].long().gather(1, pos // c["page"]), pos % c["page"]
    k = s["k_pages"][page, :, slot].float().permute(0, 2, 3, 1)  # (B, Hkv, dh, N)
    v = s["v_pages"][page, :, slot].float().transpose(1, 2)      # (B, Hkv, N, dh)
    q = s["q"].float().unflatten(1, (Hkv, G))
    p = _softmax((q @ k).mul_(1.0 / math.sqrt(c["dh"])), visible[:, None, None])
    got = {"out": (p @ v).flatten(1, 2).to(s["q"].dtype)}
    if c["mass"]:
        s["mass"].transpose(1, 2).index_put_((page, slot), p.sum(2).transpose(1, 2), accumulate=True)
        got["mass"] = s["mass"]
    return got


def _plain_evict(s):
    c, n = s["case"], s["lengths"].long()[:, None, None]
    pos = torch.arange(c["hi"], device="cuda")[None, None]
    heads = torch.arange(c["Hkv"], device="cuda")[None, :, None]

    def place(p):
        return s["table"].long().gather(1, (p // c["page"]).flatten(1)).view(p.shape), heads, p % c["page"]

    here = torch.minimum(pos, n - 1).expand(c["B"], c["Hkv"], -1)
    head = s["text_len"].long().clamp(min=c["sinks"], max=c["budget"])[:, None, None]
    recent = torch.clamp(c["budget"] - head, max=c["recent"])
    key = s["mass"][place(here)]
    key = torch.where((pos < head) | (pos >= n - recent), math.inf, key)
    key = torch.where(pos < n, key, -math.inf)
    kept = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., :c["budget"]].sort(-1)[0]  # of equal weights the earlier key stays
    kept = torch.where(kept < n, kept, -1)
    left = torch.clamp(n, max=c["budget"])
    to = torch.minimum(torch.arange(kept.shape[-1], device="cuda"), left - 1).expand_as(kept)
    src, dst = place(kept.gather(2, to)), place(to)
    for pages in (s["k_pages"], s["v_pages"], s["mass"]):
        pages[dst] = pages[src]
    return {"kept": kept.to(torch.int32), "lengths": left.view(-1).to(torch.int32), "k_pages": s["k_pages"], "v_pages": s["v_pages"],
            "mass": s["mass"]}


# ---- the framework's own ---------------------------------------------------------------------------------------------------------
def _own(s):
    from valle_amd import ops

    c = s["case"]
    if c["op"] == "window":
        return ops.window_attention(s["q"], s["k"], s["v"], s["seq_off"], window=c["window"], sinks=c["sinks"], text_len=s["text_len"])
    if c["op"] == "write":
        ops.paged_kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["start"], seq_off=s["seq_off"], mass=s["mass"])
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "mass": s["mass"]}
    if c["op"] == "decode":
        mass = s["mass"] if c["mass"] else None
        got = {"out": ops.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], window=c["window"],
                                                 sinks=c["sinks"], text_len=s["text_len"], mass=mass)}
        if c["mass"]:
            got["mass"] = s["mass"]
        return got
    kept, lengths = ops.kv_evict(s["k_pages"], s["v_pages"], s["mass"], s["table"], s["lengths"], c["budget"], recent=c["recent"],
                                 sinks=c["sinks"], text_len=s["text_len"])
    return {"kept": kept, "lengths": lengths, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "mass": s["mass"]}


PLAIN = {"window": _plain_window, "write": _plain_write, "decode": _plain_decode, "evict": _plain_evict}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------
def _seen(n, i, text, window, sinks):
    """How many of n keys row i sees: the text prefix, and of the keys up to i the last `window` and the first `sinks`."""
    head = min(n, max(text, min(sinks, i + 1) if window else 0))
    low = max(0, i + 1 - window) if window else 0
    return head + max(0, i + 1 - max(low, head))


def work(case):
    c = case
    es = 2 if c["dtype"] == "bf16" else 4
    lengths = _lengths(c)
    rows = sum(lengths)
    if c["op"] == "window":
        seen = sum(_seen(n, i, t, c["window"], c["sinks"]) for n, t in zip(lengths, _texts(c)) for i in range(n))
        return {"bytes": es * rows * c["dh"] * 2 * (c["H"] + c["Hkv"]), "flops": 4 * c["H"] * c["dh"] * seen}
    if c["op"] == "write":
        return {"bytes": rows * c["Hkv"] * (4 * es * c["dh"] + 4), "flops": 0}
    if c["op"] == "decode":
        seen = sum(_seen(n, n - 1, t, c["window"], c["sinks"]) for n, t in zip(lengths, _texts(c)))
        return {"bytes": es * c["dh"] * (2 * c["Hkv"] * seen + 2 * c["H"] * c["B"]) + (8 * c["Hkv"] * seen if c["mass"] else 0),
                "flops": 4 * c["H"] * c["dh"] * seen}
    # the keys up to the first one that leaves stay where they are; that one's place goes by the weights, and is near the protected ones
    moved = sum(max(0, c["budget"] - max(t, c["sinks"])) for n, t in zip(lengths, _texts(c)) if n > c["budget"])
    over = sum(n for n in lengths if n > c["budget"])
    return {"bytes": c["Hkv"] * (moved * (4 * es * c["dh"] + 4) + 4 * over + 4 * c["B"] * c["budget"]), "flops": 0}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------
def _attend(q, k, v, see):
    """softmax(q k^T / sqrt(dh)) v of one head over the keys that `see` (rows, keys) allows, and the weights."""
    z = torch.where(see, q.double() @ k.double().T / math.sqrt(q.shape[-1]), -math.inf)
    e = torch.exp(z - z.max(1, keepdim=True)[0])
    w = e / e.sum(1, keepdim=True)
    return w @ v.double(), w


def _see(rows, n, text, window, sinks):
    i, j = rows[:, None], torch.arange(n, device="cuda")[None]
    causal = j <= i
    if window:
        causal = causal & ((j > i - window) | (j < sinks))
    return causal | (j < text)


def _slots(table, b, page, n):
    """Where the n keys of sequence b are: page and slot of each."""
    p = torch.arange(n, device="cuda")
    return table[b][p // page].long(), p % page


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "window":
        out, off = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), s["seq_off"].tolist()
        for b, text in enumerate(_texts(c)):
            rows, n = slice(off[b], off[b + 1]), off[b + 1] - off[b]
            see = _see(torch.arange(n, device="cuda"), n, text, c["window"], c["sinks"])
            for h in range(c["H"]):
                kv = h // (c["H"] // c["Hkv"])
                out[rows, h] = _attend(s["q"][rows, h], s["k"][rows, kv], s["v"][rows, kv], see)[0]
        return out
    if c["op"] == "write":
        off, start = s["seq_off"].tolist(), s["start"].tolist()
        kp, vp, mass = s["k_pages"].double(), s["v_pages"].double(), s["mass"].double()
        for b in range(c["B"]):
            n = off[b + 1] - off[b]
            page, slot = (x[start[b]:] for x in _slots(s["table"], b, c["page"], start[b] + n))
            for h in range(c["Hkv"]):
                kp[page, h, slot] = s["k"][off[b]:off[b + 1], h].double()
                vp[page, h, slot] = s["v"][off[b]:off[b + 1], h].double()
                mass[page, h, slot] = 0.0
        return {"k_pages": kp, "v_pages": vp, "mass": mass}
    if c["op"] == "decode":
        out, mass = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), s["mass"].double()
        G = c["H"] // c["Hkv"]
        for b, (n, text) in enumerate(zip(_lengths(c), _texts(c))):
            page, slot = _slots(s["table"], b, c["page"], n)
            see = _see(torch.tensor([n - 1], device="cuda"), n, text, c["window"], c["sinks"])
            for h in range(c["Hkv"]):
                group = slice(h * G, (h + 1) * G)
                out[b, group], w = _attend(s["q"][b, group], s["k_pages"][page, h, slot], s["v_pages"][page, h, slot], see)
                mass[page, h, slot] += w.sum(0)
        return {"out": out, "mass": mass} if c["mass"] else {"out": out}
    kp, vp, mass = s["k_pages"].double(), s["v_pages"].double(), s["mass"].double()
    kept = torch.full((c["B"], c["Hkv"], c["budget"]), -1, dtype=torch.int32)
    for b, (n, text) in enumerate(zip(_lengths(c), _texts(c))):
        page, slot = _slots(s["table"], b, c["page"], n)
        first = min(c["budget"], n, max(text, c["sinks"]))
        last = min(c["recent"], c["budget"] - first)
        for h in range(c["Hkv"]):
            stay = list(range(n))
            if n > c["budget"]:
                w = mass[page, h, slot].tolist()
                middle = sorted(range(first, n - last), key=lambda p: (-w[p], p))[:c["budget"] - first - last]
                stay = list(range(first)) + sorted(middle) + list(range(n - last, n))
            kept[b, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            of = torch.tensor(stay, device="cuda")
            for pages in (kp, vp, mass):
                pages[page[:len(stay)], h, slot[:len(stay)]] = pages[page[of], h, slot[of]]
    lengths = torch.tensor([min(n, c["budget"]) for n in _lengths(c)], dtype=torch.int32)
    return {"kept": kept.cuda(), "lengths": lengths.cuda(), "k_pages": kp, "v_pages": vp, "mass": mass}
