"""Serving steps over a paged key/value cache, for timing: rotary positions, appending a step's keys and values to the pages, and
attention of the new tokens over them.

A case is a dict with a "kind" (rotate, append, attention) and its sizes; `listed()` holds the cases that are quoted and
`draw(rng)` gives more of the same ranges. `prepare` makes on the GPU what a serving loop has in hand, `run` is one pass --
the plain form in elementary torch operations, or with `own` the package's calls -- and `exact` the same values in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------ the cases

def _rotate(name, **c):
    return dict(dict(kind="rotate", rotated=c["dim"], layout="half", scaling="none", base=1e4, far=c["tokens"]), **c, name=name)


def _append(name, **c):
    return dict(dict(kind="append", decodes=0, ragged=0, dim=128, rotated=128, layout="half", scaling="none", base=1e6, cache=c["type"], page=16),
                **c, name=name)


def _attention(name, **c):
    return dict(dict(kind="attention", decodes=0, ragged=0, pad=0, dim=128, page=16, softcap=0.0, window=0, slopes=False, prefix=0), **c, name=name)


def listed():
    return [
        # One token's queries at a far position: the smallest call, bound by its launch.
        _rotate("rotate-token", tokens=1, heads=32, dim=128, type="bf16", base=1e6, far=131072),
        # A prompt's queries, half of each head rotated, frequencies interpolated by wavelength for long contexts.
        _rotate("rotate-4096", tokens=4096, heads=32, dim=128, rotated=64, type="bf16", scaling="bands", base=5e5, far=65536),
        # A long sequence in the interleaved layout with yarn-scaled frequencies (1536 x 1536 and text, 24 heads).
        _rotate("rotate-interleaved-9293", tokens=9293, heads=24, dim=128, type="fp16", layout="interleaved", scaling="yarn", far=9293),
        # A decode step of 64 sequences: each token's k and v to its page, q and k rotated.
        _append("append-decode-64", batch=64, chunk=1, cached=8191, ragged=1, heads=32, kv_heads=8, type="bf16"),
        # Prompt chunks of three sequences, from the fp32 linears of text generation into a 16-bit cache of odd pages.
        _append("append-ragged-fp32", batch=3, chunk=2049, cached=1000, ragged=2, heads=32, kv_heads=8, type="fp32", cache="bf16", page=24,
                layout="interleaved"),
        # A whole long prompt.
        _append("append-16384", batch=1, chunk=16384, cached=0, heads=32, kv_heads=8, type="fp16", page=64, scaling="linear", base=1e4),
        # One token of one sequence over the cache of the decode layer, in fp32 as text generation runs.
        _attention("decode-1-fp32", batch=1, chunk=1, cached=2047, heads=32, kv_heads=8, type="fp32"),
        # One token each of 61 sequences of very different lengths, in a batch padded to 64.
        _attention("decode-61", batch=61, chunk=1, cached=16383, ragged=3, pad=3, heads=32, kv_heads=8, type="bf16"),
        # A chunk of a prompt over what earlier chunks left in the cache: the largest.
        _attention("chunk-2048", batch=1, chunk=2048, cached=14336, heads=32, kv_heads=8, type="bf16", page=64),
        # A chunk of a prompt together with the decode steps of 30 other sequences; small heads, odd pages.
        _attention("mixed-1001", batch=1, decodes=30, chunk=1001, cached=4999, ragged=4, heads=24, kv_heads=8, dim=64, type="fp16", page=24),
        # Prompts whose scores are capped, in a sliding window.
        _attention("capped-window-4096", batch=2, chunk=4096, cached=0, heads=16, kv_heads=8, type="bf16", softcap=50.0, window=2048, page=32),
        # Ragged prompts with a distance bias and a prefix that every token sees; ungrouped heads.
        _attention("biased-prefix", batch=5, chunk=777, cached=1500, ragged=5, heads=12, kv_heads=12, type="fp16", slopes=True, prefix=300),
    ]


def _log(rng, lo, hi, multiple=1):
    """A size spread over the logarithm of [lo, hi], in whole multiples."""
    return max(-(-lo // multiple), min(hi // multiple, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple))) * multiple


def _drawn(rng):
    kind = rng.choice(["rotate", "append", "attention", "attention", "attention"])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 7, 8])
    rotary = dict(layout=rng.choice(["half", "half", "interleaved"]), scaling=rng.choice(["none", "none", "linear", "ntk", "bands", "yarn"]),
                  base=rng.choice([1e4, 5e5, 1e6]))
    type_ = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "rotate":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        tokens = _log(rng, 1, 12000)
        return dict(kind=kind, tokens=tokens, heads=_log(rng, 1, 40), dim=dim, rotated=rng.choice([dim, dim, dim // 32 * 16]), type=type_,
                    far=max(tokens, _log(rng, 1000, 1000000)), **rotary)
    batch = _log(rng, 1, 128)
    chunk = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
    seqs = dict(batch=batch, decodes=rng.choice([0, 0, 0, rng.randint(1, 40)]), chunk=chunk, cached=_log(rng, 1, 32768) - 1, ragged=rng.randint(1, 1 << 20),
                heads=heads, kv_heads=kv, dim=dim, page=rng.choice([8, 16, 16, 24, 32, 64, 100, 128]), type=type_)
    if kind == "append":
        return dict(kind=kind, cache=rng.choice([type_, "bf16"]), rotated=rng.choice([dim, dim, dim // 2]), **seqs, **rotary)
    return dict(kind=kind, pad=rng.choice([0, 0, rng.randint(1, 9)]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]),
                window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]), slopes=rng.random() < 0.2, prefix=rng.choice([0, 0, 0, _log(rng, 1, 2000)]), **seqs)


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        flops = 2.0e11 if c["type"] != "fp32" else 1.0e10
        if w["bytes"] <= 6.0e8 and w["flops"] <= flops and (c["kind"] == "rotate" or _pages(c) * c["page"] * c["kv_heads"] * c["dim"] <= 6.0e8):
            return c


# ------------------------------------------------------------------------------------------------------------ sizes

def _lengths(c):
    """(new tokens, length with them) of each sequence: the first as large as the case says, the others ragged."""
    rng = random.Random(c["ragged"])
    out = []
    for i in range(c["batch"] + c["decodes"]):
        whole = i == 0 or not c["ragged"]
        new = c["chunk"] if whole else 1 if i >= c["batch"] else _log(rng, 1, c["chunk"])
        cached = c["cached"] if whole else _log(rng, 1, c["cached"] + 1) - 1
        out.append((new, cached + new))
    return out


def _prefixes(c):
    """Keys that every token of a sequence sees: the first sequence's as many as the case says."""
    rng = random.Random(c["ragged"] + 1)
    return [c["prefix"] if b == 0 else rng.randint(0, c["prefix"]) for b in range(c["batch"] + c["decodes"])]


def _pages(c):
    return sum(-(-length // c["page"]) for _, length in _lengths(c))


def _first_key(c, n):
    return max(0, n - c["window"] + 1) if c["window"] else 0


def _visible(c, new, length, prefix):
    """Keys seen by each new token of a sequence, summed, and the keys that any of them sees."""
    p = min(prefix, length)
    pairs = 0
    for n in range(length - new, length):
        lo, hi = _first_key(c, n), n + 1
        pairs += hi - lo + max(0, p - hi) + min(p, lo)
    lo = _first_key(c, length - new)
    return pairs, length - lo + min(p, lo)


def work(case):
    c = case
    if c["kind"] == "rotate":
        return {"bytes": 2 * BYTES[c["type"]] * c["tokens"] * c["heads"] * c["dim"] + 4 * c["tokens"], "flops": 3.0 * c["tokens"] * c["heads"] * c["rotated"]}
    seqs = _lengths(c)
    tokens, e = sum(new for new, _ in seqs), BYTES[c["type"]]
    if c["kind"] == "append":
        values = tokens * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": values * (e + BYTES[c["cache"]]), "flops": 3.0 * tokens * (c["heads"] + c["kv_heads"]) * c["rotated"]}
    seen = [_visible(c, new, length, prefix) for (new, length), prefix in zip(seqs, _prefixes(c))]
    return {"bytes": e * c["dim"] * (2 * tokens * c["heads"] + 2 * c["kv_heads"] * sum(keys for _, keys in seen)),
            "flops": 4.0 * c["dim"] * c["heads"] * sum(pairs for pairs, _ in seen)}


# ------------------------------------------------------------------------------------------------------------ inputs

SCALING = {"none": {}, "linear": dict(factor=4.0), "ntk": dict(factor=4.0), "bands": dict(factor=8.0, original=8192, low=1.0, high=4.0),
           "yarn": dict(factor=4.0, original=4096, fast=32.0, slow=1.0)}


def prepare(case, seed):
    c = case
    g = torch.Generator(DEV).manual_seed(seed)
    t = TYPES[c["type"]]

    def normal(*shape, dtype=t):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    s = {"case": c}
    if c["kind"] == "rotate":
        # Queries as a projection leaves them, and positions anywhere up to the context's end.
        s["x"] = normal(c["tokens"], c["heads"], c["dim"])
        s["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        s["positions"][-1] = c["far"] - 1
        return _handles(s)
    seqs = _lengths(c)
    tokens, pages = sum(new for new, _ in seqs), _pages(c)
    # Pages as an allocator that has run for a while hands them out: in no order, a few of no sequence.
    order = torch.randperm(pages + 3, generator=g, device=DEV).to(torch.int32).cpu()
    width = max(-(-length // c["page"]) for _, length in seqs)
    table, at, starts = torch.zeros(len(seqs), width, dtype=torch.int32), 0, [0]
    for b, (new, length) in enumerate(seqs):
        n = -(-length // c["page"])
        table[b, :n] = order[at:at + n]
        at += n
        starts.append(starts[-1] + new)
    s["table"] = table.to(DEV)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["lengths"] = torch.tensor([length for _, length in seqs], dtype=torch.int32, device=DEV)
    shape = (pages + 3, c["page"], c["kv_heads"], c["dim"])
    ct = TYPES[c.get("cache", c["type"])]
    s["k_pages"], s["v_pages"] = normal(*shape, dtype=ct), normal(*shape, dtype=ct)
    if c["kind"] == "append":
        # q, k and v as views of one projection's output.
        qkv = normal(tokens, c["heads"] + 2 * c["kv_heads"], c["dim"])
        s["q"], s["k"], s["v"] = qkv.split((c["heads"], c["kv_heads"], c["kv_heads"]), 1)
        s["q_out"] = torch.zeros(tokens, c["heads"], c["dim"], dtype=ct, device=DEV)
        return _handles(s)
    s["q"] = normal(tokens + c["pad"], c["heads"], c["dim"])
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["heads"] + 1, device=DEV) / c["heads"]).float() if c["slopes"] else None
    s["prefix"] = torch.tensor(_prefixes(c), dtype=torch.int32, device=DEV) if c["prefix"] else None
    return _handles(s)


def _handles(s):
    """The package's handles, which a program keeps over its steps: frequencies, the cache's pages, the batch."""
    if own and "handles" not in s:
        import __graft_entry__
        __graft_entry__.load_package()
        from comfyui_rdna2_attention_amd import paged_kv, rotary
        c, h = s["case"], {}
        if c["kind"] != "attention":
            h["rotary"] = rotary.Rotary(c["rotated"], base=c["base"], layout=c["layout"], scaling=None if c["scaling"] == "none" else c["scaling"],
                                        device=DEV, **SCALING[c["scaling"]])
        if c["kind"] != "rotate":
            h["cache"] = paged_kv.Cache(s["k_pages"], s["v_pages"])
            h["batch"] = paged_kv.Batch(s["table"], s["starts"], s["lengths"])
        s["handles"] = h
    return s


# ------------------------------------------------------------------------------------------------------------ one pass

def run(state):
    s = _handles(state)
    c = s["case"]
    if own:
        from comfyui_rdna2_attention_amd import paged_kv, rotary
        h = s["handles"]
        if c["kind"] == "rotate":
            return rotary.rotate(s["x"], s["positions"], h["rotary"])
        if c["kind"] == "append":
            paged_kv.append(h["cache"], h["batch"], s["k"], s["v"], rotary=h["rotary"], q=s["q"], q_out=s["q_out"])
            return s["q_out"], s["k_pages"], s["v_pages"]
        return paged_kv.attention(h["cache"], h["batch"], s["q"], scale=c["dim"] ** -0.5, softcap=c["softcap"], window=c["window"], slopes=s["slopes"],
                                  prefix=s["prefix"])
    if c["kind"] == "rotate":
        return _plain_rotate(c, s["x"], s["positions"]).to(s["x"].dtype)
    if c["kind"] == "append":
        return _plain_append(c, s)
    return _plain_attention(c, s)


def _plain_frequencies(c):
    """Radians per position of each pair."""
    r, base, o = c["rotated"], c["base"], SCALING[c["scaling"]]
    i = torch.arange(r // 2, dtype=torch.float64, device=DEV)
    if c["scaling"] == "ntk":
        base = base * o["factor"] ** (r / (r - 2))
    f = base ** (-2.0 * i / r)
    factor = 1.0
    if c["scaling"] == "linear":
        f = f / o["factor"]
    elif c["scaling"] == "bands":
        turns = o["original"] * f / (2 * math.pi)  # over the original context
        keep = ((turns - o["low"]) / (o["high"] - o["low"])).clamp(0, 1)
        f = f * keep + f / o["factor"] * (1 - keep)
    elif c["scaling"] == "yarn":
        pair = lambda turns: r * math.log(o["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(o["fast"])), 0), min(math.ceil(pair(o["slow"])), r - 1)
        stretch = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - stretch) + f / o["factor"] * stretch
        factor = 0.1 * math.log(o["factor"]) + 1.0
    return f, factor


def _plain_rotate(c, x, positions):
    """fp32 rotation; the angles in 64 bits (far positions)."""
    f, factor = _plain_frequencies(c)
    angle = positions.double()[:, None, None] * f
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    x, r = x.float(), c["rotated"]
    y = x.clone()
    if c["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_append(c, s):
    t = torch.arange(s["k"].shape[0], device=DEV)
    b = torch.searchsorted(s["starts"][1:].contiguous(), t.to(torch.int32), right=True)
    position = s["lengths"][b] - s["starts"][b + 1] + t
    page, row = s["table"][b, position // c["page"]].long(), position % c["page"]
    s["q_out"].copy_(_plain_rotate(c, s["q"], position))
    s["k_pages"][page, row] = _plain_rotate(c, s["k"], position).to(s["k_pages"].dtype)
    s["v_pages"][page, row] = s["v"].to(s["v_pages"].dtype)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _plain_attention(c, s):
    H, kv, D = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros_like(s["q"])
    at = 0
    for b, (new, length) in enumerate(_lengths(c)):
        pages = s["table"][b, :-(-length // c["page"])].long()
        keys = s["k_pages"][pages].flatten(0, 1)[:length].float().permute(1, 2, 0).contiguous()  # (kv, D, length)
        values = s["v_pages"][pages].flatten(0, 1)[:length].float().transpose(0, 1).contiguous()
        j = torch.arange(length, device=DEV)
        step = max(1, (1 << 28) // (H * length))
        for i in range(0, new, step):
            m = min(step, new - i)
            n = torch.arange(length - new + i, length - new + i + m, device=DEV)[:, None]
            q = s["q"][at + i:at + i + m].float().view(m, kv, H // kv, D).permute(1, 2, 0, 3).reshape(kv, -1, D)
            x = torch.bmm(q, keys).view(H, m, length) * D ** -0.5
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            if c["slopes"]:
                x = x - s["slopes"][:, None, None] * (n - j).abs()
            see = j <= n
            if c["window"]:
                see = see & (n - j < c["window"])
            if c["prefix"]:
                see = see | (j < s["prefix"][b])
            x = torch.where(see, x, -torch.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.bmm(p.view(kv, -1, length), values).view(H, m, D) / p.sum(-1, keepdim=True)
            out[at + i:at + i + m] = o.transpose(0, 1).to(out.dtype)
        at += new
    return out


# ------------------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    c = case
    if work(c)["flops"] > 4e12:
        return None
    s = prepare(c, seed)
    if c["kind"] == "rotate":
        return _turn(c, s["x"].double(), s["positions"])
    out = s["q"].new_zeros(s["q"].shape, dtype=torch.float64)
    table, k_pages, v_pages = s["table"].long(), s["k_pages"].double(), s["v_pages"].double()
    group, at = c["heads"] // c["kv_heads"], 0
    for b, (new, length) in enumerate(_lengths(c)):
        slots = torch.arange(length, device=DEV)
        page, row = table[b, slots // c["page"]], slots % c["page"]
        mine = slice(at, at + new)
        at += new
        if c["kind"] == "append":
            n = slots[length - new:]
            k_pages[page[n], row[n]] = _turn(c, s["k"][mine].double(), n)
            v_pages[page[n], row[n]] = s["v"][mine].double()
            out[mine] = _turn(c, s["q"][mine].double(), n)
            continue
        for h in range(c["kv_heads"]):
            K, V = k_pages[page, row, h], v_pages[page, row, h]
            for i in range(0, new, 2048):
                n = slots[length - new + i:length - new + min(new, i + 2048)]
                gap = n[:, None] - slots[None]
                hidden = gap < 0
                if c["window"]:
                    hidden |= gap >= c["window"]
                if c["prefix"]:
                    hidden &= (slots >= s["prefix"][b])[None]
                for head in range(h * group, (h + 1) * group):
                    rows = slice(mine.start + i, mine.start + i + len(n))
                    score = s["q"][rows, head].double() @ K.T / math.sqrt(c["dim"])
                    if c["softcap"]:
                        score = c["softcap"] * torch.tanh(score / c["softcap"])
                    if c["slopes"]:
                        score -= s["slopes"][head].double() * gap.abs()
                    out[rows, head] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ V
    return (out, k_pages, v_pages) if c["kind"] == "append" else out


def _turn(c, x, positions):
    """Each pair as a complex number, times e^(i angle)."""
    R, o = c["rotated"], SCALING[c["scaling"]]
    freq, gain = [], 1.0
    for i in range(R // 2):
        base = c["base"] * (o["factor"] ** (R / (R - 2)) if c["scaling"] == "ntk" else 1.0)
        w = math.pow(base, -2.0 * i / R)
        slow = w / o.get("factor", 1.0)
        if c["scaling"] == "linear":
            w = slow
        elif c["scaling"] == "bands":
            length = 2 * math.pi / w
            if length > o["original"] / o["low"]:
                w = slow
            elif length >= o["original"] / o["high"]:
                mix = (o["original"] / length - o["low"]) / (o["high"] - o["low"])
                w = (1 - mix) * slow + mix * w
        elif c["scaling"] == "yarn":
            first, last = (R * math.log(o["original"] / (2 * math.pi * n)) / (2 * math.log(c["base"])) for n in (o["fast"], o["slow"]))
            first, last = max(math.floor(first), 0), min(math.ceil(last), R - 1)
            ramp = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
            w = slow * ramp + w * (1 - ramp)
            gain = 0.1 * math.log(o["factor"]) + 1.0
        freq.append(w)
    angle = positions.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.full_like(angle, gain), angle)
    head, rest = x[..., :R], x[..., R:]
    if c["layout"] == "half":
        z = torch.complex(head[..., :R // 2].contiguous(), head[..., R // 2:].contiguous()) * turn
        head = torch.cat((z.real, z.imag), -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], R // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat((head, rest), -1)
