"""Serving and training steps around a key/value cache held in 8 bits, for timing: norms of queries and keys with the rotary turn (and their
gradients), appends that quantize on the way, reading a cache back, and attention over it.

The cache's codes are int8 with a scale in fp32 for each block of tokens and KV head. A case is a dict with a "kind" (norm, append, read,
attention) and its sizes; `listed()` holds the cases that are quoted and `draw(rng)` gives more of the same ranges. `prepare` makes
on the GPU what a program has in hand, `run` is one pass -- the plain form in elementary torch operations, or with `own` the package's
calls -- and `exact` the same values in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-6
FLOOR = 1e-30  # the least scale


# ------------------------------------------------------------------------------------------------------------ the cases

def _norm(name, **c):
    return dict(dict(kind="norm", rotated=c["dim"], layout="half", base=1e6, weights=c["type"], train=False), **c, name=name)


def _append(name, **c):
    return dict(dict(kind="append", ragged=0, dim=128, rotated=128, layout="half", base=1e6, page=64, block=32, norm=False), **c, name=name)


def _read(name, **c):
    return dict(dict(kind="read", ragged=0, dim=128, page=64, block=32), **c, name=name)


def _attention(name, **c):
    return dict(dict(kind="attention", ragged=0, dim=128, page=64, block=32, softcap=0.0, window=0, slopes=False, prefix=0), **c, name=name)


def listed():
    return [
        # One token's queries and keys at a far position: the smallest call, bound by its launch.
        _norm("norm-token", tokens=1, heads=32, kv_heads=8, dim=128, far=131072, type="bf16"),
        # A training step's forward and backward in fp32: an odd number of tokens, interleaved pairs in half of each head.
        _norm("norm-train-1101-fp32", tokens=1101, heads=16, kv_heads=8, dim=128, rotated=64, layout="interleaved", base=1e4, far=1101, type="fp32", train=True),
        # The same for a batch of long sequences in bf16, with its weights in fp32.
        _norm("norm-train-8192", tokens=8192, heads=32, kv_heads=8, dim=128, far=8192, type="bf16", weights="fp32", train=True),
        # A decode step of 64 sequences: each token normed, turned and quantized into its block, and the blocks read back.
        _append("append-decode-64", batch=64, chunk=1, cached=8191, ragged=1, heads=32, kv_heads=8, type="bf16", out="bf16", norm=True),
        # Prompt chunks of three sequences from the fp32 linears of text generation, into small blocks of odd pages of small heads.
        _append("append-ragged-fp32", batch=3, chunk=2049, cached=1000, ragged=2, heads=24, kv_heads=8, dim=64, rotated=64, layout="interleaved",
                base=1e4, page=48, block=16, type="fp32", out="fp16"),
        # A whole long prompt.
        _append("append-16384", batch=1, chunk=16384, cached=0, heads=32, kv_heads=8, type="fp16", out="fp16", block=64, norm=True),
        # The cached part of one short sequence, as another program takes it over.
        _read("read-257", batch=1, cached=257, kv_heads=8, block=16, page=16, out="fp16"),
        # 24 sequences' caches read back for a program that keeps them in bf16.
        _read("read-24", batch=24, cached=8192, ragged=3, kv_heads=8, out="bf16"),
        # One token of one sequence: the smallest attention, bound by latency.
        _attention("decode-1", batch=1, chunk=1, cached=2047, heads=32, kv_heads=8, type="fp16", block=16, page=16),
        # One token each of 64 sequences: a serving step, bound by the cache's bytes.
        _attention("decode-64", batch=64, chunk=1, cached=8191, heads=32, kv_heads=8, type="bf16"),
        # A chunk of a prompt over what earlier chunks left in the cache: the largest.
        _attention("chunk-2048", batch=1, chunk=2048, cached=14336, heads=32, kv_heads=8, type="bf16", block=64),
        # Ragged prompts of small ungrouped heads, capped scores in a sliding window, with a prefix that every token sees.
        _attention("capped-window-prefix", batch=5, chunk=777, cached=1500, ragged=5, heads=12, kv_heads=12, dim=64, type="fp16", page=48, block=16,
                   softcap=50.0, window=600, prefix=40),
    ]


def _log(rng, lo, hi, multiple=1):
    """A size spread over the logarithm of [lo, hi], in whole multiples."""
    return max(-(-lo // multiple), min(hi // multiple, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple))) * multiple


def _drawn(rng):
    kind = rng.choice(["norm", "norm", "append", "append", "read", "attention", "attention", "attention"])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 7, 8])
    type_ = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    turn = dict(layout=rng.choice(["half", "half", "interleaved"]), base=rng.choice([1e4, 5e5, 1e6]))
    if kind == "norm":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        tokens = _log(rng, 1, 9000)
        return dict(kind=kind, tokens=tokens, heads=heads, kv_heads=kv, dim=dim, rotated=rng.choice([dim, dim, dim // 32 * 16]), type=type_,
                    weights=rng.choice([type_, "fp32"]), far=max(tokens, _log(rng, 1000, 1000000)), train=rng.random() < 0.6, **turn)
    block = rng.choice([16, 32, 32, 64])
    seqs = dict(batch=_log(rng, 1, 128), cached=_log(rng, 1, 32768) - 1, ragged=rng.randint(1, 1 << 20), kv_heads=kv, dim=dim,
                page=block * rng.choice([1, 1, 2, 3, 4]), block=block)
    if kind == "read":
        return dict(kind=kind, out=rng.choice(["bf16", "bf16", "fp16"]), **dict(seqs, cached=seqs["cached"] + 1))
    chunk = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
    if kind == "append":
        out = type_ if type_ != "fp32" else rng.choice(["bf16", "fp16"])
        return dict(kind=kind, chunk=chunk, heads=heads, type=type_, out=out, rotated=rng.choice([dim, dim, dim // 2]), norm=rng.random() < 0.5, **seqs, **turn)
    return dict(kind=kind, chunk=chunk, heads=heads, type=type_ if type_ != "fp32" else "bf16", softcap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]),
                window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]), slopes=rng.random() < 0.2, prefix=rng.choice([0, 0, 0, _log(rng, 1, 2000)]), **seqs)


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] > 1.0e9 or w["flops"] > 2.0e11:
            continue
        if c["kind"] != "norm":
            lengths = _lengths(c)
            padded = len(lengths) * max(length for _, length in lengths)
            if _pages(c) * c["page"] * c["kv_heads"] * c["dim"] > 6.0e8 or padded * c["kv_heads"] * c["dim"] > 1.2e9:
                continue
            if c["kind"] == "attention" and padded * c["chunk"] * c["heads"] > 1.0e9:
                continue
        return c


# ------------------------------------------------------------------------------------------------------------ sizes

def _lengths(c):
    """(new tokens, length with them) of each sequence: the first as large as the case says, the others ragged (a read's tokens are all "new")."""
    rng = random.Random(c["ragged"])
    out = []
    for i in range(c["batch"]):
        whole = i == 0 or not c["ragged"]
        if c["kind"] == "read":
            n = c["cached"] if whole else _log(rng, 1, c["cached"])
            out.append((n, n))
            continue
        new = c["chunk"] if whole else _log(rng, 1, c["chunk"])
        cached = c["cached"] if whole else _log(rng, 1, c["cached"] + 1) - 1
        out.append((new, cached + new))
    return out


def _touched(c):
    """(tokens, length) of each sequence from the start of the first block that an append writes into."""
    return [(length - (length - new) // c["block"] * c["block"], length) for new, length in _lengths(c)]


def _prefixes(c):
    """Keys that every token of a sequence sees: the first sequence's as many as the case says."""
    rng = random.Random(c["ragged"] + 1)
    return [c["prefix"] if b == 0 else rng.randint(0, c["prefix"]) for b in range(c["batch"])]


def _pages(c):
    return sum(-(-length // c["page"]) for _, length in _lengths(c))


def _visible(c, new, length, prefix):
    """Keys seen by each new token of a sequence, summed, and the keys that any of them sees."""
    p, first = min(prefix, length), lambda n: max(0, n - c["window"] + 1) if c["window"] else 0
    pairs = 0
    for n in range(length - new, length):
        lo, hi = first(n), n + 1
        pairs += hi - lo + max(0, p - hi) + min(p, lo)
    lo = first(length - new)
    return pairs, length - lo + min(p, lo)


def work(case):
    c = case
    if c["kind"] == "norm":
        values = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        # Forward: in and out. Backward: the input and the output's gradient in, the input's gradient out.
        return {"bytes": values * BYTES[c["type"]] * (5 if c["train"] else 2) + 4 * c["tokens"], "flops": (25.0 if c["train"] else 8.0) * values}
    seqs, kv = _lengths(c), c["kv_heads"] * c["dim"]
    tokens, scales = sum(new for new, _ in seqs), 8.0 * c["kv_heads"] / c["block"]
    if c["kind"] == "read":
        return {"bytes": tokens * (2 * kv * (1 + BYTES[c["out"]]) + scales), "flops": 2.0 * tokens * kv}
    if c["kind"] == "append":
        rows, q = sum(n for n, _ in _touched(c)), c["heads"] * c["dim"]
        into = tokens * ((q + 2 * kv) * BYTES[c["type"]] + q * BYTES[c["out"]] + 2 * kv + scales)
        return {"bytes": into + rows * (2 * kv * (1 + BYTES[c["out"]]) + scales), "flops": 8.0 * tokens * (q + 2 * kv)}
    seen = [_visible(c, new, length, prefix) for (new, length), prefix in zip(seqs, _prefixes(c))]
    keys = sum(keys for _, keys in seen)
    return {"bytes": 2 * BYTES[c["type"]] * tokens * c["heads"] * c["dim"] + keys * (2 * kv + scales), "flops": 4.0 * c["dim"] * c["heads"] * sum(pairs for pairs, _ in seen)}


# ------------------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(DEV).manual_seed(seed)

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    s, D = {"case": c}, c["dim"]
    if c["kind"] in ("norm", "append"):
        s["weights"] = [1.0 + 0.2 * normal(D, dtype=torch.float32) for _ in range(2)]
        s["weights"] = [w.to(TYPES[c.get("weights", c["type"])]) for w in s["weights"]]
    if c["kind"] == "norm":
        # Queries and keys as one projection leaves them, of sizes that differ from channel to channel; positions anywhere up to the context's end.
        t = TYPES[c["type"]]
        size = torch.exp(0.7 * normal(c["heads"] + c["kv_heads"], D, dtype=torch.float32))
        qk = (normal(c["tokens"], c["heads"] + c["kv_heads"], D, dtype=torch.float32) * size).to(t)
        s["q"], s["k"] = qk.split((c["heads"], c["kv_heads"]), 1)
        s["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        s["positions"][-1] = c["far"] - 1
        if c["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["weights"] = [w.requires_grad_() for w in s["weights"]]
            s["gradients"] = [normal(c["tokens"], h, D, dtype=t) for h in (c["heads"], c["kv_heads"])]
        return s
    seqs = _lengths(c)
    pages = _pages(c) + 3
    # Pages as an allocator that has run for a while hands them out: in no order, a few of no sequence.
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
    width = max(-(-length // c["page"]) for _, length in seqs)
    table, at = torch.zeros(len(seqs), width, dtype=torch.int32), 0
    for b, (_, length) in enumerate(seqs):
        n = -(-length // c["page"])
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = table.to(DEV)
    s["starts"] = _starts(seqs)
    s["lengths"] = torch.tensor([length for _, length in seqs], dtype=torch.int32, device=DEV)
    # Blocks of normal values, quantized by their largest: codes of about a third of 127, scales that differ by block and head.
    for x in ("k", "v"):
        s[x + "_codes"] = (normal(pages, c["page"], c["kv_heads"], D, dtype=torch.float32) * 36).round_().clamp_(-127, 127).to(torch.int8)
        s[x + "_scales"] = 0.03 * torch.exp(0.3 * normal(pages, c["page"] // c["block"], c["kv_heads"], dtype=torch.float32))
    tokens = sum(new for new, _ in seqs)
    if c["kind"] == "append":
        # q, k and v as views of one projection's output, some tokens larger than others.
        size = torch.exp(0.4 * normal(tokens, 1, 1, dtype=torch.float32))
        qkv = (normal(tokens, c["heads"] + 2 * c["kv_heads"], D, dtype=torch.float32) * size).to(TYPES[c["type"]])
        s["q"], s["k"], s["v"] = qkv.split((c["heads"], c["kv_heads"], c["kv_heads"]), 1)
        s["q_out"] = torch.zeros(tokens, c["heads"], D, dtype=TYPES[c["out"]], device=DEV)
        s["touched"] = _starts(_touched(c))
        s["touched_tokens"] = sum(n for n, _ in _touched(c))
    if c["kind"] == "read":
        s["tokens"] = tokens
    if c["kind"] == "attention":
        s["q"] = normal(tokens, c["heads"], D, dtype=TYPES[c["type"]])
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["heads"] + 1, device=DEV) / c["heads"]).float() if c["slopes"] else None
        s["prefix"] = torch.tensor(_prefixes(c), dtype=torch.int32, device=DEV) if c["prefix"] else None
    return s


def _starts(seqs):
    starts = [0]
    for new, _ in seqs:
        starts.append(starts[-1] + new)
    return torch.tensor(starts, dtype=torch.int32, device=DEV)


def _handles(s):
    """The package's handles, which a program keeps over its steps: frequencies, norms, the cache's pages, the batch."""
    if "handles" not in s:
        import __graft_entry__
        __graft_entry__.load_package()
        from comfyui_rdna2_attention_amd import paged_kv, rotary
        c, h = s["case"], {}
        if c["kind"] in ("norm", "append"):
            h["rotary"] = rotary.Rotary(c["rotated"], base=c["base"], layout=c["layout"], device=DEV)
            h["norm"] = rotary.HeadNorm(*s["weights"], eps=EPS) if c.get("norm", True) else None
        if c["kind"] != "norm":
            h["cache"] = paged_kv.QuantizedCache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
            h["batch"] = paged_kv.Batch(s["table"], s["starts"], s["lengths"])
        if c["kind"] == "append":
            h["touched"] = paged_kv.Batch(s["table"], s["touched"], s["lengths"])
        s["handles"] = h
    return s["handles"]


# ------------------------------------------------------------------------------------------------------------ one pass

def run(state):
    s = state
    c = s["case"]
    if own:
        h = _handles(s)
        from comfyui_rdna2_attention_amd import paged_kv, rotary
        if c["kind"] == "norm":
            y = rotary.norm_rotate(s["q"], s["k"], s["positions"], h["rotary"], h["norm"])
            return _with_gradients(s, y) if c["train"] else y
        if c["kind"] == "append":
            paged_kv.append(h["cache"], h["batch"], s["k"], s["v"], rotary=h["rotary"], q=s["q"], q_out=s["q_out"], norm=h["norm"])
            return (s["q_out"], *paged_kv.read(h["cache"], h["touched"], s["touched_tokens"], TYPES[c["out"]]))
        if c["kind"] == "read":
            return paged_kv.read(h["cache"], h["batch"], s["tokens"], TYPES[c["out"]])
        return paged_kv.attention(h["cache"], h["batch"], s["q"], scale=c["dim"] ** -0.5, softcap=c["softcap"], window=c["window"], slopes=s["slopes"],
                                  prefix=s["prefix"])
    if c["kind"] == "norm":
        y = tuple(_plain_turn(c, _plain_norm(x, w), s["positions"]).to(x.dtype) for x, w in zip((s["q"], s["k"]), s["weights"]))
        return _with_gradients(s, y) if c["train"] else y
    if c["kind"] == "append":
        _plain_append(c, s)
        return (s["q_out"], *_plain_read(c, s, s["touched"], s["touched_tokens"]))
    if c["kind"] == "read":
        return _plain_read(c, s, s["starts"], s["tokens"])
    return _plain_attention(c, s)


def _with_gradients(s, y):
    gradients = torch.autograd.grad(y, (s["q"], s["k"], *s["weights"]), s["gradients"])
    return (*(t.detach() for t in y), *gradients)


def _plain_norm(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _plain_turn(c, x, positions):
    """The turn in 32 bits; the angles in 64 (far positions)."""
    r = c["rotated"]
    f = c["base"] ** (-2.0 * torch.arange(r // 2, dtype=torch.float64, device=DEV) / r)
    angle = positions.double()[:, None, None] * f
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if c["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, x[..., r:]), -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), x[..., r:]), -1)


def _rows(c, s, starts, tokens):
    """Sequence, position, page and row of each of a batch's tokens."""
    t = torch.arange(tokens, device=DEV)
    b = torch.searchsorted(starts[1:].contiguous(), t.to(torch.int32), right=True)
    position = s["lengths"][b] - starts[b + 1] + t
    return b, position, s["table"][b, position // c["page"]].long(), position % c["page"]


def _plain_append(c, s):
    b, position, page, row = _rows(c, s, s["starts"], s["k"].shape[0])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q, k = _plain_norm(q, s["weights"][0]), _plain_norm(k, s["weights"][1])
    s["q_out"].copy_(_plain_turn(c, q, position))
    per = c["page"] // c["block"]
    block, offset = page * per + row // c["block"], row % c["block"]
    first = s["starts"][:-1].long()  # each sequence's first new token: its block may hold older ones
    for x, codes, scales in ((_plain_turn(c, k, position), s["k_codes"], s["k_scales"]), (v, s["v_codes"], s["v_scales"])):
        blocks, old = codes.view(-1, c["block"], *codes.shape[2:]), scales.view(-1, scales.shape[-1])
        most = torch.zeros_like(old).scatter_reduce_(0, block[:, None].expand(-1, old.shape[1]), x.abs().amax(-1), "amax")
        new = torch.clamp(most / 127, min=FLOOR)
        at = block[first]
        kept = torch.where(offset[first][:, None] > 0, old[at], 0.0)
        new[at] = torch.maximum(new[at], kept)
        blocks[at] = torch.round(blocks[at].float() * (kept / new[at])[:, None, :, None]).to(torch.int8)
        codes[page, row] = torch.round(x / new[block][..., None]).clamp(-127, 127).to(torch.int8)
        old[block] = new[block]


def _plain_read(c, s, starts, tokens):
    _, _, page, row = _rows(c, s, starts, tokens)
    return tuple((s[x + "_codes"][page, row].float() * s[x + "_scales"][page, row // c["block"]][..., None]).to(TYPES[c["out"]]) for x in ("k", "v"))


def _plain_attention(c, s):
    """All sequences padded to the longest, in 32 bits."""
    H, kv, D, B = c["heads"], c["kv_heads"], c["dim"], c["batch"]
    new, longest = (max(x[i] for x in _lengths(c)) for i in (0, 1))
    j = torch.arange(longest, device=DEV)
    page, row = s["table"][:, j // c["page"]].long(), (j % c["page"]).expand(B, -1)
    keys, values = (s[x + "_codes"][page, row].float() * s[x + "_scales"][page, row // c["block"]][..., None] for x in ("k", "v"))
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(new, device=DEV)
    rows = (s["starts"][:-1, None] + torch.minimum(i, counts[:, None] - 1)).long()  # (B, new), the last one again where a sequence has fewer
    n = (s["lengths"].long() - counts)[:, None] + torch.minimum(i, counts[:, None] - 1)
    q = s["q"][rows].float().view(B, new, kv, H // kv, D).permute(0, 2, 3, 1, 4).reshape(B * kv, -1, D)
    x = torch.bmm(q, keys.permute(0, 2, 3, 1).reshape(B * kv, D, longest).contiguous()).view(B, H, new, longest) * D ** -0.5
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    gap = n[:, :, None] - j
    if c["slopes"]:
        x = x - s["slopes"][None, :, None, None] * gap.abs()[:, None]
    see = gap >= 0
    if c["window"]:
        see = see & (gap < c["window"])
    if c["prefix"]:
        see = see | (j < s["prefix"][:, None, None])
    see = see & (j < s["lengths"][:, None, None])
    x = torch.where(see[:, None], x, -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.bmm(p.view(B * kv, -1, longest), values.permute(0, 2, 1, 3).reshape(B * kv, longest, D)).view(B, H, new, D) / p.sum(-1, keepdim=True)
    out = torch.empty_like(s["q"])
    out[rows] = o.transpose(1, 2).to(out.dtype)
    return out


# ------------------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    c = case
    if work(c)["flops"] > 4e12:
        return None
    s = prepare(c, seed)
    if c["kind"] == "norm":
        out, grads, weights = [], [], []
        for i, x in enumerate((s["q"], s["k"])):
            x, w = x.detach().double(), s["weights"][i].detach().double()
            inv = 1.0 / (x.square().sum(-1, keepdim=True) / c["dim"] + EPS).sqrt()
            unit = x * inv
            out.append(_rotated(c, unit * w, s["positions"], 1))
            if c["train"]:
                back = _rotated(c, s["gradients"][i].double(), s["positions"], -1)
                weights.append((back * unit).sum((0, 1)))
                back = back * w
                grads.append(inv * (back - unit * (back * unit).sum(-1, keepdim=True) / c["dim"]))
        return (*out, *grads, *weights)
    codes = {x: s[x + "_codes"].double() for x in ("k", "v")}
    scales = {x: s[x + "_scales"].double() for x in ("k", "v")}
    if c["kind"] == "append":
        return _exact_append(c, s, codes, scales)
    if c["kind"] == "read":
        return _gathered(c, s, codes, scales, [(0, length) for _, length in _lengths(c)])
    out = s["q"].new_zeros(s["q"].shape, dtype=torch.float64)
    group, at = c["heads"] // c["kv_heads"], 0
    for b, (new, length) in enumerate(_lengths(c)):
        keys, values = (x.transpose(0, 1).contiguous() for x in _gathered(c, s, codes, scales, [(0, length)], b))
        slots, mine = torch.arange(length, device=DEV), slice(at, at + new)
        at += new
        gap = slots[length - new:, None] - slots
        hidden = gap < 0
        if c["window"]:
            hidden |= gap >= c["window"]
        if c["prefix"]:
            hidden &= (slots >= s["prefix"][b])[None]
        for head in range(c["heads"]):
            score = s["q"][mine, head].double() @ keys[head // group].T.contiguous() / math.sqrt(c["dim"])
            if c["softcap"]:
                score = c["softcap"] * torch.tanh(score / c["softcap"])
            if c["slopes"]:
                score -= s["slopes"][head].double() * gap.abs()
            out[mine, head] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ values[head // group]
    return out


def _gathered(c, s, codes, scales, spans, only=None):
    """The values at positions from .. to - 1 of each sequence (or of one), one sequence after the other."""
    out = []
    for x in ("k", "v"):
        parts = []
        for b, (lo, hi) in enumerate(spans):
            n = torch.arange(lo, hi, device=DEV)
            page, row = s["table"][b if only is None else only].long()[n // c["page"]], n % c["page"]
            parts.append(codes[x][page, row] * scales[x][page, row // c["block"]].unsqueeze(-1))
        out.append(torch.cat(parts))
    return tuple(out)


def _exact_append(c, s, codes, scales):
    """Block by block: the new tokens' largest value, or the scale that the block has, sets its scale."""
    seqs, at = _lengths(c), 0
    q_out = torch.zeros_like(s["q_out"], dtype=torch.float64)
    unit = lambda x, i: x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * s["weights"][i].double() if c["norm"] else x  # noqa: E731
    for b, (new, length) in enumerate(seqs):
        n, mine = torch.arange(length - new, length, device=DEV), slice(at, at + new)
        at += new
        q_out[mine] = _rotated(c, unit(s["q"][mine].double(), 0), n, 1)
        tokens = {"k": _rotated(c, unit(s["k"][mine].double(), 1), n, 1), "v": s["v"][mine].double()}
        lo = (length - new) // c["block"] * c["block"]
        blocks = -(-length // c["block"]) - lo // c["block"]
        where = torch.arange(blocks, device=DEV) * c["block"] + lo
        page, part = s["table"][b].long()[where // c["page"]], where % c["page"] // c["block"]
        for x, y in tokens.items():
            whole = y.new_zeros(blocks * c["block"], *y.shape[1:])
            whole[length - new - lo:length - lo] = y
            scale = torch.clamp(whole.view(blocks, c["block"], *y.shape[1:]).abs().amax((1, 3)) / 127, min=FLOOR)
            older = length - new - lo
            if older:
                had = scales[x][page[0], part[0]]
                scale[0] = torch.maximum(scale[0], had)
                row = (lo % c["page"]) + torch.arange(older, device=DEV)
                codes[x][page[0], row] = torch.round(codes[x][page[0], row] * (had / scale[0])[:, None])
            codes[x][s["table"][b].long()[n // c["page"]], n % c["page"]] = torch.round(y / scale[(n - lo) // c["block"]].unsqueeze(-1))
            scales[x][page, part] = scale
    return (q_out, *_gathered(c, s, codes, scales, [(length - rows, length) for rows, length in _touched(c)]))


def _rotated(c, x, positions, sign):
    """Each pair as a complex number, times e^(i angle)."""
    R = c["rotated"]
    freq = torch.tensor([math.pow(c["base"], -2.0 * i / R) for i in range(R // 2)], dtype=torch.float64, device=DEV)
    angle = positions.double()[:, None, None] * freq * sign
    turn = torch.polar(torch.ones_like(angle), angle)
    head, rest = x[..., :R], x[..., R:]
    if c["layout"] == "half":
        z = torch.complex(head[..., :R // 2].contiguous(), head[..., R // 2:].contiguous()) * turn
        head = torch.cat((z.real, z.imag), -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], R // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat((head, rest), -1)
