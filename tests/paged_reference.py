"""Plain 64-bit forms of the paged cache's operators, on the CPU, for the tests: one token, one head at a time where that is plainest."""
import math

import torch


def turned(x, positions, rotary, inverse=False):
    """rotary.rotate of x (tokens, heads, D): (values, the bound on what 32-bit turns are off by)."""
    x, turns = x.double(), rotary.turns.cpu()
    half = rotary.dim // 2
    angle = positions.cpu().double()[:, None] * turns * (2 * math.pi) * (-1 if inverse else 1)
    c, s = (torch.cos(angle) * rotary.factor)[:, None], (torch.sin(angle) * rotary.factor)[:, None]
    i = torch.arange(half)
    at, to = (2 * i, 2 * i + 1) if rotary.layout == "interleaved" else (i, i + half)
    a, b = x[..., at], x[..., to]
    y, off = x.clone(), torch.zeros_like(x)
    y[..., at], y[..., to] = a * c - b * s, a * s + b * c
    # Four roundings (cosine or sine, product, sum) of at most 2^-24 of |a| + |b| each, and the angle's: half of 2^-24 of a quarter turn
    # of at most half, times pi / 2, and the series' 2 to 3 last places: together below 8 x 2^-24 of (|a| + |b|) factor.
    size = (a.abs() + b.abs()) * rotary.factor * 8 * 2.0 ** -24
    off[..., at], off[..., to] = size, size
    return y, off


def rounding(t, dtype):
    """Half a step of dtype at t, and half its smallest one."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) * 1.001 + (info.smallest_normal * info.eps / 2)


def sequences(starts, lengths, tokens):
    """(b, first row, new tokens, position of the first) of a batch."""
    for b in range(len(lengths)):
        first, end = min(max(int(starts[b]), 0), tokens), min(max(int(starts[b + 1]), 0), tokens)
        new = max(end - first, 0)
        yield b, first, new, max(int(lengths[b]), 0) - new


def appended(k, v, k_pages, v_pages, table, starts, lengths, rotary):
    """append's pages in 64 bits and the bound on their 32-bit turns: (k, v, bound of k), for the pages in 64 bits."""
    k_pages, v_pages = k_pages.double().clone(), v_pages.double().clone()
    off = torch.zeros_like(k_pages)
    P, S = k_pages.shape[:2]
    for b, first, new, p0 in sequences(starts, lengths, len(k)):
        for i in range(new):
            n = int(lengths[b]) - new + i
            if n < 0 or n // S >= table.shape[1] or not 0 <= int(table[b, n // S]) < P:
                continue
            page = int(table[b, n // S])
            kt, o = (k[first + i:first + i + 1].double(), 0.0) if rotary is None else turned(k[first + i:first + i + 1], torch.tensor([n]), rotary)
            k_pages[page, n % S], off[page, n % S] = kt[0], o if rotary is None else o[0]
            v_pages[page, n % S] = v[first + i].double()
    return k_pages, v_pages, off


def attended(q, k_pages, v_pages, table, starts, lengths, scale=None, softcap=0.0, window=0, slopes=None, prefix=None):
    """paged_kv.attention in 64 bits and the bound on what its arithmetic is off by before the last rounding, both (tokens, heads, D),
    rows of no sequence 0; and which rows belong to a sequence. Tokens together where every value that any of them sees is finite, else one
    by one, with only what that one sees."""
    T, H, D = q.shape
    P, S, Hkv, _ = k_pages.shape
    scale = D ** -0.5 if scale is None else scale
    out, off = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    mine = torch.zeros(T, dtype=torch.bool)
    for b, first, new, p0 in sequences(starts, lengths, T):
        mine[first:first + new] = True
        keys = min(max(int(lengths[b]), 0), table.shape[1] * S)
        j = torch.arange(keys)
        page = table[b].long()[j // S]
        there = (page >= 0) & (page < P)
        page = torch.where(there, page, 0)
        K, V = k_pages[page, j % S].double(), v_pages[page, j % S].double()  # (keys, Hkv, D)
        n = torch.arange(p0, p0 + new)[:, None]
        see = j <= n
        if window:
            see &= n - j < window
        if prefix is not None:
            see |= j < int(prefix[b])
        see &= there
        if not see.any():
            continue
        used = see.any(0)
        K, V, see, j = K[used], V[used], see[:, used], j[used]
        rows = slice(first, first + new)
        if torch.isfinite(K).all() and torch.isfinite(V).all():
            out[rows], off[rows] = _rows(q[rows], K, V, see, n, j, scale, softcap, slopes)
        else:
            for i in range(new):
                one, s = slice(first + i, first + i + 1), see[i]
                if s.any():
                    out[one], off[one] = _rows(q[one], K[s], V[s], see[i:i + 1, s], n[i:i + 1], j[s], scale, softcap, slopes)
    return out, off, mine


def _rows(q, K, V, see, n, j, scale, softcap, slopes):
    """Attention of q (rows, heads, D) over K, V (keys, Hkv, D), row i over the keys of see[i], and its bound."""
    R, H, D = q.shape
    Hkv, keys = K.shape[1], K.shape[0]
    low = q.dtype != torch.float32
    u = torch.finfo(q.dtype).eps / 2 if low else 0.0
    grouped = lambda t: t.view(R, Hkv, H // Hkv, -1).permute(1, 2, 0, 3).reshape(Hkv, -1, t.shape[-1])  # noqa: E731
    back = lambda t: t.view(Hkv, H // Hkv, R, -1).permute(2, 0, 1, 3).reshape(R, H, -1)  # noqa: E731
    Kt, Vt = K.permute(1, 2, 0).contiguous(), V.permute(1, 0, 2).contiguous()
    qd = grouped(q.double())
    x = back(torch.bmm(qd, Kt)) * scale  # (rows, heads, keys)
    size = back(torch.bmm(qd.abs(), Kt.abs())) * scale
    hidden = ~see[:, None]
    # Scores: D products and sums and the scale in 32 bits; tanh's and the bias's own roundings.
    delta = (D + 4) * 2.0 ** -24 * size.masked_fill(hidden, 0).amax(2, keepdim=True)
    if softcap:
        x = softcap * torch.tanh(x / softcap)
        delta = delta + softcap * 4e-7 * (1 if low else 0.5)
    if slopes is not None:
        bias = slopes.double()[None, :, None] * (n - j).abs().double()[:, None]
        x = x - bias
        delta = delta + 2.0 ** -23 * bias.abs().masked_fill(hidden, 0).amax(2, keepdim=True)
    delta = delta + 2.0 ** -23 * x.abs().masked_fill(hidden, 0).amax(2, keepdim=True) + 2.0 ** -21  # to the log2 domain, less the maximum; 2^x
    some = see.any(1)[:, None, None]
    w = torch.softmax(torch.where(some, x.masked_fill(hidden, -math.inf), 0.0), 2) * some
    out, spread = back(torch.bmm(grouped(w), Vt)), back(torch.bmm(grouped(w), Vt.abs()))
    # Each weight is off by delta and its rounding, in the numerator and in the sum; sums of the keys' terms in 32 bits.
    return out, spread * 2 * (delta + u + keys * 2.0 ** -24) * 1.01
