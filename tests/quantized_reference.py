"""Plain 64-bit forms of norm_rotate and of the quantized cache's operators, on the CPU, for the tests, with the bounds that their arithmetic in 32 bits keeps."""
import torch

from paged_reference import attended, sequences, turned

U = 2.0 ** -24  # half a step of fp32, relative


def normed(x, w, eps):
    """w x / sqrt(mean(x^2) + eps) of heads (..., D) in 64 bits, and what 32 bits are off by, relative."""
    x, w, D = x.double(), w.double(), x.shape[-1]
    y = x * (1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()) * w
    # A lane's 16 squares and the D / 16 lanes' sums of them, all positive: a rounding each; the mean, eps, root and quotient, two products.
    return y, (16 + D // 16 + 8) * U


def norm_turned(x, w, positions, rotary, eps):
    """norm_rotate of one tensor (tokens, heads, D): (values, bound)."""
    z, rel = normed(x, w, eps)
    y, off = turned(z, positions, rotary)
    return y, off + rel * turned_size(z, rotary)


def turned_size(z, rotary):
    """What the turn may make of an error of each value: its size plus its partner's, times the factor."""
    half = rotary.dim // 2
    i = torch.arange(half)
    at, to = (2 * i, 2 * i + 1) if rotary.layout == "interleaved" else (i, i + half)
    size = z.abs().clone()
    size[..., at] = size[..., to] = (z[..., at].abs() + z[..., to].abs()) * rotary.factor
    return size


def norm_turned_back(x, w, grad, positions, rotary, eps):
    """The gradients of x and w for the gradient of norm_turned's values: ((x's, bound), (w's, bound))."""
    x, w, D = x.double(), w.double(), x.shape[-1]
    inv = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    u, rel = x * inv, (16 + D // 16 + 8) * U
    g, g_off = turned(grad, positions, rotary, inverse=True)
    gw, gw_off = g * w, g_off * w.abs() + U * (g * w).abs()
    mean = (gw * u).mean(-1, keepdim=True)
    mean_off = (gw_off * u.abs() + (rel + (16 + D // 16 + 2) * U) * (gw * u).abs()).mean(-1, keepdim=True)
    gx = inv * (gw - u * mean)
    gx_off = inv * (gw_off + u.abs() * mean_off + (rel + 3 * U) * (u * mean).abs()) + (rel + 4 * U) * inv * (gw.abs() + (u * mean).abs())
    terms = g * u
    # Sums of all terms in some order: a rounding for each, at most.
    gw_sum_off = (g_off * u.abs() + (rel + 2 * U) * terms.abs()).sum((0, 1)) + (terms.shape[0] * terms.shape[1] + 2) * U * terms.abs().sum((0, 1))
    return (gx, gx_off), (terms.sum((0, 1)), gw_sum_off)


def values(codes, scales):
    """What codes (pages, page, heads, D) and scales (pages, blocks, heads) stand for, in 64 bits."""
    per = codes.shape[1] // scales.shape[1]
    return codes.double() * scales.double().repeat_interleave(per, 1)[..., None]


def quantized(new, off, codes, scales, table, starts, lengths, block):
    """What append makes of the new tokens' values (tokens, heads, D), known to within `off`: per block and head, a list of
    (page, block of the page, first new row, rows, token of the first new row, older rows kept)."""
    P, S = codes.shape[:2]
    out = []
    for b, first, n, p0 in sequences(starts, lengths, len(new)):
        p0 = int(lengths[b]) - n
        i = 0
        while i < n:
            at = p0 + i
            rows = min(block - at % block, n - i)
            entry = at // S
            if 0 <= at and entry < table.shape[1] and 0 <= int(table[b, entry]) < P:
                out.append((int(table[b, entry]), at % S // block, at % block, rows, first + i))
            i += rows
    return out


def check_appended(got_codes, got_scales, new, off, codes, scales, table, starts, lengths, block):
    """Asserts that codes and scales are what append leaves: scales of the largest value, codes within half a scale of the values, older rows rounded
    to the new scale, all else as it was."""
    touched = torch.zeros(got_codes.shape[:3], dtype=torch.bool)
    touched_scales = torch.zeros(got_scales.shape, dtype=torch.bool)
    for page, part, row, rows, token in quantized(new, off, codes, scales, table, starts, lengths, block):
        for h in range(codes.shape[2]):
            x, o = new[token:token + rows, h], off[token:token + rows, h]
            had = float(scales[page, part, h]) if row else 0.0
            s = float(got_scales[page, part, h])
            where = f"page {page} block {part} head {h} rows {row}+{rows}"
            r0 = part * block
            touched[page, r0:r0 + row + rows, h] = True
            touched_scales[page, part, h] = True
            if not torch.isfinite(x).all() or not had < float("inf"):
                assert s != s, where
                continue
            want, slack = max(float(x.abs().max()) / 127, 1e-30, had), float(o.max()) / 127
            assert abs(s - want) <= slack + 4 * U * want, f"{where}: scale {s} for {want}"
            c = got_codes[page, r0 + row:r0 + row + rows, h].double()
            wrong = (c * s - x).abs() - (s * (0.5 + 2.0 ** -16) + o)
            assert (wrong <= 0).all() and c.abs().max() <= 127, f"{where}: a code off by {float(wrong.max() / s)} scales more than half"
            if row:
                old, now = codes[page, r0:r0 + row, h].double() * had, got_codes[page, r0:r0 + row, h].double() * s
                if s == had:
                    assert torch.equal(got_codes[page, r0:r0 + row, h], codes[page, r0:r0 + row, h]), where
                assert ((now - old).abs() <= s * (0.5 + 2.0 ** -16)).all(), f"{where}: older rows"
    assert torch.equal(got_codes[~touched], codes[~touched]) and torch.equal(got_scales[~touched_scales].nan_to_num(7.0), scales[~touched_scales].nan_to_num(7.0))


def attended_quantized(q, k, v, k_scales, v_scales, table, starts, lengths, window=0, prefix=None, **options):
    """attention over a quantized cache in 64 bits, its bound, and which rows belong to a sequence. q is fp16, or bf16 whose values fp16 holds. P is rounded to
    fp16 once, relative to the largest scale of V of the blocks that the row sees: weights below 2^-21 of that by up to 2^-32 of it for each key. The sums are
    those of attention over fp16."""
    h = q.half()
    assert torch.equal(h.float(), q.float())
    kp, vp = values(k, k_scales), values(v, v_scales)
    out, off, mine = attended(h, kp, vp, table, starts, lengths, window=window, prefix=prefix, **options)
    P, S, kv, _ = k.shape
    block = S // k_scales.shape[1]
    for b, first, new, p0 in sequences(starts, lengths, len(q)):
        keys = min(max(int(lengths[b]), 0), table.shape[1] * S)
        if not keys or not new:
            continue
        j, n = torch.arange(keys), torch.arange(p0, p0 + new)[:, None]
        page = table[b].long()[j // S]
        there = (page >= 0) & (page < P)
        see = j <= n
        if window:
            see &= n - j < window
        if prefix is not None:
            see |= j < int(prefix[b])
        see &= there
        see = torch.nn.functional.pad(see, (0, -keys % block)).view(new, -1, block).any(-1)  # (rows, blocks)
        at = torch.arange(0, keys, block)
        scale = v_scales[torch.where(there[at], page[at], 0), at % S // block].double()  # (blocks, KV heads)
        scale = torch.where(torch.isfinite(scale), scale, 0.0)
        for i in range(kv):
            most = torch.where(see, scale[:, i], 0.0).amax(1) * 127  # (rows)
            group = q.shape[1] // kv
            off[first:first + new, i * group:(i + 1) * group] += (most * 2.0 ** -32 * keys)[:, None, None]
    return out, off, mine
