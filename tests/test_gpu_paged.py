"""paged_kv.append and paged_kv.attention on the GPU against plain 64-bit forms: every type, head layouts, page sizes that end inside
a tile, sequences from nothing to thousands of keys, masks that leave rows empty, pages that hold NaN where no row may look."""
import math

import pytest
import torch

from comfyui_rdna2_attention_amd import paged_kv, rotary
from helpers import gen
from paged_reference import appended, attended, rounding, turned

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def batch_of(seqs, page, g, spare=2, width=0):
    """(table, starts, lengths, pages) of sequences (new, length): page ids in random order, unused entries far out of range."""
    need = [-(-max(length, 0) // page) for _, length in seqs]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(seqs), max([*need, 1]) + width), 1 << 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + [new for new, _ in seqs], dtype=torch.int32).cumsum(0, dtype=torch.int32)
    return table, starts, torch.tensor([length for _, length in seqs], dtype=torch.int32), pages


def hide(pages_t, table, lengths, value):
    """`value` into every row of the pages that no sequence holds."""
    P, S = pages_t.shape[:2]
    used = torch.zeros(P, S, dtype=torch.bool)
    for b in range(len(lengths)):
        for n in range(min(int(lengths[b]), table.shape[1] * S)):
            if 0 <= int(table[b, n // S]) < P:
                used[int(table[b, n // S]), n % S] = True
    pages_t[~used] = value


def check(got, ref, off, dtype, rows=None):
    got = got.cpu().double()
    if rows is not None:
        got, ref, off = got[rows], ref[rows], off[rows]
    bound = off + rounding(ref.abs() + off, dtype)
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {ref[bad][0]}, "
                           f"worst {float(((got - ref).abs() / bound)[bad].nan_to_num(9e9).max()):.2f} of the bound")


def tile_rows(T, B, heads, kv, D, type_):
    """Rows of the tiles that a call's sizes choose, by the workspace they take: 16, 32 or 128."""
    size = paged_kv.get_kernels().paged_attn_workspace(T, B, heads, kv, D, {"fp16": 0, "bf16": 1, "fp32": 2}[type_])
    return {(grid * (32 + 2 * mt * (D + 2) * 4)): mt for mt in (16, 32, 128) for grid in (512, 768)}[size]


def attend(dev, type_, D, heads, kv, page, seqs, seed, rows_behind=0, tiles=None, garbage=float("nan"), table_edit=None, view=None, **options):
    g = gen(seed)
    t = TYPES[type_]
    table, starts, lengths, pages = batch_of(seqs, page, g)
    k, v = (torch.randn(pages, page, kv, D, generator=g).to(t) for _ in range(2))
    hide(k, table, lengths, garbage)
    hide(v, table, lengths, garbage)
    if table_edit is not None:
        table_edit(table)
    T = int(starts[-1]) + rows_behind
    q = torch.randn(T, heads, D, generator=g).to(t)
    assert tiles is None or type_ == "fp32" or tile_rows(T, len(seqs), heads, kv, D, type_) == tiles
    print(f"attention {type_} D={D} heads={heads}/{kv} page={page} seqs={seqs[:6]}{'...' if len(seqs) > 6 else ''} {options}", flush=True)
    on = lambda x: x.to(dev) if isinstance(x, torch.Tensor) else x  # noqa: E731
    kd, vd = on(k), on(v)
    if view is not None:
        kd, vd = view(kd), view(vd)
    got = paged_kv.attention(paged_kv.Cache(kd, vd), paged_kv.Batch(on(table), on(starts), on(lengths)), on(q), **{n: on(x) for n, x in options.items()})
    ref, off, mine = attended(q, k, v, table, starts, lengths, **options)
    assert got.shape == q.shape and got.dtype == t
    check(got, ref, off, t)
    assert not got.cpu()[~mine].any()
    return got


# One new token of each sequence, short chunks, long ones, nothing cached, nothing new, sequences of no tokens at all.
BATCHES = {
    "one": [(1, 1)],
    "decode": [(1, 1), (1, 33), (1, 128), (1, 129), (1, 700)],
    "long": [(1, 5000)],
    "chunk": [(70, 70)],
    "short-chunks": [(3, 40), (2, 2), (5, 257)],
    "mixed": [(1, 300), (130, 391), (0, 50), (1, 2), (0, 0), (37, 37)],
    "chunk-over-cache": [(200, 1100)],
}


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("heads,kv,D,page", [(4, 1, 128, 16), (6, 2, 64, 24), (3, 3, 128, 5), (8, 1, 64, 128)])
@pytest.mark.parametrize("type_", TYPES)
def test_attention(dev, type_, heads, kv, D, page, name):
    attend(dev, type_, D, heads, kv, page, BATCHES[name], seed=len(name) + heads + page)


# Enough KV heads for tiles of 128 rows: groups of 1, 2 and 5, pages that are and are not whole runs of 8 keys.
WIDE = [(48, 24, 64, 16), (24, 24, 128, 24), (70, 14, 128, 8), (30, 30, 64, 7), (24, 24, 128, 13), (44, 22, 128, 64)]


@pytest.mark.parametrize("seqs", [[(200, 200)], [(130, 1000)], [(1, 300), (260, 391), (0, 50), (1, 2), (0, 0), (297, 297)], [(150, 151), (129, 640)]])
@pytest.mark.parametrize("heads,kv,D,page", WIDE)
@pytest.mark.parametrize("type_", ["fp16", "bf16"])
def test_wide_attention(dev, type_, heads, kv, D, page, seqs):
    attend(dev, type_, D, heads, kv, page, seqs, seed=heads + page, tiles=128)


@pytest.mark.parametrize("options", ["window1", "window7", "window100", "window150", "prefix", "prefix-window", "softcap", "slopes", "all", "scale"])
@pytest.mark.parametrize("type_,heads,kv,D,page", [("bf16", 24, 24, 128, 16), ("fp16", 48, 24, 64, 20), ("fp16", 72, 24, 128, 8), ("bf16", 26, 26, 64, 32)])
def test_wide_scores(dev, type_, heads, kv, D, page, options):
    seqs = [(130, 390), (90, 90), (3, 200), (275, 333)]
    slopes = torch.linspace(-0.01, 0.5, heads)
    prefix = torch.tensor([0, 50, 210, 300], dtype=torch.int32)
    o = {"window1": dict(window=1), "window7": dict(window=7), "window100": dict(window=100), "window150": dict(window=150), "prefix": dict(prefix=prefix),
         "prefix-window": dict(prefix=prefix, window=20), "softcap": dict(softcap=2.0), "slopes": dict(slopes=slopes),
         "all": dict(prefix=prefix, window=64, softcap=30.0, slopes=slopes), "scale": dict(scale=0.7)}[options]
    attend(dev, type_, D, heads, kv, page, seqs, seed=3, tiles=128, **o)


@pytest.mark.parametrize("softcap,scale", [(0.05, 0.3), (50.0, 0.1), (50.0, 20.0), (1400.0, 5.0), (1500.0, 5.0), (20000.0, 5.0)])
@pytest.mark.parametrize("type_,heads,kv,D,tiles", [("bf16", 24, 24, 128, 128), ("fp16", 48, 24, 64, 128), ("fp16", 2, 2, 128, 32), ("fp32", 2, 2, 64, 16)])
def test_caps_low_and_high(dev, type_, heads, kv, D, tiles, softcap, scale):
    """Caps that every score reaches, that none comes near, and past what the tiles of 128 rows add behind the softmax's own product."""
    g = gen(int(softcap) + D)
    slopes = torch.rand(heads, generator=g)
    for o in ({}, {"slopes": slopes}):
        attend(dev, type_, D, heads, kv, 16, [(130, 390)] if tiles == 128 else [(40, 390)], seed=D + heads, tiles=tiles, softcap=softcap, scale=scale, **o)


@pytest.mark.parametrize("page", [8, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_wide_rows_that_see_nothing(dev, D, page):
    """As below, in tiles of 128 rows: rows before the sequence's first position, and pages that the cache does not have, among whole ones."""
    got = attend(dev, "bf16", D, 24, 24, page, [(200, 120), (90, 0), (100, 220)], seed=4, tiles=128)
    assert not got[:80].any() and not got[200:290].any() and got[80:200].any(-1).all()

    def edit(table):
        table[0, :] = -1
        table[1, 1] = 10 ** 9
        table[2, 3:] = torch.where(torch.arange(table.shape[1] - 3) % 4 == 1, -5, table[2, 3:])
    got = attend(dev, "fp16", D, 24, 24, page, [(100, 160), (133, 133), (140, 400), (1, 170)], seed=5, table_edit=edit, tiles=128)
    assert not got[:100].any()


@pytest.mark.parametrize("seed", range(12))
def test_wide_random(dev, seed):
    """Seeded random batches in tiles of 128 rows."""
    g = gen(1900 + seed)
    pick = lambda *a: a[int(torch.randint(0, len(a), (1,), generator=g))]  # noqa: E731
    upto = lambda n: int(torch.randint(0, n + 1, (1,), generator=g))  # noqa: E731
    kv = pick(21, 24, 42)
    heads = kv * pick(1, 2, 3)
    seqs = [(new, new + upto(pick(10, 200, 700))) for new in [130 + upto(200)] + [pick(1, 100 + upto(150), upto(90) + 60) for _ in range(1 + upto(2))]]
    o = {}
    if upto(2) == 0:
        o["window"] = 1 + upto(250)
    if upto(3) == 0:
        o["softcap"] = 5.0
    if upto(3) == 0:
        o["slopes"] = torch.rand(heads, generator=g)
    if upto(3) == 0:
        o["prefix"] = torch.randint(0, 250, (len(seqs),), generator=g, dtype=torch.int32)
    rows = sum(n for n, _ in seqs) * (heads // kv) // len(seqs)
    D = pick(64, 128)
    attend(dev, pick("fp16", "bf16"), D, heads, kv, pick(1, 7, 8, 12, 16, 48, 256), seqs, seed=seed, rows_behind=upto(2), tiles=128 if rows > 64 else None, **o)


@pytest.mark.parametrize("options", ["window1", "window7", "window100", "prefix", "prefix-window", "softcap", "slopes", "all", "scale"])
@pytest.mark.parametrize("type_,D,page", [("bf16", 128, 16), ("fp16", 64, 20), ("fp32", 128, 16), ("fp32", 64, 3)])
def test_scores(dev, type_, D, page, options):
    heads, seqs = 4, [(1, 290), (90, 90), (3, 200), (75, 333)]
    slopes = torch.tensor([0.5, 0.11, 0.02, 0.0])
    prefix = torch.tensor([0, 50, 210, 300], dtype=torch.int32)
    o = {"window1": dict(window=1), "window7": dict(window=7), "window100": dict(window=100), "prefix": dict(prefix=prefix),
         "prefix-window": dict(prefix=prefix, window=20), "softcap": dict(softcap=2.0), "slopes": dict(slopes=slopes),
         "all": dict(prefix=prefix, window=64, softcap=30.0, slopes=slopes), "scale": dict(scale=0.7)}[options]
    attend(dev, type_, D, heads, 2, page, seqs, seed=3, **o)


@pytest.mark.parametrize("type_", TYPES)
def test_rows_that_see_nothing(dev, type_):
    """Lengths below the new tokens (their first rows come before the sequence), lengths of zero with new tokens, and a table whose
    pages do not exist: rows of zeros, and the others as if the missing keys were not there."""
    got = attend(dev, type_, 128, 4, 2, 8, [(5, 3), (4, 0), (1, 20), (40, 20)], seed=4)
    assert not got[:2].any() and not got[5:9].any() and got[2:5].any(-1).all()

    def edit(table):
        table[0, :] = torch.tensor([-1, 1 << 29] + [-7] * (table.shape[1] - 2), dtype=torch.int32)
        table[2, 1] = -1
        table[3, 2] = 10 ** 9
    got = attend(dev, type_, 128, 4, 2, 8, [(5, 16), (3, 30), (2, 40), (33, 33), (1, 17)], seed=5, table_edit=edit)
    assert not got[:5].any()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("new,length,copies", [(40, 40, 1), (9, 300, 1), (150, 150, 1), (150, 150, 12), (200, 330, 12)])
def test_values_that_are_not_finite(dev, type_, new, length, copies):
    """inf and NaN in the keys and values of later tokens do not reach the rows that do not see them; rows that do see them get them."""
    g = gen(new)
    t = TYPES[type_]
    table, starts, lengths, pages = batch_of([(new, length)], 16, g)
    k, v = (torch.randn(pages, 16, 2, 128, generator=g).to(t) for _ in range(2))
    q = torch.randn(new, 4, 128, generator=g).to(t)
    bad = length - new // 2  # this token's value is NaN in one head, the next one's key is inf
    v[int(table[0, bad // 16]), bad % 16, 0, 5] = float("nan")
    v[int(table[0, bad // 16]), bad % 16, 1, 70] = float("inf")
    k[int(table[0, (bad + 1) // 16]), (bad + 1) % 16, 1] = float("nan")
    k, v, q = k.repeat(1, 1, copies, 1), v.repeat(1, 1, copies, 1), q.repeat(1, copies, 1)  # 12: tiles of 128 rows
    print(f"not finite {type_} {new} of {length} x {copies}", flush=True)
    assert type_ == "fp32" or tile_rows(new, 1, 4 * copies, 2 * copies, 128, type_) == (128 if copies > 1 else 32)
    got = paged_kv.attention(paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), q.to(dev)).cpu()
    ref, off, _ = attended(q, k, v, table, starts, lengths)
    at = bad - (length - new)
    check(got, ref, off, t, rows=slice(0, at))
    assert torch.isfinite(got[:at]).all()
    nan, inf = [h for h in range(4 * copies) if h % 4 < 2], [h for h in range(4 * copies) if h % 4 >= 2]
    assert got[at:, nan, 5].isnan().all() and (got[at, inf, 70] == float("inf")).all() and got[at + 1:, inf].isnan().all()
    keep = [d for d in range(128) if d != 5]
    check(got[at:, nan][..., keep], ref[at:, nan][..., keep], off[at:, nan][..., keep], t)


@pytest.mark.parametrize("new,length,kv", [(1, 300, 1), (40, 40, 1), (100, 400, 1), (130, 400, 24)])
@pytest.mark.parametrize("type_", ["bf16", "fp32"])
def test_scores_far_from_zero(dev, type_, new, length, kv):
    """Scores near -10^35 and 10^35: the softmax is of their differences, wherever they lie. q sees keys as +-10^17 (1 + steps of 1/8): products
    exact in both types, and one key's score above all others by more than 2^100."""
    t = TYPES[type_]
    g = gen(new)
    table, starts, lengths, pages = batch_of([(new, length)], 16, g)
    step = torch.randint(0, 4, (pages, 16, kv, 1), generator=g)
    k = (2.0 ** 57 * (1 + step / 8)).expand(pages, 16, kv, 64).to(t).contiguous()
    v = torch.randn(pages, 16, kv, 64, generator=g).to(t)
    q = torch.full((new, 2 * kv, 64), 2.0 ** 57).to(t)
    q[:, 1::2] = -q[:, 1::2]
    got = paged_kv.attention(paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), q.to(dev)).cpu()
    ref, off, _ = attended(q, k, v, table, starts, lengths)
    # Equal scores stay equal (the same operations on the same values) and all others' weights are 0: a mean of values, in 32 bits and P = 1.
    bound = length * 2.0 ** -23 * v.double().abs().max() + rounding(ref, t)
    assert ((got.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("kv", [2, 24])
@pytest.mark.parametrize("type_", ["bf16", "fp16"])
def test_maximum_that_rises_slowly(dev, type_, kv):
    """Scores that grow with the key's position, by any amount a tile: rows whose maximum keeps moving, or stays just below what moves it."""
    g = gen(77)
    t = TYPES[type_]
    for slope in (0.02, 0.05, 0.11, 0.3, 1.0):
        table, starts, lengths, pages = batch_of([(140, 900)], 16, g)
        k = torch.randn(pages, 16, kv, 64, generator=g) * 0.1
        for n in range(900):
            k[int(table[0, n // 16]), n % 16, :, 0] = slope * n
        v = torch.randn(pages, 16, kv, 64, generator=g)
        q = torch.randn(140, 2 * kv, 64, generator=g) * 0.1
        q[..., 0] = 1.0
        k, v, q = k.to(t), v.to(t), q.to(t)
        got = paged_kv.attention(paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), q.to(dev))
        ref, off, _ = attended(q, k, v, table, starts, lengths)
        check(got, ref, off, t)


@pytest.mark.parametrize("gap", [6.3, 13.7, 18.3, 25.1])
@pytest.mark.parametrize("type_,new,kv,tiles", [("fp16", 1, 2, 16), ("fp16", 40, 1, 32), ("fp16", 140, 24, 128), ("bf16", 140, 24, 128), ("bf16", 1, 2, 16), ("fp32", 1, 2, 16)])
def test_light_keys_beside_heavy_ones(dev, type_, new, kv, tiles, gap):
    """Every 32nd key weighs 2^gap times the others and has value 0, the others 1: a row that sees a heavy and b light keys gives
    b 2^-gap / (a + b 2^-gap), nothing but the light keys' weights. Each of those is rounded to the type, as is the heavy ones' (2 u), its
    score has an error of 2^-23 of gap in the log2 domain and 2^x one of 2^-22, sums of n keys n 2^-23; in fp16 a weight that falls below
    the normal range is off by half of 2^-24, with m lifted 2^7 (2^9) below the maximum at least."""
    length, t = 2000, TYPES[type_]
    assert tile_rows(new, 1, kv, kv, 64, type_) == tiles
    pages = torch.zeros(125, 16, kv, 64)
    k, v, q = pages.clone(), pages.clone() + 1.0, torch.zeros(new, kv, 64)
    k[..., 0] = -1.0
    k[::2, 0] = 0.0
    v[::2, 0] = 0.0
    q[..., 0] = 1.0
    cache = paged_kv.Cache(k.to(t).to(dev), v.to(t).to(dev))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    batch = paged_kv.Batch(torch.arange(125, dtype=torch.int32, device=dev)[None], i32([0, new]), i32([length]))
    got = paged_kv.attention(cache, batch, q.to(t).to(dev), scale=gap * math.log(2.0)).cpu().double()
    n = torch.arange(length - new + 1, length + 1, dtype=torch.float64)
    heavy = (n / 32).ceil()
    light = (n - heavy) * 2.0 ** -gap
    ref = (light / (heavy + light))[:, None, None].expand_as(got)
    u = 0.0 if type_ == "fp32" else torch.finfo(t).eps / 2
    off = ref * (2 * u + (gap * 2 ** -23 + 2.0 ** -22) * 1.4 + length * 2.0 ** -23) + (31 * 2.0 ** -32 if type_ == "fp16" else 0.0)
    check(got, ref, off, t)


def test_many_sequences(dev):
    """More sequences than a workgroup has threads, most of them short, some empty."""
    g = gen(11)
    seqs = [(int(n), int(n) + int(c)) for n, c in zip(torch.randint(0, 3, (700,), generator=g), torch.randint(0, 40, (700,), generator=g))]
    attend(dev, "fp16", 64, 2, 1, 8, seqs, seed=12, rows_behind=3)
    attend(dev, "bf16", 64, 4, 1, 8, [(0, 5)] * 300 + [(17, 40)], seed=13)


def test_rows_of_no_sequence(dev):
    """A padded batch: with out given, rows behind the last sequence (and before the first) stay as they were; made by the call, they are 0."""
    attend(dev, "bf16", 128, 8, 2, 16, [(1, 50), (1, 9)], seed=14, rows_behind=6)
    g = gen(15)
    table, starts, lengths, pages = batch_of([(2, 50), (1, 9)], 16, g)
    k, v = (torch.randn(pages, 16, 2, 64, generator=g).half() for _ in range(2))
    q = torch.randn(9, 4, 64, generator=g).half()
    starts = starts + 2
    out = torch.full((9, 6, 64), 7.0, dtype=torch.float16, device=dev)
    cache, batch = paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev))
    got = paged_kv.attention(cache, batch, q.to(dev), out=out[:, 1:5])
    assert got.data_ptr() == out[:, 1:5].data_ptr()
    ref, off, mine = attended(q, k, v, table, starts, lengths)
    assert mine.tolist() == [False] * 2 + [True] * 3 + [False] * 4
    check(got, ref, off, torch.float16, rows=mine)
    assert paged_kv.attention(cache, batch, q.to(dev)[:0]).shape == (0, 4, 64)
    left = out.cpu()
    assert (left[~mine] == 7).all() and (left[:, 0] == 7).all() and (left[:, 5] == 7).all()


def test_malformed_starts_stay_inside(dev):
    """starts that fall or leave the rows: nothing outside q and out is touched, and the well-formed sequences are right."""
    g = gen(16)
    table, _, _, pages = batch_of([(2, 50), (1, 9), (3, 30)], 16, g)
    k, v = (torch.randn(pages, 16, 2, 64, generator=g).half() for _ in range(2))
    guard = torch.zeros(26, 4, 64, dtype=torch.float16, device=dev)
    q = torch.randn(6, 4, 64, generator=g).half()
    starts, lengths = torch.tensor([0, 2, 1 << 30, 5], dtype=torch.int32), torch.tensor([50, 9, 30], dtype=torch.int32)
    cache, batch = paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev))
    out = paged_kv.attention(cache, batch, q.to(dev), out=guard[10:16]).cpu()
    ref, off, _ = attended(q, k, v, table, starts, lengths)
    check(out[:2], ref[:2], off[:2], torch.float16)
    assert not guard[:10].any() and not guard[16:].any()


def test_length_past_capacity(dev):
    """A length past the table counts as the table's capacity, in the keys that are read; the positions are the length's."""
    g = gen(17)
    table = torch.randperm(8, generator=g)[:6].to(torch.int32).view(2, 3)
    starts, lengths = torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([60, 2 ** 31 - 1], dtype=torch.int32)
    k, v = (torch.randn(8, 16, 1, 64, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(3, 2, 64, generator=g).bfloat16()
    got = paged_kv.attention(paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), q.to(dev))
    ref, off, _ = attended(q, k, v, table, starts, lengths)
    check(got, ref, off, torch.bfloat16)


def test_orders_of_memory(dev):
    """Pools with heads before tokens, with K and V in one tensor, with gaps between rows; q as a part of a projection, and unaligned."""
    seqs = [(1, 100), (20, 45)]
    attend(dev, "fp16", 64, 4, 2, 16, seqs, seed=18, view=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    attend(dev, "bf16", 128, 4, 2, 16, seqs, seed=19, view=lambda t: torch.stack((t, t * 0), 1)[:, 0])
    attend(dev, "fp32", 64, 4, 2, 16, seqs, seed=20, view=lambda t: torch.cat((t, t * 0), 3)[..., :64])
    attend(dev, "fp16", 128, 4, 2, 16, seqs, seed=21, view=lambda t: t.permute(2, 1, 3, 0).contiguous().permute(3, 1, 0, 2).contiguous())
    g = gen(22)
    table, starts, lengths, pages = batch_of(seqs, 16, g)
    k, v = (torch.randn(pages, 16, 2, 64, generator=g).half() for _ in range(2))
    cache, batch = paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev))
    fused = torch.randn(21, 8 * 64, generator=g).half()
    ref, off, _ = attended(fused.view(21, 8, 64)[:, :4], k, v, table, starts, lengths)
    check(paged_kv.attention(cache, batch, fused.to(dev).view(21, 8, 64)[:, :4]), ref, off, torch.float16)
    odd = torch.randn(21 * 256 + 1, generator=g).half()
    ref, off, _ = attended(odd[1:].view(21, 4, 64), k, v, table, starts, lengths)
    check(paged_kv.attention(cache, batch, odd.to(dev)[1:].view(21, 4, 64)), ref, off, torch.float16)


def test_offsets_past_32_bits(dev):
    """Pages of more than 2^31 values (2^32 bytes): the last ones are written and read."""
    g = gen(23)
    P, S, kv, D = 132000, 16, 8, 128
    k, v = (torch.empty(P, S, kv, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    assert k.numel() > 2 ** 31
    table = torch.tensor([[P - 1, 3, P - 2]], dtype=torch.int32)
    starts, lengths = torch.tensor([0, 40], dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    kn, vn = (torch.randn(40, kv, D, generator=g).bfloat16() for _ in range(2))
    cache, batch = paged_kv.Cache(k, v), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev))
    paged_kv.append(cache, batch, kn.to(dev), vn.to(dev))
    assert torch.equal(k[P - 1].cpu(), kn[:16]) and torch.equal(v[P - 2, :8].cpu(), vn[32:])
    q = torch.randn(40, 8, D, generator=g).bfloat16()
    small = torch.zeros(3, S, kv, D, dtype=torch.bfloat16)
    ks, vs = small.clone(), small.clone()
    ks.view(-1, kv, D)[:40], vs.view(-1, kv, D)[:40] = kn, vn
    ref, off, _ = attended(q, ks, vs, torch.tensor([[0, 1, 2]], dtype=torch.int32), starts, lengths)
    check(paged_kv.attention(cache, batch, q.to(dev)), ref, off, torch.bfloat16)


@pytest.mark.parametrize("seed", range(16))
def test_random(dev, seed):
    """Seeded random batches, heads, pages and scores."""
    g = gen(900 + seed)
    pick = lambda *a: a[int(torch.randint(0, len(a), (1,), generator=g))]  # noqa: E731
    upto = lambda n: int(torch.randint(0, n + 1, (1,), generator=g))  # noqa: E731
    kv = pick(1, 2, 3)
    heads = kv * pick(1, 2, 5, 8, 16)
    seqs = []
    for _ in range(1 + upto(6)):
        new = pick(1, 1, upto(4), upto(90))
        seqs.append((new, new + upto(pick(10, 200, 900))))
    o = {}
    if upto(2) == 0:
        o["window"] = 1 + upto(150)
    if upto(3) == 0:
        o["softcap"] = 5.0
    if upto(3) == 0:
        o["slopes"] = torch.rand(heads, generator=g)
    if upto(3) == 0:
        o["prefix"] = torch.randint(0, 150, (len(seqs),), generator=g, dtype=torch.int32)
    attend(dev, pick("fp16", "bf16", "fp32"), pick(64, 128), heads, kv, pick(1, 7, 8, 12, 16, 48, 256), seqs, seed=seed, rows_behind=upto(2), **o)


# ---------------------------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("page,D,heads,kv", [(16, 128, 8, 2), (5, 64, 3, 3), (1, 96, 2, 1), (24, 256, 1, 1), (128, 128, 40, 8)])
@pytest.mark.parametrize("type_,cache_type", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "fp32")])
def test_append(dev, type_, cache_type, page, D, heads, kv):
    g = gen(page + D)
    t, ct = TYPES[type_], TYPES[cache_type]
    table, starts, lengths, pages = batch_of([(1, 1), (0, 7), (9, 30), (4, 4), (1, 77)], page, g, width=1)
    k0, v0 = (torch.randn(pages, page, kv, D, generator=g).to(ct) for _ in range(2))
    T = int(starts[-1])
    qkv = torch.randn(T + 2, heads + 2 * kv, D, generator=g).to(t)  # two rows behind the last sequence
    q, k, v = qkv.split((heads, kv, kv), 1)
    rot = rotary.Rotary(D // 2 // 16 * 16 if page == 16 else D, layout="interleaved" if page == 24 else "half", device=dev)
    kd, vd, fused = k0.to(dev), v0.to(dev), qkv.to(dev)
    qd = fused.split((heads, kv, kv), 1)
    q_out = torch.full((T + 2, heads, D), 3.0, dtype=ct, device=dev)
    print(f"append {type_} -> {cache_type} page={page} D={D} heads={heads}/{kv}", flush=True)
    got = paged_kv.append(paged_kv.Cache(kd, vd), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), qd[1], qd[2], rotary=rot, q=qd[0], q_out=q_out)
    assert got is q_out and torch.equal(fused.cpu(), qkv)
    rk, rv, off = appended(k[:T], v[:T], k0, v0, table, starts, lengths, rot)
    check(kd, rk, off, ct)
    check(vd, rv, torch.zeros_like(off), ct)
    untouched = off == 0
    assert torch.equal(kd.cpu()[(rk == k0.double()) & untouched], k0[(rk == k0.double()) & untouched])
    n = torch.cat([torch.arange(int(lengths[b]) - int(starts[b + 1] - starts[b]), int(lengths[b])) for b in range(len(lengths))])
    rq, off = turned(q[:T], n, rot)
    check(q_out[:T], rq, off, ct)
    assert (q_out[T:] == 3).all()


def test_append_same_turn_as_rotate(dev):
    """append turns keys and queries with rotate's bits, and without a rotary copies; q in place; more sequences than a wave has lanes."""
    g = gen(31)
    B, page, kv, D = 5000, 8, 2, 64
    new = torch.randint(0, 3, (B,), generator=g)
    seqs = [(int(n), int(n) + int(c)) for n, c in zip(new, torch.randint(0, 20, (B,), generator=g))]
    table, starts, lengths, pages = batch_of(seqs, page, g)
    T = int(starts[-1])
    q, k, v = (torch.randn(T, h, D, generator=g).half().to(dev) for h in (4, kv, kv))
    n = torch.cat([torch.arange(length - m, length) for m, length in seqs])
    rot = rotary.Rotary(64, device=dev)
    for r in (rot, None):
        cache = paged_kv.Cache(*(torch.zeros(pages, page, kv, D, dtype=torch.float16, device=dev) for _ in range(2)))
        batch = paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev))
        mine = q.clone()
        assert paged_kv.append(cache, batch, k, v, rotary=r, q=mine) is mine
        want_q, want_k = (q, k) if r is None else (rotary.rotate(q, n.to(dev), r), rotary.rotate(k, n.to(dev), r))
        b = torch.repeat_interleave(torch.arange(B), new)
        page_of, row = table[b, n // page].long().to(dev), (n % page).to(dev)
        assert torch.equal(mine, want_q) and torch.equal(cache.k[page_of, row], want_k) and torch.equal(cache.v[page_of, row], v)
    assert paged_kv.append(cache, batch, k[:0], v[:0]) is None


def test_append_drops_what_has_no_place(dev):
    """Negative positions, positions past the table, pages that the cache does not have, starts outside the rows: nothing is written,
    the rest is."""
    g = gen(32)
    table = torch.tensor([[0, 1], [2, -1], [1 << 30, 3], [4, 5]], dtype=torch.int32)
    starts, lengths = torch.tensor([1, 6, 11, 20, 24], dtype=torch.int32), torch.tensor([3, 10, 12, 18], dtype=torch.int32)
    k0, v0 = (torch.randn(7, 8, 1, 64, generator=g) for _ in range(2))
    k, v, q = torch.randn(26, 1, 64, generator=g), torch.randn(26, 1, 64, generator=g), torch.randn(26, 2, 64, generator=g)
    rot = rotary.Rotary(64, device=dev)
    kd, vd, qd = k0.to(dev), v0.to(dev), q.to(dev)
    paged_kv.append(paged_kv.Cache(kd, vd), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), k.to(dev), v.to(dev), rotary=rot, q=qd)
    rk, rv, off = appended(k, v, k0, v0, table, starts, lengths, rot)
    check(kd, rk, off, torch.float32)
    assert torch.equal(vd.cpu(), rv.float())
    assert torch.equal(qd.cpu()[:1], q[:1]) and torch.equal(qd.cpu()[24:], q[24:]) and not torch.equal(qd.cpu()[1:24], q[1:24])
    starts = torch.tensor([0, 5, 3, 1 << 30, -5], dtype=torch.int32)  # falls, and leaves the rows: no fault
    paged_kv.append(paged_kv.Cache(kd, vd), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), k.to(dev), v.to(dev), rotary=rot, q=qd)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------- a run of them together

@pytest.mark.parametrize("type_", TYPES)
def test_serving_steps(dev, type_):
    """Prompts in chunks, then single tokens, of sequences that come, grow and take new pages: each step appends (turning q and k) and
    attends; every output is that of dense causal attention over the sequence's whole history, in 64 bits on the rounded keys."""
    g = gen(41)
    t = TYPES[type_]
    kv, heads, D, page, pages = 2, 8, 64, 8, 40
    rot = rotary.Rotary(D, base=1e6, device=dev)
    cache = paged_kv.Cache(*(torch.full((pages, page, kv, D), float("nan"), dtype=t, device=dev) for _ in range(2)))
    free = torch.randperm(pages, generator=g).tolist()
    held, done = [[] for _ in range(3)], [0, 0, 0]
    history = [[torch.zeros(0, kv, D, dtype=torch.float64), torch.zeros(0, kv, D, dtype=torch.float64)] for _ in range(3)]
    for step, new in enumerate([(40, 0, 0), (30, 17, 0), (1, 1, 0), (1, 1, 9), (1, 1, 1), (1, 0, 1), (1, 1, 1)]):
        for b in range(3):
            done[b] += new[b]
            while len(held[b]) * page < done[b]:
                held[b].append(free.pop())
        table = torch.zeros(3, 12, dtype=torch.int32)
        for b in range(3):
            table[b, :len(held[b])] = torch.tensor(held[b], dtype=torch.int32)
        starts = torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        batch = paged_kv.Batch(table.to(dev), starts.to(dev), torch.tensor(done, dtype=torch.int32, device=dev))
        T = sum(new)
        q, k, v = (torch.randn(T, h, D, generator=g).to(t) for h in (heads, kv, kv))
        print(f"step {step} {type_} new={new}", flush=True)
        qr = paged_kv.append(cache, batch, k.to(dev), v.to(dev), rotary=rot, q=q.to(dev))
        out = paged_kv.attention(cache, batch, qr)
        kr = torch.cat([rotary.rotate(k[starts[b]:starts[b + 1]].to(dev), torch.arange(done[b] - new[b], done[b], device=dev), rot) for b in range(3)]).cpu()
        for b in range(3):
            rows = slice(int(starts[b]), int(starts[b + 1]))
            history[b][0] = torch.cat((history[b][0], kr[rows].double()))
            history[b][1] = torch.cat((history[b][1], v[rows].double()))
            if new[b]:
                ref, off, _ = attended(qr[rows].cpu(), history[b][0][None], history[b][1][None], torch.tensor([[0]], dtype=torch.int32),
                                       torch.tensor([0, new[b]]), torch.tensor([done[b]]))
                check(out[rows], ref, off, t)


def test_captured_steps(dev):
    """Two captured graphs of append and attention, their batches' contents changed between replays, with eager calls between and beside:
    each replay equals the eager call on the same contents, bit for bit."""
    g = gen(42)
    kv, heads, D, page, B = 2, 8, 128, 16, 4
    rot = rotary.Rotary(D, device=dev)

    def world(seed):
        h = gen(seed)
        cache = paged_kv.Cache(*(torch.randn(64, page, kv, D, generator=h).bfloat16().to(dev) for _ in range(2)))
        batch = paged_kv.Batch(torch.randperm(64, generator=h)[:B * 12].view(B, 12).to(torch.int32).to(dev), torch.arange(B + 1, dtype=torch.int32, device=dev),
                               torch.tensor([3, 60, 150, 1], dtype=torch.int32, device=dev))
        return cache, batch, *(torch.randn(B, n, D, generator=h).bfloat16().to(dev) for n in (heads, kv, kv))

    def step(w, out=None):
        cache, batch, q, k, v = w
        qr = paged_kv.append(cache, batch, k, v, rotary=rot, q=q, q_out=torch.empty_like(q))
        return paged_kv.attention(cache, batch, qr, out=out)

    worlds, graphs, outs = [world(50), world(51)], [], []
    for w in worlds:
        step(w)
        torch.cuda.synchronize()
        graph, out = torch.cuda.CUDAGraph(), torch.zeros(B, heads, D, dtype=torch.bfloat16, device=dev)
        with torch.cuda.graph(graph):
            step(w, out)
        graphs.append(graph)
        outs.append(out)
    side = torch.cuda.Stream()
    for i in range(5):
        for w in worlds:
            w[1].lengths += 1 + 3 * i
            for t in w[2:]:
                t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for w, out in zip(worlds, outs):
            assert torch.equal(out, step(w)), i


def test_calls_at_once(dev):
    """Calls on two streams at a time, each on its own cache, give the bits of calls one by one."""
    jobs = []
    for s in range(4):
        g = gen(60 + s)
        kv, seqs = (2, [(1, 900 + 100 * s), (60, 300), (1, 5)]) if s % 2 else (24, [(1, 900), (160, 300 + 50 * s), (140, 140)])
        table, starts, lengths, pages = batch_of(seqs, 16, g)
        cache = paged_kv.Cache(*(torch.randn(pages, 16, kv, 128, generator=g).half().to(dev) for _ in range(2)))
        jobs.append((cache, paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), torch.randn(int(starts[-1]), 2 * kv, 128, generator=g).half().to(dev)))
    want = [paged_kv.attention(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for r in range(3):
        for i, j in enumerate(jobs):
            with torch.cuda.stream(streams[(i + r) % 2]):
                got.append(paged_kv.attention(*j))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 4]), i
