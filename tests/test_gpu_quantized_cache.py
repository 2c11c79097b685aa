"""The quantized cache on the GPU against plain 64-bit forms: appends into blocks new, half filled and of changing scales, reading back, attention over every
mask and type, blocks of NaN and of anything where no row may look, and steps of them together."""
import pytest
import torch

from comfyui_rdna2_attention_amd import paged_kv, rotary
from helpers import gen
from paged_reference import rounding, sequences, turned
from quantized_reference import attended_quantized, check_appended, norm_turned, normed, values
from test_gpu_paged import BATCHES, batch_of, check

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def codes_of(pages, page, kv, D, block, g, spread=0.3):
    """Codes and scales as quantized normal values leave them."""
    c = lambda: (torch.randn(pages, page, kv, D, generator=g) * 36).round().clamp(-127, 127).to(torch.int8)  # noqa: E731
    s = lambda: 0.03 * torch.exp(spread * torch.randn(pages, page // block, kv, generator=g))  # noqa: E731
    return c(), c(), s(), s()


def on(dev, *ts):
    return [t.to(dev) if isinstance(t, torch.Tensor) else t for t in ts]


# ---------------------------------------------------------------------------------------------------------------- append

SEQS = [(1, 1), (0, 7), (9, 30), (4, 4), (1, 77), (100, 131), (16, 48), (1, 65), (33, 33)]


def new_values(k, v, q, starts, lengths, rot, norm):
    """The 64-bit values that k, v and q become, with bounds."""
    T = int(starts[-1])
    n = torch.cat([torch.arange(int(lengths[b]) - new, int(lengths[b])) for b, _, new, _ in sequences(starts, lengths, T)])
    out = []
    for x, w in ((k[:T], None if norm is None else norm.k.cpu()), (q[:T], None if norm is None else norm.q.cpu())):
        if w is not None:
            y, off = norm_turned(x, w, n, rot, norm.eps)
        elif rot is not None:
            y, off = turned(x, n, rot)
        else:
            y, off = x.double(), torch.zeros_like(x, dtype=torch.float64)
        out.append((y, off))
    return out[0], (v[:T].double(), torch.zeros_like(v[:T], dtype=torch.float64)), out[1]


@pytest.mark.parametrize("page,block,D,heads,kv", [(16, 16, 128, 8, 2), (48, 16, 64, 3, 3), (32, 32, 96, 2, 1), (64, 32, 80, 5, 5), (64, 64, 256, 1, 1), (128, 64, 128, 40, 8),
                                                   (96, 32, 16, 7, 1), (64, 64, 64, 6, 2)])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("type_,out", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16"), ("fp32", "bf16"), ("fp16", "bf16")])
def test_append(dev, type_, out, normed, page, block, D, heads, kv):
    g = gen(page + D + block)
    t, ot = TYPES[type_], TYPES[out]
    table, starts, lengths, pages = batch_of(SEQS, page, g, width=1)
    k0, v0, ks0, vs0 = codes_of(pages, page, kv, D, block, g, spread=1.0)
    T = int(starts[-1])
    qkv = (torch.randn(T + 2, heads + 2 * kv, D, generator=g) * torch.exp(0.7 * torch.randn(T + 2, 1, 1, generator=g))).to(t)  # two rows behind the last sequence
    q, k, v = qkv.split((heads, kv, kv), 1)
    rot = rotary.Rotary(max(D // 2 // 16 * 16, 16) if page == 16 else D, layout="interleaved" if page in (48, 128) else "half", device=dev)
    norm = rotary.HeadNorm(*((1 + 0.3 * torch.randn(D, generator=g)).to(t if page > 32 else torch.float32).to(dev) for _ in range(2)), eps=1e-5) if normed else None
    kd, vd, ksd, vsd, fused = on(dev, k0, v0, ks0, vs0, qkv)
    qd = fused.split((heads, kv, kv), 1)
    q_out = torch.full((T + 2, heads, D), 3.0, dtype=ot, device=dev)
    print(f"append {type_} -> {out} page={page} block={block} D={D} heads={heads}/{kv} normed={normed}", flush=True)
    got = paged_kv.append(paged_kv.QuantizedCache(kd, vd, ksd, vsd), paged_kv.Batch(*on(dev, table, starts, lengths)), qd[1], qd[2], rotary=rot, q=qd[0], q_out=q_out, norm=norm)
    assert got is q_out and torch.equal(fused.cpu(), qkv) and (q_out[T:] == 3).all()
    (rk, koff), (rv, voff), (rq, qoff) = new_values(k, v, q, starts, lengths, rot, norm)
    check(q_out[:T], rq, qoff, ot)
    check_appended(kd.cpu(), ksd.cpu(), rk, koff, k0, ks0, table, starts, lengths, block)
    check_appended(vd.cpu(), vsd.cpu(), rv, voff, v0, vs0, table, starts, lengths, block)


def test_append_many_sequences_of_chunks(dev):
    """More sequences than a wave has lanes, each of several tokens; norms without a turn; then the same tokens again, which changes nothing."""
    g = gen(51)
    B, page, kv, D = 300, 32, 1, 64
    new = torch.randint(0, 24, (B,), generator=g)
    seqs = [(int(n), int(n) + int(c)) for n, c in zip(new, torch.randint(0, 70, (B,), generator=g))]
    table, starts, lengths, pages = batch_of(seqs, page, g)
    T = int(starts[-1])
    assert T >= 4 * B
    q, k, v = (torch.randn(T, h, D, generator=g).bfloat16() for h in (2, kv, kv))
    norm = rotary.HeadNorm(*((1 + 0.3 * torch.randn(D, generator=g)).to(dev) for _ in range(2)), eps=1e-5)
    k0, v0, ks0, vs0 = codes_of(pages, page, kv, D, 16, g)
    kd, vd, ksd, vsd = on(dev, k0, v0, ks0, vs0)
    cache, batch = paged_kv.QuantizedCache(kd, vd, ksd, vsd), paged_kv.Batch(*on(dev, table, starts, lengths))
    out = paged_kv.append(cache, batch, k.to(dev), v.to(dev), q=q.to(dev), q_out=torch.empty(T, 2, D, dtype=torch.float16, device=dev), norm=norm)
    (rk, krel), (rq, qrel) = normed(k, norm.k.cpu(), 1e-5), normed(q, norm.q.cpu(), 1e-5)
    check(out, rq, rq.abs() * qrel, torch.float16)
    check_appended(kd.cpu(), ksd.cpu(), rk, rk.abs() * krel, k0, ks0, table, starts, lengths, 16)
    check_appended(vd.cpu(), vsd.cpu(), v.double(), v.double() * 0, v0, vs0, table, starts, lengths, 16)
    before = [t.clone() for t in (kd, vd, ksd, vsd)]
    paged_kv.append(cache, batch, k.to(dev), v.to(dev), norm=norm)
    assert all(torch.equal(a, b) for a, b in zip(before, (kd, vd, ksd, vsd)))


@pytest.mark.parametrize("type_", ["fp16", "fp32"])
def test_appends_by_tokens_and_by_blocks_agree(dev, type_):
    """Steps of few tokens a sequence and of many take different launches: the same codes, scales and queries, bit for bit."""
    g = gen(52)
    t, kv, D, page = TYPES[type_], 3, 128, 32
    rot, norm = rotary.Rotary(64, device=dev), rotary.HeadNorm(*((1 + 0.3 * torch.randn(D, generator=g)).to(dev) for _ in range(2)))
    seqs = [(3, 40), (1, 1), (3, 33), (2, 64), (3, 90)]
    table, starts, lengths, pages = batch_of(seqs, page, g)
    T = int(starts[-1])
    q, k, v = (torch.randn(T, h, D, generator=g).to(t).to(dev) for h in (6, kv, kv))
    first = on(dev, *codes_of(pages, page, kv, D, 16, g, spread=1.0))
    results = []
    for spare in (0, 40):  # tokens of no sequence behind: the mean decides
        c = [x.clone() for x in first]
        pad = lambda x: torch.cat((x, x[:1].expand(spare, *x.shape[1:]))) if spare else x  # noqa: E731
        out = torch.zeros(T + spare, 6, D, dtype=torch.float16, device=dev)
        paged_kv.append(paged_kv.QuantizedCache(*c), paged_kv.Batch(*on(dev, table, starts, lengths)), pad(k), pad(v), rotary=rot, q=pad(q), q_out=out, norm=norm)
        results.append((*c, out[:T]))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("block", [16, 32, 64])
def test_append_token_by_token(dev, block):
    """Single tokens one after the other: each block's scale is that of its largest value so far, what was written is off by half a scale for each time
    that it was rounded, and a block that begins anew forgets its old scale. In place queries; no rotation."""
    g = gen(block)
    kv, D, page, B = 2, 64, 64, 3
    cache = paged_kv.QuantizedCache.empty(9, page, kv, D, block=block, device=dev)
    cache.k_scales.fill_(float("nan"))  # of an earlier owner
    cache.v_scales.fill_(1e9)
    table = torch.randperm(9, generator=g)[:9].view(3, 3).to(torch.int32).to(dev)
    starts = torch.arange(B + 1, dtype=torch.int32, device=dev)
    sizes = torch.exp(torch.randn(150, B, 1, 1, generator=g)).half()
    k, v = (torch.randn(150, B, kv, D, generator=g).half() * sizes for _ in range(2))
    batch = paged_kv.Batch(table, starts, torch.zeros(B, dtype=torch.int32, device=dev))
    for i in range(150):
        batch.lengths += 1
        q = k[i].to(dev).repeat(1, 2, 1)
        same = q.clone()
        assert paged_kv.append(cache, batch, k[i].to(dev), v[i].to(dev), q=q) is q and torch.equal(q, same)
    got = paged_kv.read(cache, paged_kv.Batch(table, starts * 150, batch.lengths), B * 150, torch.float32)
    for x, y, scales in ((k, got[0], cache.k_scales), (v, got[1], cache.v_scales)):
        y = y.cpu().view(B, 150, kv, D)
        for b in range(B):
            for i in range(0, 150, block):
                n = min(block, 150 - i)
                rows = x[i:i + n, b].double()  # (n, kv, D)
                top = rows.abs().amax(2).cummax(0)[0] / 127  # the scale after each token
                s = scales[table[b, i // page], i % page // block].cpu().double()
                assert torch.allclose(s, top[-1], rtol=4e-7)
                grown = torch.cat((torch.ones(1, kv), (top[1:] > top[:-1] * (1 + 1e-6)).double()))
                # Half of each scale that a value was rounded to, at most: of the scale at its own time, and after each growth.
                off = torch.stack([(top[j] + (top[j + 1:] * grown[j + 1:]).sum(0)) for j in range(n)]) * (0.5 + 2.0 ** -15)
                assert ((y[b, i:i + n].double() - rows).abs() <= off[..., None] + 1e-6 * rows.abs()).all(), (b, i)


def test_append_values_that_are_not_finite(dev):
    """A NaN or an infinity makes its block's scale NaN, of that head and of keys or values alone; later tokens of the block leave it so, a new first one ends it."""
    g = gen(5)
    kv, D = 2, 64
    cache = paged_kv.QuantizedCache.empty(2, 32, kv, D, block=16, device=dev)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
    k, v = (torch.randn(40, kv, D, generator=g) for _ in range(2))
    k[3, 0, 5], v[20, 1, 60], k[36, 1, 0] = float("nan"), float("-inf"), float("inf")
    batch = lambda new, length: paged_kv.Batch(table, *on(dev, torch.tensor([0, new], dtype=torch.int32), torch.tensor([length], dtype=torch.int32)))  # noqa: E731
    paged_kv.append(cache, batch(40, 40), k.to(dev), v.to(dev))
    ks, vs = (torch.cat((s[1], s[0])).cpu() for s in (cache.k_scales, cache.v_scales))
    assert torch.isnan(ks[:3]).tolist() == [[True, False], [False, False], [False, True]] and torch.isnan(vs[:3]).tolist() == [[False, False], [False, True], [False, False]]
    paged_kv.append(cache, batch(2, 42), k[:2].to(dev), v[:2].to(dev))
    assert torch.isnan(cache.k_scales[0, 0]).tolist() == [False, True]
    back = paged_kv.read(cache, batch(40, 42), 40, torch.float32)
    assert torch.isnan(back[0][30:, 1]).all() and not torch.isnan(back[0][30:, 0]).any() and torch.isnan(back[0][:14, 0]).all() and torch.isnan(back[1][14:30, 1]).all()
    paged_kv.append(cache, batch(16, 48), v[:16].to(dev), v[:16].to(dev))
    assert torch.isfinite(cache.k_scales[0, 0]).all()


def test_append_extremes(dev):
    """All zeros (the least scale, 1e-30), values at the ends of each type, one value that is far larger than the rest."""
    for t in TYPES.values():
        top = torch.finfo(t).max
        x = torch.zeros(48, 1, 64, dtype=t)
        x[16:32] = torch.randn(16, 1, 64, generator=gen(1)).clamp(-1, 1).to(t) * (top / 4)
        x[20, 0, 7] = -top
        x[32:] = torch.finfo(t).tiny * torch.randn(16, 1, 64, generator=gen(2)).to(t)
        x[32, 0, 0] = 5.0
        cache = paged_kv.QuantizedCache.empty(1, 48, 1, 64, block=16, device=dev)
        batch = paged_kv.Batch(*on(dev, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 48], dtype=torch.int32), torch.tensor([48], dtype=torch.int32)))
        empty = [s.cpu().clone() for s in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
        paged_kv.append(cache, batch, x.to(dev), x.to(dev))
        assert float(cache.k_scales[0, 0, 0]) == pytest.approx(1e-30) and not cache.k[0, :16].any()
        check_appended(cache.k.cpu(), cache.k_scales.cpu(), x.double(), torch.zeros_like(x, dtype=torch.float64), empty[0], empty[2], batch.table.cpu(), [0, 48], [48], 16)


def test_append_drops_what_has_no_place(dev):
    """Negative positions, positions past the table, pages that the cache does not have: nothing is written but q; starts that fall or leave the rows stay
    inside. Sequences by the thousand."""
    g = gen(32)
    table = torch.tensor([[0, 1], [2, -1], [1 << 30, 3], [4, 5]], dtype=torch.int32)
    starts, lengths = torch.tensor([1, 26, 51, 80, 98], dtype=torch.int32), torch.tensor([3, 40, 50, 70], dtype=torch.int32)
    k0, v0, ks0, vs0 = codes_of(7, 32, 1, 64, 16, g)
    k, v, q = torch.randn(100, 1, 64, generator=g), torch.randn(100, 1, 64, generator=g), torch.randn(100, 2, 64, generator=g).half()
    rot = rotary.Rotary(64, device=dev)
    kd, vd, ksd, vsd, qd = on(dev, k0, v0, ks0, vs0, q.float())
    out = torch.full((100, 2, 64), 3.0, dtype=torch.float16, device=dev)
    cache = paged_kv.QuantizedCache(kd, vd, ksd, vsd)
    paged_kv.append(cache, paged_kv.Batch(*on(dev, table, starts, lengths)), k.to(dev), v.to(dev), rotary=rot, q=qd, q_out=out)
    n = torch.cat([torch.arange(int(lengths[b]) - new, int(lengths[b])) for b, _, new, _ in sequences(starts, lengths, 100)])
    rk, koff = turned(k[1:98], n, rot)
    pad = lambda x: torch.cat((x[:1] * 0, x, x[:2] * 0))  # noqa: E731
    check_appended(kd.cpu(), ksd.cpu(), pad(rk), pad(koff), k0, ks0, table, starts, lengths, 16)
    check_appended(vd.cpu(), vsd.cpu(), v.double(), pad(koff * 0), v0, vs0, table, starts, lengths, 16)
    rq, qoff = turned(q[1:98], n, rot)
    check(out[1:98], rq, qoff, torch.float16)
    assert (out[0] == 3).all() and (out[98:] == 3).all()
    for bad in ([0, 5, 3, 1 << 30, -5], [-9, 200, 300, 400, 500], [99, 2, 2, 2, 100], [0, 100, 2, -2000000000, 50]):
        for long in ([3, 40, 50, 70], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
            batch = paged_kv.Batch(*on(dev, table, torch.tensor(bad, dtype=torch.int32), torch.tensor(long, dtype=torch.int32)))
            paged_kv.append(cache, batch, k.to(dev), v.to(dev), rotary=rot, q=qd, q_out=out)
            paged_kv.read(cache, batch, 100)
            torch.cuda.synchronize()
    B = 5000
    new = torch.randint(0, 3, (B,), generator=g)
    seqs = [(int(a), int(a) + int(c)) for a, c in zip(new, torch.randint(0, 20, (B,), generator=g))]
    table, starts, lengths, pages = batch_of(seqs, 16, g)
    T = int(starts[-1])
    k, v = (torch.randn(T, 1, 64, generator=g).half() for _ in range(2))
    k0, v0, ks0, vs0 = codes_of(pages, 16, 1, 64, 16, g)
    kd, vd, ksd, vsd = on(dev, k0, v0, ks0, vs0)
    cache, batch = paged_kv.QuantizedCache(kd, vd, ksd, vsd), paged_kv.Batch(*on(dev, table, starts, lengths))
    paged_kv.append(cache, batch, k.to(dev), v.to(dev))
    check_appended(kd.cpu(), ksd.cpu(), k.double(), k.double() * 0, k0, ks0, table, starts, lengths, 16)
    back = paged_kv.read(cache, batch, T, torch.float32)
    n = torch.cat([torch.arange(length - a, length) for a, length in seqs])
    b = torch.repeat_interleave(torch.arange(B), new)
    assert torch.equal(back[1].cpu(), vd.cpu()[table[b, n // 16].long(), n % 16].float() * vsd.cpu()[table[b, n // 16].long(), 0][..., None])
    assert paged_kv.append(cache, batch, k[:0].to(dev), v[:0].to(dev)) is None and paged_kv.read(cache, batch, 0)[0].shape == (0, 1, 64)


# ------------------------------------------------------------------------------------------------------------------ read

@pytest.mark.parametrize("page,block,D,kv", [(16, 16, 128, 2), (48, 16, 64, 3), (64, 32, 80, 5), (128, 64, 256, 9)])
@pytest.mark.parametrize("out", TYPES)
def test_read(dev, out, page, block, D, kv):
    """Exactly code x scale, rounded once; 0 behind the last sequence, at negative positions, past the table and on pages that the cache does not have."""
    g = gen(page + D)
    seqs = [(70, 70), (0, 5), (3, 200), (40, 20), (130, 130)]
    table, starts, lengths, pages = batch_of(seqs, page, g)
    table[2, 0] = pages  # not there; and the last sequence's end is past the table
    lengths[4] = table.shape[1] * page + 30
    k, v, ks, vs = codes_of(pages, page, kv, D, block, g)
    ks[int(table[0, 0]), 0, 0] = float("nan")
    vs[int(table[0, 0]), 0, 0] = float("inf")
    T = int(starts[-1]) + 3
    got = paged_kv.read(paged_kv.QuantizedCache(*on(dev, k, v, ks, vs)), paged_kv.Batch(*on(dev, table, starts, lengths)), T, TYPES[out])
    for y, c, s in ((got[0], k, ks), (got[1], v, vs)):
        want = torch.zeros(T, kv, D)
        for b, first, new, _ in sequences(starts, lengths, T):
            for i in range(new):
                n = int(lengths[b]) - new + i
                if n >= 0 and n // page < table.shape[1] and 0 <= int(table[b, n // page]) < pages:
                    p, r = int(table[b, n // page]), n % page
                    scale = s[p, r // block][:, None]
                    want[first + i] = c[p, r].float() * torch.where(torch.isfinite(scale), scale, torch.nan)
        want = want.to(TYPES[out])
        assert y.shape == want.shape and torch.equal(y.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
        assert torch.isnan(want).any()


# ------------------------------------------------------------------------------------------------------------- attention

def attend(dev, type_, D, heads, kv, page, block, seqs, seed, rows_behind=0, table_edit=None, view=None, edit=None, spread=0.3, **options):
    g = gen(seed)
    t = TYPES[type_]
    table, starts, lengths, pages = batch_of(seqs, page, g)
    k, v, ks, vs = codes_of(pages, page, kv, D, block, g, spread)
    # Blocks that no sequence holds: NaN; rows behind a sequence's end in its last block: the largest codes.
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(len(seqs)):
        n = torch.arange(min(max(int(lengths[b]), 0), table.shape[1] * page))
        used[table[b].long()[n // page], n % page] = True
    k[~used], v[~used] = 127, -127
    held = used.view(pages, page // block, block).any(-1)
    ks[~held], vs[~held] = float("nan"), float("inf")
    if edit is not None:
        edit(k, v, ks, vs, table)
    if table_edit is not None:
        table_edit(table)
    T = int(starts[-1]) + rows_behind
    q = torch.randn(T, heads, D, generator=g).to(t)
    q = torch.where(q.abs() < 2.0 ** -10, 0, q)  # as fp16 holds it
    print(f"attention {type_} D={D} heads={heads}/{kv} page={page} block={block} seqs={seqs[:6]}{'...' if len(seqs) > 6 else ''} {options}", flush=True)
    kd, vd, ksd, vsd = on(dev, k, v, ks, vs)
    if view is not None:
        kd, vd = view(kd), view(vd)
    got = paged_kv.attention(paged_kv.QuantizedCache(kd, vd, ksd, vsd), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev),
                             **{n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in options.items()})
    ref, off, mine = attended_quantized(q, k, v, ks, vs, table, starts, lengths, **options)
    assert got.shape == q.shape and got.dtype == t
    over = ref.abs() - off >= torch.finfo(t).max * (1 + torch.finfo(t).eps / 4)  # from half a step past the largest number on, values round to infinity
    assert torch.equal(got.cpu()[over].double(), ref[over].sign() * torch.inf)
    edge = ref.abs() + off >= torch.finfo(t).max
    assert torch.isfinite(got.cpu()[~edge]).all()
    check(torch.where(edge, 0, got.cpu()), torch.where(edge, 0, ref), off, t)
    assert not got.cpu()[~mine].any()
    return got


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("heads,kv,D,page,block", [(4, 1, 128, 16, 16), (6, 2, 64, 48, 16), (3, 3, 128, 64, 32), (8, 1, 64, 128, 64), (24, 24, 128, 32, 32)])
@pytest.mark.parametrize("type_", ["fp16", "bf16"])
def test_attention(dev, type_, heads, kv, D, page, block, name):
    attend(dev, type_, D, heads, kv, page, block, BATCHES[name], seed=len(name) + heads + page)


# Enough rows and KV heads that tiles of many rows are taken.
@pytest.mark.parametrize("seqs", [[(200, 200)], [(130, 1000)], [(1, 300), (260, 391), (0, 50), (1, 2), (0, 0), (297, 297)], [(150, 151), (129, 640)]])
@pytest.mark.parametrize("heads,kv,D,page,block", [(48, 24, 64, 16, 16), (24, 24, 128, 48, 16), (70, 14, 128, 32, 32), (30, 30, 64, 64, 64), (24, 24, 128, 96, 32), (44, 22, 128, 64, 64)])
@pytest.mark.parametrize("type_", ["fp16", "bf16"])
def test_wide_attention(dev, type_, heads, kv, D, page, block, seqs):
    attend(dev, type_, D, heads, kv, page, block, seqs, seed=heads + page)


@pytest.mark.parametrize("options", ["window1", "window7", "window100", "window150", "prefix", "prefix-window", "softcap", "high-cap", "slopes", "all", "scale"])
@pytest.mark.parametrize("type_,heads,kv,D,page,block", [("bf16", 24, 24, 128, 16, 16), ("fp16", 48, 24, 64, 32, 16), ("fp16", 72, 24, 128, 64, 32), ("bf16", 26, 26, 64, 64, 64),
                                                         ("fp16", 4, 2, 128, 16, 16), ("bf16", 5, 5, 64, 96, 32)])
def test_scores(dev, type_, heads, kv, D, page, block, options):
    seqs = [(130, 390), (90, 90), (3, 200), (275, 333)] if kv > 8 else [(5, 390), (1, 90), (3, 200), (1, 333)]
    slopes = torch.linspace(-0.01, 0.5, heads)
    prefix = torch.tensor([0, 50, 210, 300], dtype=torch.int32)
    o = {"window1": dict(window=1), "window7": dict(window=7), "window100": dict(window=100), "window150": dict(window=150), "prefix": dict(prefix=prefix),
         "prefix-window": dict(prefix=prefix, window=20), "softcap": dict(softcap=2.0), "high-cap": dict(softcap=5000.0), "slopes": dict(slopes=slopes),
         "all": dict(slopes=slopes, softcap=4.0, window=70, prefix=prefix), "scale": dict(scale=0.7)}[options]
    attend(dev, type_, D, heads, kv, page, block, seqs, seed=7, **o)


@pytest.mark.parametrize("new,kv", [(1, 2), (5, 2), (40, 2), (150, 24)])
@pytest.mark.parametrize("window,prefix", [(100, 4), (513, 40), (1, 1), (700, 300), (2000, 260)])
def test_first_keys_and_a_window(dev, new, kv, window, prefix):
    """A prefix of a few keys, a window, and none of the many keys between: single tokens and chunks at the end of long caches, in their midst, beside short ones
    whose window reaches the prefix, and with pages missing in the prefix, between, and in the window."""
    def edit(table):
        table[1, 0], table[1, 10], table[1, 41] = -1, 1 << 20, -5

    prefixes = torch.tensor([prefix, prefix, prefix, 0, prefix], dtype=torch.int32)
    seqs = [(new, 3000), (new, 2700), (new, max(new, 350)), (new, 1500), (new, 1024)]
    attend(dev, "fp16", 64, 2 * kv, kv, 64, 32, seqs, seed=21, table_edit=edit, window=window, prefix=prefixes)
    attend(dev, "bf16", 128, kv, kv, 48, 16, seqs[:2], seed=22, window=window, prefix=prefixes[:2], softcap=20.0)


@pytest.mark.parametrize("type_,D,options", [("fp16", 128, {}), ("bf16", 64, dict(softcap=30.0)), ("fp16", 64, dict(window=9000)), ("bf16", 128, dict(window=12000, prefix=70))])
def test_long_runs(dev, type_, D, options):
    """Runs of more tiles than their lanes hold scales and pages of (64): 64 KV heads, two tiles of 128 rows each, over 17000 keys; eight of the heads against 64 bits."""
    g = gen(53)
    t, kv, page, block, new, length = TYPES[type_], 64, 64, 32, 150, 17000
    table, starts, lengths, pages = batch_of([(new, length)], page, g)
    k, v, ks, vs = on(dev, *codes_of(pages, page, kv, D, block, g, spread=0.6))
    q = torch.randn(new, kv, D, generator=g).to(t)
    q = torch.where(q.abs() < 2.0 ** -10, 0, q)
    o = dict(options)
    if "prefix" in o:
        o["prefix"] = torch.tensor([o["prefix"]], dtype=torch.int32)
    got = paged_kv.attention(paged_kv.QuantizedCache(k, v, ks, vs), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev),
                             **{n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in o.items()})
    for h in range(0, kv, 8):
        one = slice(h, h + 1)
        ref, off, _ = attended_quantized(q[:, one], *(x[:, :, one].cpu() for x in (k, v, ks, vs)), table, starts, lengths, **o)
        check(got[:, one], ref, off, t)


@pytest.mark.parametrize("type_,D,missing,options", [("fp16", 128, (0, 100, 265), {}), ("bf16", 64, (3, 131, 200), dict(softcap=30.0)), ("fp16", 64, (130, 190), dict(window=9000, prefix=70))])
def test_missing_pages_in_long_runs(dev, type_, D, missing, options):
    """Pages that the cache does not have, where they lie in the first tiles of a run, past its 64th, or at its end: their keys are masked, whatever the codes that are read instead."""
    g = gen(54)
    t, kv, page, block, new, length = TYPES[type_], 64, 64, 32, 150, 17000
    table, starts, lengths, pages = batch_of([(new, length)], page, g)
    for i, at in enumerate(missing):
        table[0, at] = (-1, pages, 2 ** 31 - 1)[i]
    k, v, ks, vs = on(dev, *codes_of(pages, page, kv, D, block, g))
    vs[0] *= 1000.0  # what page 0 holds would show
    table[0][table[0] == 0] = 1
    q = torch.randn(new, kv, D, generator=g).to(t)
    q = torch.where(q.abs() < 2.0 ** -10, 0, q)
    o = dict(options)
    if "prefix" in o:
        o["prefix"] = torch.tensor([o["prefix"]], dtype=torch.int32)
    got = paged_kv.attention(paged_kv.QuantizedCache(k, v, ks, vs), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev),
                             **{n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in o.items()})
    for h in range(3, kv, 12):
        one = slice(h, h + 1)
        ref, off, _ = attended_quantized(q[:, one], *(x[:, :, one].cpu() for x in (k, v, ks, vs)), table, starts, lengths, **o)
        check(got[:, one], ref, off, t)


@pytest.mark.parametrize("type_,kv", [("fp16", 2), ("bf16", 2), ("fp16", 24), ("bf16", 24)])
def test_rows_that_see_nothing(dev, type_, kv):
    """Lengths below the new tokens (negative positions), lengths of zero, pages that the cache does not have, rows behind the last sequence."""
    def edit(table):
        table[1, :2] = torch.tensor([-1, 1 << 20])
        table[2] = -7
    attend(dev, type_, 64, 2 * kv, kv, 16, 16, [(140, 20), (60, 60), (3, 40), (1, 0), (150, 200)], seed=11, rows_behind=5, table_edit=edit)
    attend(dev, type_, 128, kv, kv, 64, 32, [(150, 100), (2, 1), (160, 0)], seed=12, rows_behind=1, window=3)


@pytest.mark.parametrize("type_", ["fp16", "bf16"])
@pytest.mark.parametrize("new,length,kv", [(1, 200, 2), (5, 90, 2), (130, 180, 24)])
def test_blocks_of_nan(dev, type_, new, length, kv):
    """A block whose scale is not finite makes NaN of every row that sees any of its keys, and leaves the others as they are."""
    D, page, block = 64, 32, 16
    for which, bad in (("k", float("nan")), ("v", float("nan")), ("k", float("inf")), ("v", float("inf"))):
        g = gen(13)
        table, starts, lengths, pages = batch_of([(new, length), (new, length)], page, g)
        k, v, ks, vs = codes_of(pages, page, kv, D, block, g)
        q = torch.randn(2 * new, kv, D, generator=g).to(TYPES[type_])
        q = torch.where(q.abs() < 2.0 ** -10, 0, q)
        first = length - new // 2 - 1  # a position in a block that some rows see part of
        part = (int(table[0, first // page]), first % page // block, 0)
        clean = paged_kv.attention(paged_kv.QuantizedCache(*on(dev, k, v, ks, vs)), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev)).cpu()
        (ks if which == "k" else vs)[part] = bad
        got = paged_kv.attention(paged_kv.QuantizedCache(*on(dev, k, v, ks, vs)), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev)).cpu()
        sees = torch.zeros(2 * new, kv, dtype=torch.bool)
        sees[:new, 0] = torch.arange(length - new, length) >= first // block * block
        assert torch.isnan(got[sees]).all(), (which, bad)
        print(type_, new, which, bad, flush=True)
        ref, off, _ = attended_quantized(q, k, v, torch.where(torch.isfinite(ks), ks, 0), torch.where(torch.isfinite(vs), vs, 0), table, starts, lengths)
        check(got, ref, off, TYPES[type_], rows=~sees)
        assert torch.isfinite(clean).all()


@pytest.mark.parametrize("new,kv", [(1, 2), (130, 24)])
def test_scales_far_apart(dev, new, kv):
    """Values of one block 10^6 times the others', seen by all, by some, or by later rows only: the rows that do not see it keep their precision. Keys whose
    scores are far from zero. Caches of tiny and of large values."""
    D, page, block = 128, 32, 16

    def large(at, by=1e6):
        def edit(k, v, ks, vs, table):
            vs[int(table[0, at // page]), at % page // block] *= by
        return edit

    for at in (0, 200, 299):
        attend(dev, "fp16", D, kv, kv, page, block, [(new, 300), (new, 260)], seed=14, edit=large(at))
        attend(dev, "bf16", D, kv, kv, page, block, [(new, 300), (new, 260)], seed=15, edit=large(at, 1e-6))
    attend(dev, "fp16", D, kv, kv, page, block, [(new, 300)], seed=16, spread=2.5)

    def sized(by_k, by_v):
        def edit(k, v, ks, vs, table):
            ks *= by_k
            vs *= by_v
        return edit

    attend(dev, "bf16", D, kv, kv, page, block, [(new, 300)], seed=17, edit=sized(30.0, 1e8))
    attend(dev, "fp16", D, kv, kv, page, block, [(new, 300)], seed=18, edit=sized(1e-20, 1e-3))
    attend(dev, "bf16", D, kv, kv, page, block, [(new, 300)], seed=19, edit=sized(1e-20, 1e-25))


@pytest.mark.parametrize("type_", ["fp16", "bf16"])
@pytest.mark.parametrize("new,kv,D", [(1, 2, 64), (1, 2, 128), (3, 8, 128), (130, 24, 128), (130, 24, 64)])
def test_scales_of_zero(dev, type_, new, kv, D):
    """Blocks whose scales are 0, as `empty` makes them, at the start, between others and at the end: their keys' scores and their values are 0. A cache of nothing
    but those. Sequences that share their first pages, and a table whose entries past a length are anything."""
    page, block = 32, 16

    def nothing(which, *at):
        def edit(k, v, ks, vs, table):
            for n in at:
                for s in which(ks, vs):
                    s[int(table[0, n // page]), n % page // block] = 0.0
        return edit

    for at in ((0, 16), (100, 116, 200), (299,), tuple(range(0, 300, 16))):
        attend(dev, type_, D, kv, kv, page, block, [(new, 300), (new, 260)], seed=24, edit=nothing(lambda ks, vs: (vs,), *at))
        attend(dev, type_, D, kv, kv, page, block, [(new, 300), (new, 260)], seed=25, edit=nothing(lambda ks, vs: (ks,), *at))
        attend(dev, type_, D, kv, kv, page, block, [(new, 300), (new, 260)], seed=26, edit=nothing(lambda ks, vs: (ks, vs), *at), softcap=20.0)
    cache = paged_kv.QuantizedCache.empty(12, page, kv, D, block, dev)
    batch = paged_kv.Batch(*on(dev, torch.arange(10, dtype=torch.int32)[None], torch.tensor([0, new], dtype=torch.int32), torch.tensor([300], dtype=torch.int32)))
    assert not paged_kv.attention(cache, batch, torch.ones(new, kv, D, dtype=TYPES[type_], device=dev)).any()

    def shared(table):
        table[1, :8] = table[0, :8]
        table[1, 9:] = 2 ** 31 - 1  # (its length ends in page 8)

    attend(dev, type_, D, kv, kv, page, block, [(new, 300), (new, 270)], seed=27, table_edit=shared)


def test_rows_of_queries_far_from_one(dev):
    """Rows of q of 10^-30 to 10^30 beside one another, with zeros; a row that is not finite is NaN alone."""
    g = gen(20)
    kv, D = 2, 64
    table, starts, lengths, pages = batch_of([(7, 100)], 16, g)
    k, v, ks, vs = codes_of(pages, 16, kv, D, 16, g)
    q = torch.randn(7, kv, D, generator=g).bfloat16()
    for i, by in enumerate((1.0, 1e-30, 1e30, 0.0, 1e4, 1.0, 1.0)):
        q[i] *= by
    q[6, 1, 3] = float("inf")
    cache, batch = paged_kv.QuantizedCache(*on(dev, k, v, ks, vs)), paged_kv.Batch(*on(dev, table, starts, lengths))
    got = paged_kv.attention(cache, batch, q.to(dev), scale=0.01).cpu().double()
    kp, vp = (values(c, s)[table[0].long()].reshape(-1, kv, D)[:100] for c, s in ((k, ks), (v, vs)))
    for i in (0, 1, 3, 4, 5):
        for h in range(kv):
            x = q[i, h].double() @ kp[:94 + i, h].T * 0.01
            w = torch.softmax(x, 0)
            size = (q[i, h].double().abs() @ kp[:94 + i, h].abs().T * 0.01).max()
            off = (w @ vp[:94 + i, h].abs()) * 2 * (2.0 ** -11 + 70 * 2.0 ** -24 * size + 2.0 ** -20)
            ref = w @ vp[:94 + i, h]
            assert ((got[i, h] - ref).abs() <= off + rounding(ref.abs() + off, torch.bfloat16)).all(), (i, h)
    for h in range(kv):  # scores of 10^29: the largest takes all
        x = q[2, h].double() @ kp[:96, h].T
        assert ((got[2, h] - vp[x.argmax(), h]).abs() <= rounding(vp[x.argmax(), h].abs(), torch.bfloat16) + vp[x.argmax(), h].abs() * 2.0 ** -10).all()
    assert torch.isnan(got[6, 1]).all() and torch.isfinite(got[6, 0]).all() and torch.isfinite(got[:6]).all()


def test_many_sequences(dev):
    g = gen(14)
    seqs = [(int(n), int(n) + int(c)) for n, c in zip(torch.randint(0, 3, (700,), generator=g), torch.randint(0, 60, (700,), generator=g))]
    attend(dev, "bf16", 64, 4, 2, 16, 16, seqs, seed=15)


def test_rows_of_no_sequence(dev):
    """An out of the caller keeps the rows that belong to no sequence; starts that leave the rows, or fall, stay inside them; lengths past the table."""
    g = gen(16)
    table = torch.randperm(8, generator=g)[:6].to(torch.int32).view(2, 3)
    k, v, ks, vs = codes_of(8, 16, 1, 64, 16, g)
    q = torch.randn(9, 2, 64, generator=g).half()
    q = torch.where(q.abs() < 2.0 ** -10, 0, q)
    cache = paged_kv.QuantizedCache(*on(dev, k, v, ks, vs))
    starts, lengths = torch.tensor([2, 4, 7], dtype=torch.int32), torch.tensor([40, 2 ** 31 - 1], dtype=torch.int32)
    out = torch.full((9, 2, 64), 3.0, dtype=torch.float16, device=dev)
    version = out._version
    assert paged_kv.attention(cache, paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev), out=out) is out and out._version > version
    ref, off, mine = attended_quantized(q, k, v, ks, vs, table, starts, lengths)
    assert (out.cpu()[~mine] == 3).all()
    check(out[2:7], ref[2:7], off[2:7], torch.float16)
    guard = torch.zeros(29, 2, 64, dtype=torch.float16, device=dev)
    for bad in ([0, 2, 1 << 30], [0, 5, 3], [-4, 100, -100]):
        paged_kv.attention(cache, paged_kv.Batch(*on(dev, table, torch.tensor(bad, dtype=torch.int32), lengths)), q.to(dev), out=guard[10:19])
        torch.cuda.synchronize()
        assert not guard[:10].any() and not guard[19:].any()


def test_orders_of_memory(dev):
    """Pools with heads before tokens, with K and V in one tensor, rows with gaps; scales of any strides; q as a part of a projection, and unaligned."""
    seqs = [(1, 100), (20, 45)]
    attend(dev, "fp16", 64, 4, 2, 16, 16, seqs, seed=18, view=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    attend(dev, "bf16", 128, 4, 2, 32, 16, seqs, seed=19, view=lambda t: torch.stack((t, t * 0), 1)[:, 0])
    attend(dev, "fp16", 64, 4, 2, 64, 32, seqs, seed=20, view=lambda t: torch.cat((t, t * 0), 3)[..., :64])
    g = gen(22)
    table, starts, lengths, pages = batch_of(seqs, 32, g)
    k, v, ks, vs = codes_of(pages, 32, 2, 64, 16, g)
    other = lambda s: torch.stack((s, s * 0), 3).to(dev)[..., 0]  # noqa: E731
    turned_scales = lambda s: s.to(dev).permute(2, 0, 1).contiguous().permute(1, 2, 0)  # noqa: E731
    cache, batch = paged_kv.QuantizedCache(k.to(dev), v.to(dev), other(ks), turned_scales(vs)), paged_kv.Batch(*on(dev, table, starts, lengths))
    fused = torch.randn(21, 8 * 64, generator=g).half()
    fused = torch.where(fused.abs() < 2.0 ** -10, 0, fused)
    q = fused.view(21, 8, 64)[:, :4]
    ref, off, _ = attended_quantized(q, k, v, ks, vs, table, starts, lengths)
    check(paged_kv.attention(cache, batch, fused.to(dev).view(21, 8, 64)[:, :4]), ref, off, torch.float16)
    odd = torch.cat((torch.zeros(1), q.flatten())).half()
    check(paged_kv.attention(cache, batch, odd.to(dev)[1:].view(21, 4, 64)), ref, off, torch.float16)
    back, plain = paged_kv.read(cache, batch, 21, torch.float32), paged_kv.read(paged_kv.QuantizedCache(*on(dev, k, v, ks, vs)), batch, 21, torch.float32)
    assert torch.equal(back[0], plain[0]) and torch.equal(back[1], plain[1])


def test_offsets_past_32_bits(dev):
    """Codes past 2^32 bytes: the last pages are written, read back and attended to."""
    g = gen(23)
    P, S, kv, D = 264000, 16, 8, 128
    k, v = (torch.empty(P, S, kv, D, dtype=torch.int8, device=dev) for _ in range(2))
    assert k.numel() > 2 ** 32
    scales = [torch.zeros(P, 1, kv, device=dev) for _ in range(2)]
    table = torch.tensor([[P - 1, 3, P - 2]], dtype=torch.int32)
    starts, lengths = torch.tensor([0, 40], dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    kn, vn = (torch.randn(40, kv, D, generator=g).bfloat16() for _ in range(2))
    cache, batch = paged_kv.QuantizedCache(k, v, *scales), paged_kv.Batch(*on(dev, table, starts, lengths))
    paged_kv.append(cache, batch, kn.to(dev), vn.to(dev))
    back = paged_kv.read(cache, batch, 40, torch.float32)
    pages = table[0].long()
    small = [t[pages.to(dev)].cpu() for t in (k, v, *scales)]
    for x, y, s in ((kn, back[0], small[2]), (vn, back[1], small[3])):
        step = s.repeat_interleave(16, 1).reshape(48, kv)[:40, :, None]
        assert ((y.cpu() - x.float()).abs() <= step * 0.501).all() and (step > 0).all()
    q = torch.randn(40, 8, D, generator=g).bfloat16()
    q = torch.where(q.abs() < 2.0 ** -10, 0, q)
    ref, off, _ = attended_quantized(q, *small, torch.tensor([[0, 1, 2]], dtype=torch.int32), starts, lengths)
    check(paged_kv.attention(cache, batch, q.to(dev)), ref, off, torch.bfloat16)


@pytest.mark.parametrize("seed", range(16))
def test_random(dev, seed):
    """Seeded random batches, heads, pages, blocks and scores."""
    g = gen(1900 + seed)
    pick = lambda *a: a[int(torch.randint(0, len(a), (1,), generator=g))]  # noqa: E731
    upto = lambda n: int(torch.randint(0, n + 1, (1,), generator=g))  # noqa: E731
    kv = pick(1, 2, 3, 20)
    heads = kv * pick(1, 2, 5, 8, 16 if kv < 4 else 3)
    seqs = []
    for _ in range(1 + upto(6)):
        new = pick(1, 1, upto(4), upto(90), upto(200))
        seqs.append((new, new + upto(pick(10, 200, 900))))
    if sum(new for new, _ in seqs) == 0:
        seqs.append((1, 9))
    o = {}
    if upto(2) == 0:
        o["window"] = 1 + upto(150)
    if upto(3) == 0:
        o["softcap"] = 5.0
    if upto(3) == 0:
        o["slopes"] = torch.rand(heads, generator=g)
    if upto(3) == 0:
        o["prefix"] = torch.randint(0, 150, (len(seqs),), generator=g, dtype=torch.int32)
    block = pick(16, 32, 64)
    attend(dev, pick("fp16", "bf16"), pick(64, 128), heads, kv, block * pick(1, 2, 3), block, seqs, seed=seed, rows_behind=upto(2), spread=pick(0.1, 0.5, 1.5), **o)


# ------------------------------------------------------------------------------------------------------- a run of them together

@pytest.mark.parametrize("type_", ["fp16", "bf16", "fp32"])
def test_serving_steps(dev, type_):
    """Prompts in chunks, then single tokens, of sequences that come, grow and take new pages: each step norms, turns and appends, and attends. Every output is dense
    causal attention over the sequence's whole history as it reads back, in 64 bits; what reads back is near the history itself."""
    g = gen(41)
    t = TYPES[type_]
    ot = torch.bfloat16 if type_ == "fp32" else t
    kv, heads, D, page, pages = 2, 8, 64, 32, 20
    rot = rotary.Rotary(D, base=1e6, device=dev)
    norm = rotary.HeadNorm(*((1 + 0.2 * torch.randn(D, generator=g)).to(dev) for _ in range(2)))
    cache = paged_kv.QuantizedCache.empty(pages, page, kv, D, block=16, device=dev)
    cache.k_scales.fill_(float("nan"))
    cache.v_scales.fill_(float("nan"))
    free = torch.randperm(pages, generator=g).tolist()
    held, done = [[] for _ in range(3)], [0, 0, 0]
    history = [[torch.zeros(0, kv, D), torch.zeros(0, kv, D)] for _ in range(3)]
    for step, new in enumerate([(40, 0, 0), (30, 17, 0), (1, 1, 0), (1, 1, 9), (1, 1, 1), (1, 0, 1), (1, 1, 1)]):
        for b in range(3):
            done[b] += new[b]
            while len(held[b]) * page < done[b]:
                held[b].append(free.pop())
        table = torch.zeros(3, 6, dtype=torch.int32)
        for b in range(3):
            table[b, :len(held[b])] = torch.tensor(held[b], dtype=torch.int32)
        starts = torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        lengths = torch.tensor(done, dtype=torch.int32)
        batch = paged_kv.Batch(*on(dev, table, starts, lengths))
        T = sum(new)
        q, k, v = (torch.randn(T, h, D, generator=g).to(t) for h in (heads, kv, kv))
        print(f"step {step} {type_} new={new}", flush=True)
        qr = paged_kv.append(cache, batch, k.to(dev), v.to(dev), rotary=rot, q=q.to(dev), q_out=torch.empty(T, heads, D, dtype=ot, device=dev), norm=norm)
        n = torch.cat([torch.arange(done[b] - new[b], done[b], device=dev) for b in range(3)])
        qn, kn = rotary.norm_rotate(q.to(dev), k.to(dev), n, rot, norm)
        assert torch.equal(qr, qn.to(ot))
        out = paged_kv.attention(cache, batch, qr)
        whole = paged_kv.Batch(*on(dev, table, torch.tensor([0, *done], dtype=torch.int32).cumsum(0, dtype=torch.int32), lengths))
        back = [x.cpu() for x in paged_kv.read(cache, whole, sum(done), torch.float32)]
        at = 0
        for b in range(3):
            rows = slice(int(starts[b]), int(starts[b + 1]))
            history[b][0] = torch.cat((history[b][0], kn.cpu()[rows].float()))
            history[b][1] = torch.cat((history[b][1], v[rows].float()))
            mine = [x[at:at + done[b]] for x in back]
            at += done[b]
            for x, y in zip(mine, history[b]):  # three growths of a scale of values below 6, at most, on average
                assert done[b] == 0 or (x - y).norm() <= 0.02 * y.norm()
            if new[b]:
                ref, off = dense(qr[rows].cpu(), mine, new[b])
                check(out[rows], ref, off, ot)


def dense(q, kv_values, new):
    """Causal attention of the last `new` rows over k and v (length, KV heads, D) in 64 bits, and its bound."""
    k, v = (x.double() for x in kv_values)
    length, group = len(k), q.shape[1] // k.shape[1]
    out, off = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    hidden = torch.arange(length) > torch.arange(length - new, length)[:, None]
    for h in range(q.shape[1]):
        qd, kh, vh = q[:, h].double(), k[:, h // group], v[:, h // group]
        w = torch.softmax((qd @ kh.T * q.shape[2] ** -0.5).masked_fill(hidden, -torch.inf), -1)
        size = (qd.abs() @ kh.abs().T * q.shape[2] ** -0.5).masked_fill(hidden, 0).amax(1, keepdim=True)
        out[:, h] = w @ vh
        # Products and sums of D and of the keys' terms in 32 bits, P rounded to fp16 once.
        off[:, h] = (w @ vh.abs()) * 2 * ((q.shape[2] + 8) * 2.0 ** -24 * size + 2.0 ** -11 + (length + 16) * 2.0 ** -24)
    return out, off


def test_captured_steps(dev):
    """Two captured graphs of append, attention and reading back, their batches' contents changed between replays, with eager calls between and beside:
    each replay equals the eager calls on the same contents, bit for bit."""
    g = gen(42)
    kv, heads, D, page, B = 2, 8, 128, 32, 4
    rot = rotary.Rotary(D, device=dev)

    def world(seed):
        h = gen(seed)
        cache = paged_kv.QuantizedCache(*on(dev, *codes_of(64, page, kv, D, 16, h)))
        batch = paged_kv.Batch(*on(dev, torch.randperm(64, generator=h)[:B * 12].view(B, 12).to(torch.int32), torch.arange(B + 1, dtype=torch.int32),
                                   torch.tensor([3, 60, 150, 1], dtype=torch.int32)))
        norm = rotary.HeadNorm(*(torch.ones(D, device=dev) for _ in range(2)))
        return cache, batch, norm, *(torch.randn(B, n, D, generator=h).bfloat16().to(dev) for n in (heads, kv, kv))

    def step(w, out=None):
        cache, batch, norm, q, k, v = w
        qr = paged_kv.append(cache, batch, k, v, rotary=rot, q=q, q_out=torch.empty_like(q), norm=norm)
        return (paged_kv.attention(cache, batch, qr, out=out), *paged_kv.read(cache, batch, B))

    worlds, graphs, outs = [world(50), world(51)], [], []
    for w in worlds:
        step(w)
        torch.cuda.synchronize()
        graph, out = torch.cuda.CUDAGraph(), torch.zeros(B, heads, D, dtype=torch.bfloat16, device=dev)
        with torch.cuda.graph(graph):
            got = step(w, out)
        graphs.append(graph)
        outs.append(got)
    side = torch.cuda.Stream()
    for i in range(5):
        for w in worlds:
            w[1].lengths += 1 + 3 * i
            for t in w[3:]:
                t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for w, out in zip(worlds, outs):
            want = step(w)  # appends the same tokens again: the same codes
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_calls_at_once(dev):
    """Calls on two streams at a time, each on its own cache, give the bits of calls one by one."""
    jobs = []
    for s in range(4):
        g = gen(60 + s)
        kv, seqs = (2, [(1, 900 + 100 * s), (60, 300), (1, 5)]) if s % 2 else (24, [(1, 900), (160, 300 + 50 * s), (140, 140)])
        table, starts, lengths, pages = batch_of(seqs, 16, g)
        cache = paged_kv.QuantizedCache(*on(dev, *codes_of(pages, 16, kv, 128, 16, g)))
        jobs.append((cache, paged_kv.Batch(*on(dev, table, starts, lengths)), torch.randn(int(starts[-1]), 2 * kv, 128, generator=g).half().to(dev)))
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
