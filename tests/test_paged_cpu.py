"""The host side of rotary and paged_kv on the CPU: the frequencies against their definitions, what each call refuses (before any
launch), the entry points' own argument checks, and the 64-bit forms that the GPU tests compare with, against torch's attention."""
import ctypes
import math
import types

import pytest
import torch

from comfyui_rdna2_attention_amd import _lib, paged_kv, rotary
from helpers import gen
from paged_reference import appended, attended, turned


def test_frequencies_plain_and_linear():
    f, factor = rotary.frequencies(8, base=100.0)
    assert factor == 1.0 and f == pytest.approx([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rel=1e-15)
    assert rotary.frequencies(8, base=100.0, scaling="linear", factor=4.0)[0] == pytest.approx([x / 4 for x in f], rel=1e-15)


def test_frequencies_ntk():
    """The fastest pair is left alone, the slowest one divided by the factor."""
    f, g = rotary.frequencies(64)[0], rotary.frequencies(64, scaling="ntk", factor=8.0)[0]
    assert g[0] == f[0] == 1.0 and g[-1] == pytest.approx(f[-1] / 8, rel=1e-12)


def test_frequencies_bands():
    f, g = rotary.frequencies(64)[0], rotary.frequencies(64, scaling="bands", factor=8.0, original=1000, low=1.0, high=4.0)[0]
    for a, b in zip(f, g):
        turns = 1000 * a / (2 * math.pi)
        want = a if turns >= 4 else a / 8 if turns <= 1 else a / 8 + (a - a / 8) * (turns - 1) / 3
        assert b == pytest.approx(want, rel=1e-13)
    assert len({round(b / a, 6) for a, b in zip(f, g)}) > 3


def test_frequencies_yarn():
    f, (g, factor) = rotary.frequencies(64)[0], rotary.frequencies(64, scaling="yarn", factor=4.0, original=4096)
    assert factor == pytest.approx(0.1 * math.log(4) + 1)
    pair = lambda turns: 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(1e4))  # noqa: E731
    lo, hi = math.floor(pair(32)), math.ceil(pair(1))
    for i, (a, b) in enumerate(zip(f, g)):
        mix = min(max((i - lo) / (hi - lo), 0), 1)
        assert b == pytest.approx(a * (1 - mix) + a / 4 * mix, rel=1e-13)
    assert rotary.frequencies(64, scaling="yarn", factor=1.0, original=4096) == (pytest.approx(f), 1.0)


@pytest.mark.parametrize("options", [dict(dim=7), dict(dim=8, base=0.0), dict(dim=8, scaling="other"), dict(dim=8, scaling="bands"), dict(dim=2, scaling="ntk", factor=2.0),
                                     dict(dim=8, scaling="bands", original=10, low=4.0, high=4.0), dict(dim=8, scaling="yarn", original=10, slow=40.0),
                                     dict(dim=8, scaling="linear", factor=0.0)])
def test_frequencies_refusals(options):
    with pytest.raises(ValueError):
        rotary.frequencies(**options)


def test_rotary():
    r = rotary.Rotary(32, base=1e6, layout="interleaved", scaling="yarn", factor=2.0, original=100, device="cpu")
    f, factor = rotary.frequencies(32, 1e6, "yarn", factor=2.0, original=100)
    assert r.turns.dtype == torch.float64 and r.turns.tolist() == pytest.approx([x / (2 * math.pi) for x in f], rel=1e-15) and r.factor == factor
    r = rotary.Rotary(16, radians=[0.5] * 8, attention=1.25, device="cpu")
    assert r.factor == 1.25 and r.turns[0] == 0.5 / (2 * math.pi)
    for bad in (dict(dim=8), dict(dim=272), dict(dim=0), dict(dim=16, layout="other"), dict(dim=16, radians=[1.0]), dict(dim=16, radians=[1.0] * 8, scaling="ntk"),
                dict(dim=16, radians=[1.0] * 8, factor=2.0)):
        with pytest.raises(ValueError):
            rotary.Rotary(**bad, device="cpu")


def test_rotate_refusals():
    r = rotary.Rotary(32, device="cpu")
    x, n = torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int32)
    for bad in ((x.double(), n), (x[..., :40], n), (x[..., :16], n), (x[0], n), (x, n[:3]), (x, n.float()), (torch.zeros(4, 2, 272), n)):
        with pytest.raises(ValueError):
            rotary.rotate(*bad, r)
    for out in (x[:3], x.half(), torch.zeros(4, 2, 128)[..., ::2], torch.zeros(4 * 128 + 1)[1:].view(4, 2, 64)):
        with pytest.raises(ValueError):
            rotary.rotate(x, n, r, out=out)
    with pytest.raises(ValueError, match="current GPU"):
        rotary.rotate(x, n, r)


def test_cache_and_batch_refusals():
    k = torch.zeros(4, 8, 2, 64)
    for bad in ((k, k[:3]), (k, k.half()), (k.double(), k.double()), (k[0], k[0]), (k[..., :24], k[..., :24]), (k[:0], k[:0]), (k[..., :32], k[..., 32:].transpose(0, 1)),
                (torch.zeros(4, 8, 2, 66)[..., :64],) * 2, (torch.zeros(4 * 1024 + 1)[1:].view(4, 8, 2, 64),) * 2, (torch.zeros(4, 8, 2, 128)[..., ::2],) * 2):
        with pytest.raises(ValueError):
            paged_kv.Cache(*bad)
    table, starts, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    paged_kv.Batch(table, starts, lengths)
    paged_kv.Batch(torch.zeros(2, 9, dtype=torch.int32)[:, :3], starts, lengths)
    for bad in ((table.long(), starts, lengths), (table, starts.long(), lengths), (table, starts, lengths.float()), (table, starts[:2], lengths),
                (table, starts, lengths[:1]), (table[:, :0], starts, lengths), (table.view(-1), starts, lengths), (table[:0], starts[:1], lengths[:0]),
                (table.t().contiguous().t(), starts, lengths), (table, torch.zeros(6, dtype=torch.int32)[::2], lengths),
                (torch.zeros(8193, 1, dtype=torch.int32), torch.zeros(8194, dtype=torch.int32), torch.zeros(8193, dtype=torch.int32))):
        with pytest.raises(ValueError):
            paged_kv.Batch(*bad)


def test_outputs_of_one_memory_are_refused():
    """Expanded views as outputs: two rows would be written to one place."""
    rot, pos = rotary.Rotary(64, device="cpu"), torch.zeros(4, dtype=torch.int32)
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    for out in (x[:1].expand(4, 2, 64), x[:, :1].expand(4, 2, 64)):
        with pytest.raises(ValueError, match="each its own"):
            rotary.rotate(x, pos, rot, out=out)
        pages = torch.zeros(3, 8, 2, 64, dtype=torch.float16)
        cache = paged_kv.Cache(pages, pages.clone())
        batch = paged_kv.Batch(torch.zeros(1, 3, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32), torch.tensor([4], dtype=torch.int32))
        with pytest.raises(ValueError, match="each its own"):
            paged_kv.attention(cache, batch, x, out=out)
        with pytest.raises(ValueError, match="each its own"):
            paged_kv.append(cache, batch, x, x, q=x, q_out=out)
    one = paged_kv.Cache(pages[:, :, :1].expand(3, 8, 2, 64), pages)
    with pytest.raises(ValueError, match="one memory"):
        paged_kv.append(one, batch, x, x)


def test_calls_of_too_many_tokens_are_refused():
    """A grid has fewer than 2^32 threads; the sizes alone are looked at."""
    rot, n = rotary.Rotary(16, device="cpu"), rotary.MAX_TOKENS + 1
    x = torch.zeros(1, 1, 16, dtype=torch.float16).expand(n, 1, 16)
    with pytest.raises(ValueError, match="at most"):
        rotary.rotate(x, torch.zeros(1, dtype=torch.int32).expand(n), rot, out=x)
    pages = torch.zeros(3, 8, 1, 16, dtype=torch.float16)
    batch = paged_kv.Batch(torch.zeros(1, 3, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32), torch.tensor([4], dtype=torch.int32))
    with pytest.raises(ValueError, match="at most"):
        paged_kv.append(paged_kv.Cache(pages, pages.clone()), batch, x, x)
    lib = _lib.declare(ctypes.CDLL(_lib.LIB_PATH))
    a = 1 << 20
    for B, L in ((1, n), (n, 1), (1 << 14, 1 << 13), (1 << 40, 1 << 40)):
        assert lib.rda_rotate_positions(a, a, a, 0, a, 1.0, 0, 0, _lib.long_array([B, L, 1, 16, 16, 16, 16, 16, 16, 16, 16]), None) == 1
    dims = dict(T=n, H=0, Hkv=1, D=16, R=0, B=1, N=3, pitch=3, P=3, S=8, qt=0, qh=0, kt=16, kh=16, vt=16, vh=16, ot=0, oh=0, kp=128, kr=16, ch=16, vp=128, vr=16, wh=16)
    assert lib.rda_paged_append(None, a, a, None, a, a, a, a, a, None, 1.0, 0, 0, 0, _lib.long_array(list(dims.values())), None) == 1


def test_handles_keep_what_was_checked():
    cache, batch = handles()
    batch.lengths += 3
    assert batch.lengths.tolist() == [3, 3]
    batch.starts = torch.ones(3, dtype=torch.int32)
    assert batch.starts.tolist() == [1, 1, 1]
    for name, t in (("lengths", torch.zeros(3, dtype=torch.int32)), ("starts", torch.zeros(3)), ("table", torch.zeros(2, 4, dtype=torch.int32)),
                    ("lengths", torch.zeros(4, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            setattr(batch, name, t)
    with pytest.raises(AttributeError):
        cache.k = cache.v


def handles(dtype=torch.float32, D=64):
    cache = paged_kv.Cache(torch.zeros(4, 8, 2, D, dtype=dtype), torch.zeros(4, 8, 2, D, dtype=dtype))
    return cache, paged_kv.Batch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_append_refusals():
    cache, batch = handles(torch.float16)
    k, q = torch.zeros(3, 2, 64), torch.zeros(3, 4, 64)
    o = q.half()
    for bad in (dict(k=k.double(), v=k.double()), dict(k=k, v=k.half()), dict(k=k, v=k[:2]), dict(k=k[:, :1], v=k[:, :1]), dict(k=k[..., :48], v=k[..., :48]),
                dict(k=k, v=k, q=q), dict(k=k, v=k, q=q.half(), q_out=o), dict(k=k, v=k, q=q[:2], q_out=o[:2]), dict(k=k, v=k, q=q, q_out=o[:2]),
                dict(k=k, v=k, q=q[..., :32], q_out=o[..., :32]), dict(k=k, v=k, q_out=o), dict(k=k, v=k, q=q[:, :0], q_out=o[:, :0]),
                dict(k=k, v=k, q=q, q_out=torch.zeros(3, 4, 128, dtype=torch.float16)[..., ::2]), dict(k=k, v=k, rotary=rotary.Rotary(80, device="cpu"))):
        with pytest.raises(ValueError):
            paged_kv.append(cache, batch, **bad)
    with pytest.raises(ValueError, match="current GPU"):
        paged_kv.append(cache, batch, k, k, q=q, q_out=o)
    wide = types.SimpleNamespace(sizes=((1, 2 ** 28), 2 ** 28))
    with pytest.raises(ValueError, match="at most 2147418112 tokens"):
        paged_kv.append(cache, wide, k, k)


def test_attention_refusals():
    cache, batch = handles()
    q = torch.zeros(3, 4, 64)
    f, i = torch.zeros(4), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q[:, :0]), dict(q=q, out=q), dict(q=q, out=q[:2].clone()),
                dict(q=q, out=q.half()), dict(q=q, out=torch.zeros(3, 4, 128)[..., ::2]), dict(q=q, softcap=-1.0), dict(q=q, softcap=float("nan")), dict(q=q, scale=0.0), dict(q=q, scale=-0.1), dict(q=q, scale=float("inf")), dict(q=q, scale=float("nan")),
                dict(q=q, softcap=1e-35), dict(q=q, softcap=float("inf")),
                dict(q=q, window=-1), dict(q=q, window=2 ** 31), dict(q=q, slopes=f[:3]), dict(q=q, slopes=f.half()), dict(q=q, slopes=torch.zeros(8)[::2]),
                dict(q=q, prefix=i[:1]), dict(q=q, prefix=i.long()), dict(q=q, prefix=torch.zeros(4, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            paged_kv.attention(cache, batch, **bad)
    with pytest.raises(ValueError, match="current GPU"):
        paged_kv.attention(cache, batch, q, slopes=f, prefix=i)
    cache, batch = handles(D=96)
    with pytest.raises(ValueError, match="head dim 64 or 128"):
        paged_kv.attention(cache, batch, torch.zeros(3, 4, 96))


def test_entry_points_reject_before_any_launch():
    """Sizes, types and alignments that the entry points return 1 for, the pointers never read."""
    lib = _lib.declare(ctypes.CDLL(_lib.LIB_PATH))
    a = 1 << 20

    def attn(type_=1, window=0, softcap=0.0, q=a, ws=a, scale=0.1, **change):
        d = dict(T=4, H=8, Hkv=2, D=128, B=2, N=4, pitch=4, P=9, S=16, sqt=1024, sqh=128, sot=1024, soh=128, kp=4096, kr=256, kh=128, vp=4096, vr=256, vh=128)
        d.update(change)
        return lib.rda_paged_attn(q, a, a, a, a, a, a, None, None, ws, scale, softcap, window, 0, type_, _lib.long_array(list(d.values())), None)

    for bad in (dict(T=0), dict(H=7), dict(H=0), dict(Hkv=0), dict(D=96), dict(B=0), dict(B=8193), dict(N=0), dict(P=0), dict(S=0), dict(N=1 << 27), dict(sqt=1028),
                dict(soh=132), dict(kr=252), dict(vh=4), dict(q=a + 8), dict(ws=a + 8), dict(type_=3), dict(type_=-1), dict(window=-1), dict(softcap=-1.0),
                dict(softcap=float("nan")), dict(T=1 << 30), dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-39),
                dict(kp=1 << 32), dict(vr=1 << 32)):
        assert attn(**bad) == 1, bad
    assert lib.rda_paged_attn_workspace(4, 2, 8, 2, 128, 1) > 0 and lib.rda_paged_attn_workspace(4, 2, 8, 3, 128, 1) == 0

    def rotate(type_=0, x=a, turns=a, **change):
        d = dict(B=1, L=4, H=8, D=128, R=128, xb=0, xl=1024, xh=128, yb=0, yl=1024, yh=128)
        d.update(change)
        return lib.rda_rotate_positions(x, a, a, 0, turns, 1.0, 0, type_, _lib.long_array(list(d.values())), None)

    for bad in (dict(B=0), dict(L=0), dict(H=0), dict(H=65536), dict(D=120), dict(D=272, R=16), dict(R=0), dict(R=8), dict(R=144), dict(type_=3), dict(x=a + 2), dict(xl=1028),
                dict(yh=4), dict(turns=None)):
        assert rotate(**bad) == 1, bad

    def append(type_=0, cache=0, k=a, **change):
        d = dict(T=4, H=8, Hkv=2, D=128, R=128, B=2, N=4, pitch=4, P=9, S=16, qt=1024, qh=128, kt=256, kh=128, vt=256, vh=128, ot=1024, oh=128, kp=4096, kr=256, ch=128,
                 vp=4096, vr=256, wh=128)
        d.update(change)
        return lib.rda_paged_append(a, k, a, a, a, a, a, a, a, a, 1.0, 0, type_, cache, _lib.long_array(list(d.values())), None)

    for bad in (dict(T=0), dict(Hkv=0), dict(H=-1), dict(H=65536), dict(D=24), dict(R=144), dict(B=0), dict(N=0), dict(P=0), dict(S=0), dict(N=1 << 27), dict(type_=3),
                dict(cache=-1), dict(k=a + 4), dict(kt=252), dict(vp=4), dict(oh=4), dict(qt=4)):
        assert append(**bad) == 1, bad


def test_tile_rule():
    """The tiles that sizes choose, by the workspace of their parts: 16 rows for single tokens and fp32, 32 for short chunks and where tiles of
    128 would be few, else 128."""
    lib = _lib.declare(ctypes.CDLL(_lib.LIB_PATH))

    def rows(T, B, H, Hkv, D, type_):
        size = lib.rda_paged_attn_workspace(T, B, H, Hkv, D, type_)
        return {grid * (32 + 2 * mt * (D + 2) * 4): mt for mt in (16, 32, 128) for grid in (512, 768)}[size]

    assert rows(64, 64, 32, 8, 128, 1) == 16 and rows(1, 1, 64, 4, 64, 0) == 16 and rows(2048, 1, 32, 8, 128, 2) == 16
    assert rows(32 * 5, 32, 32, 8, 128, 1) == 32 and rows(32 * 16, 32, 32, 8, 64, 0) == 32 and rows(32 * 17, 32, 32, 8, 128, 1) == 128
    assert rows(160, 1, 32, 8, 128, 1) == 32 and rows(161, 1, 32, 8, 128, 1) == 128  # 5 and 6 tiles x 8 KV heads
    assert rows(2048, 1, 32, 8, 128, 1) == 128 and rows(1031, 31, 24, 8, 64, 0) == 128


def test_reference_against_torch():
    """The 64-bit forms: causal attention of a chunk over cached keys equals torch's with the same mask, in any pages; a turn keeps lengths
    and depends on differences of positions only; appended pages hold the tokens in order."""
    g = gen(1)
    k, v, q = torch.randn(30, 2, 16, generator=g).double(), torch.randn(30, 2, 16, generator=g).double(), torch.randn(7, 4, 16, generator=g)
    table = torch.tensor([[3, 0, 5, 1]], dtype=torch.int32)
    empty = torch.zeros(6, 8, 2, 16)
    kp, vp, _ = appended(k, v, empty, empty, table, [0, 30], [30], None)
    assert torch.equal(kp[3], k[:8]) and torch.equal(vp[1, :6], v[24:])
    out, off, mine = attended(q, kp, vp, table, [0, 7], [30], window=9)
    j, n = torch.arange(30), torch.arange(23, 30)[:, None]
    mask = (j <= n) & (n - j < 9)
    ref = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1),
                                                           v.repeat_interleave(2, 1).transpose(0, 1), attn_mask=mask).transpose(0, 1)
    assert mine.all() and torch.allclose(out, ref, rtol=1e-12, atol=1e-12) and (off > 0).all()
    r = rotary.Rotary(16, base=50.0, device="cpu")
    a, _ = turned(q, torch.arange(7) + 5, r)
    b, _ = turned(q, torch.arange(7) + 905, r)
    assert torch.allclose(a.norm(dim=-1), q.double().norm(dim=-1), rtol=1e-12)
    assert torch.allclose((a[:-1] * a[1:]).sum(-1), (b[:-1] * b[1:]).sum(-1), rtol=1e-9)
