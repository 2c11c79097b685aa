"""paged_kv's quantized cache on the CPU: refusals, the entry points' own checks, the places that appends give to blocks, and the 64-bit forms."""
import ctypes
import random
import types

import pytest
import torch

from comfyui_rdna2_attention_amd import _lib, paged_kv, rotary
from helpers import gen
from quantized_reference import attended_quantized, check_appended, values


def tensors(pages=4, page=32, heads=2, D=64, block=16):
    return (*(torch.zeros(pages, page, heads, D, dtype=torch.int8) for _ in range(2)), *(torch.zeros(pages, page // block, heads) for _ in range(2)))


def handles(**sizes):
    return paged_kv.QuantizedCache(*tensors(**sizes)), paged_kv.Batch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_cache():
    k, v, ks, vs = tensors()
    cache = paged_kv.QuantizedCache(k, v, ks, vs)
    assert cache.block == 16 and cache.k is k and cache.v_scales is vs
    assert paged_kv.QuantizedCache(k, v, ks[:, :1], vs[:, :1]).block == 32
    paged_kv.QuantizedCache(k.transpose(1, 2).contiguous().transpose(1, 2), v, ks.permute(2, 0, 1).contiguous().permute(1, 2, 0), vs)
    for bad in ((k, v[:3], ks, vs), (k.float(), v.float(), ks, vs), (k, v.half(), ks, vs), (k[0], v[0], ks, vs), (k[..., :24], v[..., :24], ks, vs), (k[:0], v[:0], ks[:0], vs[:0]),
                (k, v, ks.half(), vs.half()), (k, v, ks, vs[:3]), (k, v, ks[:, :0], vs[:, :0]), (k, v, ks[..., :1], vs[..., :1]), (k, v, ks[0], vs[0]),
                (k[:, :24], v[:, :24], ks, vs), (k[:, :24], v[:, :24], ks[:, :1], vs[:, :1]), (k[:, :8], v[:, :8], ks[:, :1], vs[:, :1]),
                (torch.zeros(4, 32, 2, 128, dtype=torch.int8)[..., ::2], v, ks, vs), (torch.zeros(4, 32, 2, 72, dtype=torch.int8)[..., :64], v, ks, vs),
                (torch.zeros(4 * 4096 + 1, dtype=torch.int8)[1:].view(4, 32, 2, 64), v, ks, vs), (k, v, ks.clone().requires_grad_(), vs)):
        with pytest.raises(ValueError):
            paged_kv.QuantizedCache(*bad)
    with pytest.raises(AttributeError):
        cache.k = cache.v
    made = paged_kv.QuantizedCache.empty(5, 48, 3, 80, block=16, device="cpu")
    assert made.k.shape == (5, 48, 3, 80) and made.v_scales.shape == (5, 3, 3) and made.block == 16 and not made.k.any()
    for bad in (dict(page_size=24), dict(page_size=48, block=32), dict(page_size=48, block=48), dict(page_size=0), dict(page_size=64, block=8)):
        with pytest.raises(ValueError):
            paged_kv.QuantizedCache.empty(2, kv_heads=1, dim=64, device="cpu", **bad)


def test_append_refusals():
    cache, batch = handles()
    k, q = torch.zeros(3, 2, 64), torch.zeros(3, 4, 64)
    o, w = q.half(), torch.ones(64)
    norm = rotary.HeadNorm(w, w)
    for bad in (dict(k=k.double(), v=k.double()), dict(k=k, v=k.half()), dict(k=k, v=k[:2]), dict(k=k[:, :1], v=k[:, :1]), dict(k=k[..., :48], v=k[..., :48]),
                dict(k=k, v=k, q=q), dict(k=k, v=k, q=q, q_out=q.clone()), dict(k=k, v=k, q=q.half(), q_out=o), dict(k=k, v=k, q=q[:2], q_out=o[:2]),
                dict(k=k, v=k, q=q, q_out=o[:2]), dict(k=k, v=k, q_out=o), dict(k=k, v=k, q=q[:, :0], q_out=o[:, :0]), dict(k=k, v=k, q=q, q_out=o[:1].expand(3, 4, 64)),
                dict(k=k, v=k, q=q, q_out=torch.zeros(3, 4, 128, dtype=torch.float16)[..., ::2]), dict(k=k, v=k, rotary=rotary.Rotary(80, device="cpu")),
                dict(k=k, v=k, norm=rotary.HeadNorm(torch.ones(48), torch.ones(48)))):
        with pytest.raises(ValueError):
            paged_kv.append(cache, batch, **bad)
    with pytest.raises(ValueError, match="current GPU"):
        paged_kv.append(cache, batch, k, k, q=q, q_out=o, norm=norm)
    with pytest.raises(ValueError, match="gradient"):
        paged_kv.append(cache, batch, k, k, norm=rotary.HeadNorm(w.clone().requires_grad_(), w))
    with pytest.raises(ValueError, match="gradient"):
        paged_kv.append(cache, batch, k.clone().requires_grad_(), k)
    plain = paged_kv.Cache(torch.zeros(4, 8, 2, 64), torch.zeros(4, 8, 2, 64))
    with pytest.raises(ValueError, match="norm_rotate"):
        paged_kv.append(plain, batch, k, k, norm=norm)
    c, v, ks, vs = tensors()
    for one in ((c[:1].expand(4, 32, 2, 64), v, ks, vs), (c, v, ks[..., :1].expand(4, 2, 2), vs)):
        with pytest.raises(ValueError, match="one memory"):
            paged_kv.append(paged_kv.QuantizedCache(*one), batch, k, k)
    many = rotary.MAX_TOKENS + 1
    x = torch.zeros(1, 2, 64, dtype=torch.float16).expand(many, 2, 64)
    with pytest.raises(ValueError, match="at most"):
        paged_kv.append(cache, batch, x, x)
    wide = types.SimpleNamespace(sizes=((1, 2 ** 27), 2 ** 27))
    with pytest.raises(ValueError, match="at most 2147418112 tokens"):
        paged_kv.append(cache, wide, k, k)


def test_read_and_attention_refusals():
    cache, batch = handles()
    plain = paged_kv.Cache(torch.zeros(4, 8, 2, 64), torch.zeros(4, 8, 2, 64))
    with pytest.raises(ValueError, match="QuantizedCache"):
        paged_kv.read(plain, batch, 3)
    for bad in (dict(tokens=-1), dict(tokens=rotary.MAX_TOKENS + 1), dict(tokens=3, dtype=torch.int8), dict(tokens=3, dtype=torch.float64)):
        with pytest.raises(ValueError, match="read takes"):
            paged_kv.read(cache, batch, **bad)
    with pytest.raises(ValueError, match="current GPU"):
        paged_kv.read(cache, batch, 3)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    f, i = torch.zeros(4), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(q=q.float()), dict(q=q.to(torch.int8)), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q[:, :0]), dict(q=q, out=q), dict(q=q, out=q[:2].clone()),
                dict(q=q, out=q.bfloat16()), dict(q=q, out=torch.zeros(3, 4, 128, dtype=torch.float16)[..., ::2]), dict(q=q, softcap=-1.0), dict(q=q, scale=0.0),
                dict(q=q, scale=float("nan")), dict(q=q, window=-1), dict(q=q, window=2 ** 31), dict(q=q, slopes=f[:3]), dict(q=q, slopes=f.half()), dict(q=q, prefix=i[:1]),
                dict(q=q, prefix=i.long())):
        with pytest.raises(ValueError):
            paged_kv.attention(cache, batch, **bad)
    with pytest.raises(ValueError, match="current GPU"):
        paged_kv.attention(cache, batch, q, slopes=f, prefix=i)
    with pytest.raises(ValueError, match="gradient"):
        paged_kv.attention(cache, batch, q.clone().requires_grad_())
    cache, batch = handles(D=96)
    with pytest.raises(ValueError, match="head dim 64 or 128"):
        paged_kv.attention(cache, batch, torch.zeros(3, 4, 96, dtype=torch.float16))


def test_entry_points_reject_before_any_launch():
    """Sizes, types and alignments that the entry points return 1 for, the pointers never read."""
    lib = _lib.declare(ctypes.CDLL(_lib.LIB_PATH))
    a = 1 << 20
    cache = dict(N=4, pitch=4, P=9, S=32, block=16)
    codes = dict(kp=8192, kr=256, kh=128, vp=8192, vr=256, vh=128, ksp=4, ksb=2, ksh=1, vsp=4, vsb=2, vsh=1)

    def append(type_=0, q_type=0, weight=0, k=a, codes_at=a, qw=None, kw=None, **change):
        d = {**dict(T=4, H=8, Hkv=2, D=128, R=128, B=2), **cache, **dict(qt=1024, qh=128, kt=256, kn=128, vt=256, vn=128, ot=1024, oh=128), **codes}
        assert set(change) <= set(d)
        return lib.rda_paged_append_i8(a, k, a, a, codes_at, a, a, a, a, a, a, a, 1.0, 0, qw, kw, weight, 0.0, type_, q_type, _lib.long_array(list({**d, **change}.values())), None)

    for bad in (dict(T=0), dict(T=rotary.MAX_TOKENS + 1), dict(Hkv=0), dict(H=-1), dict(H=65536), dict(D=24), dict(D=272), dict(R=144), dict(B=0), dict(B=8193), dict(N=0), dict(P=0),
                dict(P=1 << 31), dict(S=0), dict(S=24), dict(block=8), dict(block=128), dict(S=48, block=32), dict(N=1 << 26), dict(type_=3), dict(q_type=2), dict(q_type=-1),
                dict(weight=3), dict(k=a + 4), dict(codes_at=a + 8), dict(kt=252), dict(vp=8), dict(kr=264), dict(oh=4), dict(qt=4), dict(qw=a), dict(kw=a),
                dict(qw=a + 4, kw=a)):
        assert append(**bad) == 1, bad

    def read(type_=1, out=a, **change):
        d = {**dict(T=4, Hkv=2, D=128, B=2), **cache, **codes}
        assert set(change) <= set(d)
        return lib.rda_paged_read_i8(a, a, a, a, a, a, a, out, a, type_, _lib.long_array(list({**d, **change}.values())), None)

    for bad in (dict(T=0), dict(Hkv=0), dict(D=24), dict(D=272), dict(B=0), dict(B=8193), dict(N=0), dict(P=0), dict(S=24), dict(block=8), dict(type_=3), dict(out=a + 8), dict(vh=8)):
        assert read(**bad) == 1, bad

    def attn(type_=1, window=0, softcap=0.0, q=a, ws=a, scale=0.1, **change):
        d = {**dict(T=4, H=8, Hkv=2, D=128, B=2), **cache, **dict(sqt=1024, sqh=128, sot=1024, soh=128), **codes}
        assert set(change) <= set(d)
        return lib.rda_paged_attn_i8(q, a, a, a, a, a, a, a, a, None, None, ws, scale, softcap, window, 0, type_, _lib.long_array(list({**d, **change}.values())), None)

    for bad in (dict(T=0), dict(H=7), dict(H=0), dict(Hkv=0), dict(D=96), dict(B=0), dict(B=8193), dict(N=0), dict(P=0), dict(S=0), dict(S=40), dict(block=48), dict(N=1 << 26),
                dict(sqt=1028), dict(soh=132), dict(kr=248), dict(vh=8), dict(q=a + 8), dict(ws=a + 8), dict(type_=2), dict(type_=-1), dict(window=-1), dict(softcap=-1.0),
                dict(softcap=float("nan")), dict(T=1 << 30), dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e-39), dict(kp=1 << 32), dict(kr=1 << 28), dict(vr=1 << 28), dict(ksb=1 << 32), dict(vsp=-4)):
        assert attn(**bad) == 1, bad
    assert lib.rda_paged_attn_i8_workspace(4, 2, 8, 2, 128, 1) > 0 and lib.rda_paged_attn_i8_workspace(4, 2, 8, 2, 128, 2) == 0


def test_every_block_has_a_slot():
    """The slots that an append launches: sequence b's begin at starts[b] / block + 2 b and reach the next one's, and each block that its tokens touch, at any
    position, has one of them; a slot's sequence is the last that begins at or below it."""
    rng = random.Random(3)
    for _ in range(3000):
        block, B = rng.choice([16, 32, 64]), rng.randint(1, 9)
        new = [rng.choice([0, 1, 1, 2, block - 1, block, block + 1, rng.randint(0, 5 * block)]) for _ in range(B)]
        starts = [rng.choice([0, 0, rng.randint(0, 40)])]
        for n in new:
            starts.append(starts[-1] + n)
        T = starts[-1] + rng.choice([0, rng.randint(0, 40)])
        slots = T // block + 2 * B
        base = [s // block + 2 * b for b, s in enumerate(starts)]
        assert base[-1] <= slots
        for b, n in enumerate(new):
            p0 = rng.randint(-70, 200)
            if n:
                touched = (p0 + n - 1) // block - p0 // block + 1
                assert base[b] + touched <= base[b + 1]
        for slot in range(slots):
            b = sum(x <= slot for x in base[1:])  # what the search counts
            assert b == B or base[b] <= slot < base[b + 1] or slot < base[0]


def test_reference():
    """The forms that the GPU tests compare with, on a cache made with torch's own rounding."""
    g = gen(2)
    x = torch.randn(40, 2, 64, generator=g).double()
    codes, scales = torch.zeros(4, 32, 2, 64, dtype=torch.int8), torch.zeros(4, 2, 2)
    table, starts, lengths = torch.tensor([[2, 0, 3]], dtype=torch.int32), torch.tensor([0, 40]), torch.tensor([40])
    after, after_scales = codes.clone(), scales.clone()
    for i in range(0, 40, 16):
        rows = x[i:i + 16]
        s = (rows.abs().amax((0, 2)) / 127).float()
        page = int(table[0, i // 32])
        after_scales[page, i % 32 // 16] = s
        after[page, i % 32:i % 32 + len(rows)] = torch.round(rows / s.double()[:, None]).to(torch.int8)
    check_appended(after, after_scales, x, torch.zeros_like(x), codes, scales, table, starts, lengths, 16)
    for change in ("code", "scale", "elsewhere"):
        c, s = after.clone(), after_scales.clone()
        if change == "code":
            c[2, 3, 1, 5] += 1 if c[2, 3, 1, 5] < 100 else -1
        elif change == "scale":
            s[0, 0, 1] *= 1.001
        else:
            c[1, 0, 0, 0] = 1
        with pytest.raises(AssertionError):
            check_appended(c, s, x, torch.zeros_like(x), codes, scales, table, starts, lengths, 16)
    back = values(after, after_scales)[table[0].long()].reshape(96, 2, 64)[:40]
    assert (back - x).abs().max() <= 0.5 * after_scales.max() * 1.0001
    q = torch.randn(3, 4, 64, generator=g).half()
    out, off, mine = attended_quantized(q, after, after, after_scales, after_scales, table, torch.tensor([0, 3]), torch.tensor([40]))
    w = torch.softmax((q[2, 3].double() @ back[:, 1].T) / 8, -1)
    assert mine.all() and torch.allclose(out[2, 3], w @ back[:, 1], rtol=1e-12) and (off > 0).all()
