"""paged_kv.attention with caps far above the scores, in every tile and type: a cap that no score comes near changes nothing."""
import pytest
import torch

from comfyui_rdna2_attention_amd import paged_kv
from helpers import gen
from paged_reference import attended
from test_gpu_paged import TYPES, batch_of, check, tile_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap,scale", [(1500.0, 0.3), (1500.0, 40.0), (1e4, 0.3), (1e6, 0.3), (1e8, 0.3), (1e20, 0.3)])
@pytest.mark.parametrize("type_,heads,kv,D,tiles,new", [("bf16", 24, 24, 128, 128, 130), ("fp16", 48, 24, 64, 128, 130), ("fp16", 2, 2, 128, 32, 40),
                                                       ("bf16", 2, 2, 64, 32, 40), ("bf16", 4, 2, 128, 16, 1), ("fp32", 2, 2, 64, 16, 40)])
def test_high_caps(dev, type_, heads, kv, D, tiles, new, softcap, scale):
    """Capped scores are off by at most 2e-6 of themselves. In roundings of 2^-24: the scale's six, the series' four and 1e-8, the cap's
    four, 8e-7 together; past the series (|y| >= 1/4, |tanh y| > 0.24) 2 / (1 + 2^e) <= 1.25 at y = -1/4 has three in 1 + 2^e's sum and its
    reciprocal, the exponential adds half of 2^-23 and the last sum one: 3e-7 of the cap, 1.3e-6 of the score, with the scale's and the cap's 1.9e-6;
    towards y = -1 / +1 the same parts are less of a score near the cap. Other errors are those of attention without a cap: its bound is
    spread x 2 (delta + u + keys 2^-24) with delta >= 2^-21, so that x (1 + 2e-6 max |score| / (2^-21 + u + keys 2^-24)) of it holds with the cap."""
    g = gen(int(softcap) % 1000 + D + new)
    t, length = TYPES[type_], 390
    table, starts, lengths, pages = batch_of([(new, length)], 16, g)
    assert tile_rows(new, 1, heads, kv, D, type_) == tiles
    k, v = (torch.randn(pages, 16, kv, D, generator=g).to(t) for _ in range(2))
    q = torch.randn(new, heads, D, generator=g).to(t)
    most = scale * float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max())
    u = 0.0 if t is torch.float32 else torch.finfo(t).eps / 2
    for slopes in (None, torch.rand(heads, generator=g) * 0.1):
        print(f"cap {softcap} {type_} heads={heads}/{kv} D={D} new={new} {'biased' if slopes is not None else ''}", flush=True)
        got = paged_kv.attention(paged_kv.Cache(k.to(dev), v.to(dev)), paged_kv.Batch(table.to(dev), starts.to(dev), lengths.to(dev)), q.to(dev),
                                 scale=scale, softcap=softcap, slopes=None if slopes is None else slopes.to(dev))
        ref, _, _ = attended(q, k, v, table, starts, lengths, scale=scale, softcap=softcap, slopes=slopes)
        _, off, _ = attended(q, k, v, table, starts, lengths, scale=scale, slopes=slopes)
        check(got, ref, off * (1 + 2e-6 * most / (2.0 ** -21 + u + length * 2.0 ** -24)), t)
