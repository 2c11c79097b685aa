"""Attention where lengths pass what the table holds, with windows and prefixes: only the table's keys are there, positions and windows follow the length. Against 64 bits."""
import pytest
import torch

from comfyui_rdna2_attention_amd import paged_kv
from helpers import gen
from paged_reference import attended
from quantized_reference import attended_quantized
from test_gpu_paged import check
from test_gpu_quantized_cache import TYPES, codes_of, on

pytestmark = pytest.mark.gpu

PAGE, ENTRIES = 32, 32  # a table of 1024 keys


def batch_over(seqs, g):
    """A table of ENTRIES pages each, in random order, for sequences (new, length) of any lengths."""
    pages = len(seqs) * ENTRIES + 1
    table = torch.randperm(pages, generator=g)[:len(seqs) * ENTRIES].view(-1, ENTRIES).to(torch.int32)
    starts = torch.tensor([0] + [new for new, _ in seqs], dtype=torch.int32).cumsum(0, dtype=torch.int32)
    return table, starts, torch.tensor([length for _, length in seqs], dtype=torch.int32), pages


def attend(dev, type_, D, heads, kv, block, seqs, seed, **options):
    g = gen(seed)
    t = TYPES[type_]
    table, starts, lengths, pages = batch_over(seqs, g)
    k, v, ks, vs = codes_of(pages, PAGE, kv, D, block, g)
    q = torch.randn(int(starts[-1]), heads, D, generator=g).to(t)
    q = torch.where(q.abs() < 2.0 ** -10, 0, q)  # as fp16 holds it
    print(f"attention {type_} D={D} heads={heads}/{kv} block={block} seqs={seqs} {options}", flush=True)
    got = paged_kv.attention(paged_kv.QuantizedCache(*on(dev, k, v, ks, vs)), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev),
                             **{n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in options.items()})
    ref, off, _ = attended_quantized(q, k, v, ks, vs, table, starts, lengths, **options)
    check(got, ref, off, t)


# Windows that begin ahead of the table's end, at it, a key to either side, and far behind; prefixes of a few keys, of several units, up to the end.
@pytest.mark.parametrize("new,kv", [(1, 2), (5, 2), (40, 2), (150, 24)])
@pytest.mark.parametrize("window,prefix", [(512, 300), (100, 33), (17, 1000), (1, 1024), (600, 257)])
def test_prefix_and_window(dev, new, kv, window, prefix):
    prefixes = torch.tensor([prefix, prefix, prefix, 0, prefix], dtype=torch.int32)
    seqs = [(new, 5000), (new, 1024 + window - 1 + new // 2), (new, 1024 + window // 2 + new), (new, 3000), (new, 900)]
    attend(dev, "fp16", 64, 2 * kv, kv, 32, seqs, seed=31, window=window, prefix=prefixes)
    edges = [(new, 1024 + window - 1), (new, 1024 + window), (new, 1024 + window + new)]
    attend(dev, "bf16", 128, kv, kv, 16, edges, seed=32, window=window, prefix=prefixes[:3])
    attend(dev, "bf16", 64, kv, kv, 16, seqs[:3], seed=33, window=window, prefix=prefixes[:3], softcap=20.0)


@pytest.mark.parametrize("new,kv", [(1, 2), (5, 2), (40, 2), (150, 24)])
@pytest.mark.parametrize("window,prefix", [(17, 67), (1, 1000), (2 ** 31 - 2000, 67), (2 ** 31 - 1, 600)])
def test_last_positions(dev, new, kv, window, prefix):
    """Positions up to 2^31 - 2: a window that begins behind the table, ahead of its end by less than a tile, or far ahead of the first key. Caches in 8, 16 and 32 bits."""
    seqs = [(new, 2 ** 31 - 1), (new, 2 ** 31 - 40), (new, 2 ** 31 - 1200)]
    prefixes = torch.tensor([prefix, prefix + 5, 0], dtype=torch.int32)
    attend(dev, "fp16", 64, 2 * kv, kv, 32, seqs, seed=41, window=window, prefix=prefixes)
    attend(dev, "bf16", 128, kv, kv, 16, seqs, seed=42, window=window, prefix=prefixes)
    for type_, D in (("fp16", 128), ("bf16", 64), ("fp32", 64)):
        g = gen(43)
        table, starts, lengths, pages = batch_over(seqs, g)
        k, v = (torch.randn(pages, PAGE, kv, D, generator=g).to(TYPES[type_]) for _ in range(2))
        q = torch.randn(int(starts[-1]), kv, D, generator=g).to(TYPES[type_])
        print(f"attention over {type_} D={D} kv={kv} new={new} window={window} prefix={prefix}", flush=True)
        got = paged_kv.attention(paged_kv.Cache(*on(dev, k, v)), paged_kv.Batch(*on(dev, table, starts, lengths)), q.to(dev), window=window, prefix=prefixes.to(dev))
        ref, off, _ = attended(q, k, v, table, starts, lengths, window=window, prefix=prefixes)
        check(got, ref, off, TYPES[type_])
