"""paged_kv.append where starts fall below zero and lengths are large: a row's position then passes 2^31, and belongs to no page."""
import pytest
import torch

from comfyui_rdna2_attention_amd import paged_kv
from helpers import gen


def div_by(n, d):
    """The kernels' division by a launch-time constant, of n in 32 bits (csrc/paged.h)."""
    s = 0
    while 1 << s < d:
        s += 1
    m = (((1 << s) - d) << 32) // d + 1
    n &= 2 ** 32 - 1
    return ((n * m >> 32) + n & 2 ** 32 - 1) >> s


def test_positions_past_31_bits_divide_to_pages_that_exist():
    """Why such positions are left out: the division is of 31 bits, and what it makes of more may be a table's entry, with a row far outside its page."""
    for d in (1, 5, 16, 24, 100):
        for n in (0, 1, d - 1, d, 12345, 2 ** 31 - 1):
            assert div_by(n, d) == n // d
    entry = div_by(2 ** 32 - 3, 24)
    row = -3 - entry * 24  # of the position as 32 bits with a sign
    assert entry < 2 ** 28 and not 0 <= row < 24


@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 24])
def test_append(dev, page):
    g = gen(page)
    guard = torch.full((3, 9, page, 1, 64), 7.0, device=dev)
    k_pages, v_pages = guard[1].clone(), guard[1]  # v's pages lie between guards
    table = torch.arange(9, dtype=torch.int32, device=dev).view(3, 3)
    k, v = (torch.randn(100, 1, 64, generator=g).to(dev) for _ in range(2))
    for starts in ([0, 100, 2, -2000000000], [0, 100, 2, -2 ** 31], [5, 3, 3, -2 ** 31], [0, 100, 2, -100]):
        for length in (2 ** 31 - 1, 2 ** 31 - 50, 2000000000):
            print(starts, length, flush=True)
            batch = paged_kv.Batch(table, torch.tensor(starts, dtype=torch.int32, device=dev), torch.full((3,), length, dtype=torch.int32, device=dev))
            paged_kv.append(paged_kv.Cache(k_pages, v_pages), batch, k, v)
            torch.cuda.synchronize()
    assert (guard == 7).all() and (k_pages == 7).all()
