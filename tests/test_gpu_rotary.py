"""rotary.rotate on the GPU against 64-bit angles and turns: layouts, parts of heads, types, strides, far positions, the inverse."""
import pytest
import torch

from comfyui_rdna2_attention_amd import rotary
from helpers import gen
from paged_reference import rounding, turned

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def check(got, x, positions, rot, inverse=False):
    ref, off = turned(x, positions, rot, inverse)
    got = got.cpu().double()
    bound = off + rounding(ref.abs() + off, x.dtype)
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {ref[bad][0]}"


@pytest.mark.parametrize("tokens,heads,D,R", [(1, 1, 16, 16), (1, 32, 128, 128), (5, 3, 64, 32), (130, 7, 128, 64), (33, 40, 128, 128), (9, 5, 80, 48),
                                              (4, 33, 256, 256), (3, 2, 240, 16), (70, 66, 96, 96), (2, 300, 32, 32)])
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("type_", TYPES)
def test_rotate(dev, type_, layout, tokens, heads, D, R):
    g = gen(tokens * heads + D)
    x = torch.randn(tokens, heads, D, generator=g).to(TYPES[type_])
    positions = torch.randint(0, 5000, (tokens,), generator=g, dtype=torch.int32)
    rot = rotary.Rotary(R, layout=layout, device=dev)
    print(f"rotate {type_} {layout} {tokens} x {heads} x {D} ({R})", flush=True)
    got = rotary.rotate(x.to(dev), positions.to(dev), rot)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    check(got, x, positions, rot)
    if R < D:
        assert torch.equal(got.cpu()[..., R:], x[..., R:])


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "bands", "yarn"])
def test_far_positions_and_scalings(dev, scaling):
    """Positions to 10^6 (and past 2^31, in 64 bits, and negative ones), where a 32-bit angle would be off by a whole 0.06 radians."""
    g = gen(7)
    options = dict(factor=8.0, original=4096) if scaling in ("bands", "yarn") else dict(factor=8.0) if scaling else {}
    rot = rotary.Rotary(128, base=5e5, scaling=scaling, device=dev, **options)
    x = torch.randn(64, 2, 128, generator=g)
    positions = torch.randint(-10 ** 6, 10 ** 6, (64,), generator=g)
    positions[:3] = torch.tensor([2 ** 31 + 5, 999999, 0])
    got = rotary.rotate(x.to(dev), positions.to(dev), rot)
    check(got, x, positions, rot)


def test_layouts_of_memory(dev):
    """Batches, heads before tokens (a transposed view), rows of a fused projection, unaligned views, an out with strides, in place."""
    g = gen(8)
    rot = rotary.Rotary(64, device=dev)
    positions = torch.randint(0, 300, (3, 11), generator=g, dtype=torch.int32)
    x = torch.randn(3, 5, 11, 64, generator=g).half()
    flat = lambda t: t.reshape(33, 5, 64)  # noqa: E731
    got = rotary.rotate(x.to(dev).transpose(1, 2), positions.to(dev), rot)
    assert got.shape == (3, 11, 5, 64)
    check(flat(got), flat(x.transpose(1, 2)), positions.reshape(-1), rot)
    fused = torch.randn(33, 9 * 64, generator=g).half()
    view = fused.view(33, 9, 64)[:, 2:7]
    check(rotary.rotate(fused.to(dev).view(33, 9, 64)[:, 2:7], positions.reshape(-1).to(dev), rot), view, positions.reshape(-1), rot)
    odd = torch.randn(33 * 5 * 64 + 3, generator=g).half()
    check(rotary.rotate(odd.to(dev)[3:].view(33, 5, 64), positions.reshape(-1).to(dev), rot), odd[3:].view(33, 5, 64), positions.reshape(-1), rot)
    whole = torch.zeros(33, 8, 64, dtype=torch.float16, device=dev)
    got = rotary.rotate(view.to(dev), positions.reshape(-1).to(dev), rot, out=whole[:, 1:6])
    assert got.data_ptr() == whole[:, 1:6].data_ptr() and not whole[:, 0].any() and not whole[:, 6:].any()
    check(got, view, positions.reshape(-1), rot)
    mine = view.to(dev).contiguous()
    rotary.rotate(mine, positions.reshape(-1).to(dev), rot, out=mine)
    check(mine, view, positions.reshape(-1), rot)
    assert rotary.rotate(mine[:0], positions.reshape(-1)[:0].to(dev), rot).shape == (0, 5, 64)


@pytest.mark.parametrize("layout", rotary.LAYOUTS)
def test_inverse_is_the_gradient(dev, layout):
    """inverse=True is the gradient of the turn (yarn's factor in it), against the formula's and against differences."""
    g = gen(9)
    rot = rotary.Rotary(32, layout=layout, scaling="yarn", factor=4.0, original=64, device=dev)
    assert rot.factor > 1.1
    x, grad = torch.randn(6, 2, 48, generator=g), torch.randn(6, 2, 48, generator=g)
    positions = torch.randint(0, 900, (6,), generator=g)
    got = rotary.rotate(grad.to(dev), positions.to(dev), rot, inverse=True)
    check(got, grad, positions, rot, inverse=True)
    # The turn is linear, so a difference over any step is exact but for rounding: f(x + d) - f(x) against d . grad.
    step = torch.randn(6, 2, 48, generator=g)
    f = lambda t: (rotary.rotate(t.to(dev), positions.to(dev), rot).double() * grad.to(dev).double()).sum()  # noqa: E731
    change, slope = float(f(x + step) - f(x)), float((got.double() * step.to(dev).double()).sum())
    size = float((x.abs() + step.abs()).sum() * grad.abs().max()) * rot.factor
    assert abs(change - slope) <= 16 * 2.0 ** -24 * size
    plain = rotary.Rotary(32, layout=layout, device=dev)
    back = rotary.rotate(rotary.rotate(x.to(dev), positions.to(dev), plain), positions.to(dev), plain, inverse=True).cpu()
    assert (back - x).abs().max() <= 32 * 2.0 ** -24 * x.abs().max()


def test_side_stream_and_graph(dev):
    x = torch.randn(64, 8, 128, generator=gen(10)).bfloat16().to(dev)
    positions = torch.arange(64, dtype=torch.int32, device=dev)
    rot = rotary.Rotary(128, device=dev)
    want = rotary.rotate(x, positions, rot)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary.rotate(x, positions, rot)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rotary.rotate(x, positions, rot, out=out)
    for i in range(3):
        positions += 100
        graph.replay()
        assert torch.equal(out, rotary.rotate(x, positions, rot)), i
