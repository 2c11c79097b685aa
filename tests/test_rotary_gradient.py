"""rotary.rotate where gradients are recorded: on the CPU with a stand-in for the launch that turns in 64 bits, and on the GPU."""
import ctypes
import types

import numpy as np
import pytest
import torch

from comfyui_rdna2_attention_amd import _lib, rotary
from helpers import gen
from paged_reference import rounding, turned


@pytest.fixture
def launch(monkeypatch):
    """rotate_positions for contiguous fp32 x and y of one batch: paged_reference's turn, rounded."""
    def rotate_positions(x, y, positions, wide, turns, factor, flags, type_, dims, stream):
        _, L, H, D, R = list(dims)[:5]
        array = lambda at, c, *shape: torch.from_numpy(np.ctypeslib.as_array(ctypes.cast(at, ctypes.POINTER(c)), shape))  # noqa: E731
        assert wide and type_ == 2
        rot = types.SimpleNamespace(dim=R, turns=array(turns, ctypes.c_double, R // 2).clone(), factor=factor, layout=rotary.LAYOUTS[flags & 1])
        array(y, ctypes.c_float, L, H, D).copy_(turned(array(x, ctypes.c_float, L, H, D).clone(), array(positions, ctypes.c_long, L), rot, bool(flags & 2))[0])
        return 0

    monkeypatch.setattr(rotary, "same_device", lambda *a: None)
    monkeypatch.setattr(rotary, "get_kernels", lambda: types.SimpleNamespace(rotate_positions=rotate_positions))
    monkeypatch.setattr(_lib, "raw_stream", lambda: 0)


def plain(x, positions, rot, inverse=False):
    """The turn in elementary torch operations, for its recorded gradient: x's type throughout."""
    half = rot.dim // 2
    angle = positions.double()[:, None] * rot.turns * (2 * np.pi) * (-1 if inverse else 1)
    c, s = ((f(angle) * rot.factor)[:, None].to(x.dtype) for f in (torch.cos, torch.sin))
    i = torch.arange(half)
    at, to = (2 * i, 2 * i + 1) if rot.layout == "interleaved" else (i, i + half)
    a, b = x[..., at], x[..., to]
    return x.index_copy(-1, at, a * c - b * s).index_copy(-1, to, a * s + b * c)


@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("inverse", [False, True])
def test_gradient(launch, layout, inverse):
    """The gradient that arrives at x is the formula's, and so is the gradient's gradient."""
    g = gen(3)
    rot = rotary.Rotary(32, layout=layout, scaling="yarn", factor=4.0, original=64, device="cpu")
    x, weight, again = (torch.randn(5, 2, 48, generator=g) for _ in range(3))
    positions = torch.randint(0, 900, (5,), generator=g)
    results = []
    for f in (lambda t: rotary.rotate(t, positions, rot, inverse=inverse), lambda t: plain(t, positions, rot, inverse)):
        leaf, w = x.clone().requires_grad_(), weight.clone().requires_grad_()
        y = f(leaf)
        grad, = torch.autograd.grad(y, leaf, w, create_graph=True)
        second, = torch.autograd.grad(grad, w, again)
        results.append((y.detach(), grad.detach(), second))
    for a, b in zip(*results):
        # Sums of two products, each factor rounded, of values below 4 with a factor below 1.14: eight roundings at most between the two.
        assert (a - b).abs().max() <= 8 * 2.0 ** -24 * 2 * 4.5 * 1.14
    assert results[0][0].norm() > 1


def test_gradient_of_expanded_and_strided(launch):
    """A broadcast input's gradient is summed, and a gradient that comes expanded or in another order is read as it is."""
    rot, positions = rotary.Rotary(16, device="cpu"), torch.arange(6)
    x = torch.randn(6, 1, 16, generator=gen(4)).requires_grad_()
    rotary.rotate(x.expand(6, 3, 16), positions, rot).sum().backward()
    ones, _ = turned(torch.ones(6, 1, 16), positions, rot, inverse=True)
    assert torch.allclose(x.grad.double(), 3 * ones, rtol=0, atol=16 * 2.0 ** -24 * 6)
    x.grad = None
    rotary.rotate(x, positions, rot).transpose(0, 2).contiguous().sum().backward()
    assert torch.allclose(x.grad.double(), ones, rtol=0, atol=16 * 2.0 ** -24 * 2)


def test_what_is_not_recorded(launch):
    """Without recording, or where nothing requires a gradient, a plain tensor; an out takes no gradient; positions that changed since
    are not turned back by."""
    rot, positions = rotary.Rotary(16, device="cpu"), torch.arange(6)
    x = torch.randn(6, 2, 16, generator=gen(5))
    assert not rotary.rotate(x, positions, rot).requires_grad
    leaf, out = x.clone().requires_grad_(), torch.empty_like(x)
    with torch.no_grad():
        assert not rotary.rotate(leaf, positions, rot).requires_grad
        rotary.rotate(leaf, positions, rot, out=out)
    with pytest.raises(ValueError, match="gradient"):
        rotary.rotate(leaf, positions, rot, out=out)
    with pytest.raises(ValueError, match="gradient"):
        rotary.rotate(x, positions, rot, out=leaf)
    y = rotary.rotate(leaf, positions, rot).sum()
    positions += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="takes"):
        rotary.rotate(leaf, positions[:3], rot)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("type_", [torch.float16, torch.bfloat16, torch.float32])
def test_gradient_on_the_gpu(dev, type_, layout):
    """Types, on a stream of their own, of heads first and of one token; against the 64-bit turn back."""
    g = gen(6)
    rot = rotary.Rotary(64, layout=layout, scaling="yarn", factor=4.0, original=64, device=dev)
    for tokens, heads in ((1, 3), (37, 5)):
        x, weight = (torch.randn(tokens, heads, 80, generator=g).to(type_) for _ in range(2))
        positions = torch.randint(0, 10 ** 6, (tokens,), generator=g)
        print(f"gradient {type_} {layout} {tokens} x {heads}", flush=True)
        leaf = x.to(dev).requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = rotary.rotate(leaf.transpose(0, 1).contiguous().transpose(0, 1), positions.to(dev), rot)
            y.backward(weight.to(dev))
        side.synchronize()
        for got, src, inverse in ((y.detach(), x, False), (leaf.grad, weight, True)):
            ref, off = turned(src, positions, rot, inverse)
            assert ((got.cpu().double() - ref).abs() <= off + rounding(ref.abs() + off, type_)).all()
        torch.cuda.current_stream().wait_stream(side)


@pytest.mark.gpu
def test_captured_gradient(dev):
    """A turn and its gradient captured together, replayed while the values, the gradient and the positions change: the eager bits each time."""
    g = gen(7)
    rot = rotary.Rotary(64, device=dev)
    x = torch.randn(9, 4, 64, generator=g).bfloat16().to(dev).requires_grad_()
    weight, positions = torch.randn(9, 4, 64, generator=g).bfloat16().to(dev), torch.arange(9, dtype=torch.int32, device=dev)

    def step():
        y = rotary.rotate(x, positions, rot)
        return y.detach(), torch.autograd.grad(y, x, weight)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grad = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(9, 4, 64, generator=g).bfloat16())
            weight.copy_(torch.randn(9, 4, 64, generator=g).bfloat16())
            positions += 1000
        graph.replay()
        want = step()
        assert torch.equal(y, want[0]) and torch.equal(grad, want[1]), i
