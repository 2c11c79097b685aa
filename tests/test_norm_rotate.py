"""rotary.norm_rotate: the formula of its gradients against differences, refusals on the CPU; values and gradients on the GPU against 64 bits."""
import ctypes

import pytest
import torch

from comfyui_rdna2_attention_amd import _lib, paged_kv, rotary
from helpers import gen
from paged_reference import rounding
from quantized_reference import norm_turned, norm_turned_back

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def close(got, ref, off, dtype, what=""):
    got, bound = got.detach().cpu().double(), off + rounding(ref.abs() + off, dtype)
    bad = ~((got - ref).abs() <= bound)
    assert got.shape == ref.shape and not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {ref[bad][0]}, "
                                                      f"worst {float(((got - ref).abs() / bound)[bad].nan_to_num(9e9).max()):.2f} of the bound")


@pytest.mark.parametrize("layout", rotary.LAYOUTS)
def test_formula_against_differences(layout):
    """The 64-bit gradients against central differences of the 64-bit values, in a random direction of x and of w."""
    g = gen(1)
    rot = rotary.Rotary(16, layout=layout, scaling="yarn", factor=4.0, original=64, device="cpu")
    x, grad, dx = (torch.randn(3, 2, 32, generator=g).double() for _ in range(3))
    w, dw = torch.randn(32, generator=g).double(), torch.randn(32, generator=g).double()
    positions = torch.tensor([0, 7, 500])
    (gx, _), (gw, _) = norm_turned_back(x, w, grad, positions, rot, 1e-3)
    f = lambda a, b: (norm_turned(a, b, positions, rot, 1e-3)[0] * grad).sum()  # noqa: E731
    h = 1e-5
    assert float((f(x + h * dx, w) - f(x - h * dx, w)) / (2 * h)) == pytest.approx(float((gx * dx).sum()), rel=1e-8, abs=1e-8)
    assert float((f(x, w + h * dw) - f(x, w - h * dw)) / (2 * h)) == pytest.approx(float((gw * dw).sum()), rel=1e-8, abs=1e-8)


def test_head_norm_refusals():
    w = torch.ones(64)
    norm = rotary.HeadNorm(w, w.clone(), eps=1e-5)
    assert norm.q is w and norm.eps == 1e-5
    for bad in ((w, w[:48]), (w, w.half()), (w.double(), w.double()), (w.view(2, 32),) * 2, (w[:0],) * 2, (torch.ones(24),) * 2, (torch.ones(128)[::2],) * 2,
                (torch.ones(65)[1:],) * 2):
        with pytest.raises(ValueError):
            rotary.HeadNorm(*bad)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            rotary.HeadNorm(w, w, eps=eps)


def test_refusals():
    norm, rot, n = rotary.HeadNorm(torch.ones(64), torch.ones(64)), rotary.Rotary(32, device="cpu"), torch.zeros(4, dtype=torch.int32)
    q, k = torch.zeros(4, 3, 64), torch.zeros(4, 2, 64)
    for bad in ((q.double(), k.double(), n), (q, k.half(), n), (q[..., :48], k, n), (q, k[..., :48], n), (q[0], k[0], n), (q, k[:3], n), (q, k, n[:3]), (q, k, n.float()),
                (q[:, :0], k, n), (q, k[:, :0], n), (q.view(2, 2, 3, 64), k, n)):
        with pytest.raises(ValueError, match="takes"):
            rotary.norm_rotate(*bad, rot, norm)
    with pytest.raises(ValueError, match="from 80"):
        rotary.norm_rotate(q, k, n, rotary.Rotary(80, device="cpu"), norm)
    with pytest.raises(ValueError, match="current GPU"):
        rotary.norm_rotate(q, k, n, rot, norm)
    many = rotary.MAX_TOKENS + 1
    x, w = torch.zeros(1, 1, 16).expand(many, 1, 16), torch.ones(16)
    with pytest.raises(ValueError, match="at most"):
        rotary.norm_rotate(x, x, torch.zeros(1, dtype=torch.int32).expand(many), rotary.Rotary(16, device="cpu"), rotary.HeadNorm(w, w))


def test_replaced_weights():
    """Weights whose data is replaced after the norm was made: by values that the kernels could not address."""
    rot, n = rotary.Rotary(32, device="cpu"), torch.zeros(4, dtype=torch.int32)
    q, k = torch.zeros(4, 3, 64), torch.zeros(4, 2, 64)
    cache, batch = paged_kv.QuantizedCache.empty(2, 32, 2, 64, device="cpu"), paged_kv.Batch(n[:1].view(1, 1), torch.tensor([0, 4], dtype=torch.int32), n[:1] + 4)
    for which in (0, 1):
        for data, match in ((torch.ones(65)[1:], "16-byte"), (torch.ones(128)[::2], "contiguous"), (torch.ones(64).half(), "one type"), (torch.ones(48), "takes"), (torch.ones(64), "current GPU")):
            weights = torch.ones(64), torch.ones(64)
            norm = rotary.HeadNorm(*weights)
            weights[which].data = data
            with pytest.raises(ValueError, match=match):
                rotary.norm_rotate(q, k, n, rot, norm)
            with pytest.raises(ValueError, match=match):
                paged_kv.append(cache, batch, k, k, norm=norm)


def test_inputs_replaced_before_the_gradient():
    rot, n = rotary.Rotary(32, device="cpu"), torch.zeros(4, dtype=torch.int32)
    q, k, w = torch.zeros(4, 3, 64), torch.zeros(4, 2, 64), torch.ones(64)
    for data in (torch.ones(48), torch.ones(128)[::2], torch.ones(64).half()):
        for weights in ((data, w), (w, data)):
            with pytest.raises(ValueError, match="replaced"):
                rotary._norm_rotate_back(q, k, q, k, n, rot, *weights, 1e-6)
    for bad in ((q[:3], k, q, k, n), (q, k[:, :1], q, k, n), (q, k, q, k, n[:3]), (q, k.half(), q, k, n)):
        with pytest.raises(ValueError, match="replaced"):
            rotary._norm_rotate_back(*bad, rot, w, w, 1e-6)


def test_entry_points_reject_before_any_launch():
    lib = _lib.declare(ctypes.CDLL(_lib.LIB_PATH))
    a = 1 << 20
    sizes = dict(B=1, L=4, H=8, Hkv=2, D=128, R=128, qb=0, ql=1024, qh=128, kb=0, kl=256, kh=128)

    def forward(type_=0, weight=0, q=a, turns=a, w=a, **change):
        return lib.rda_norm_rotate(q, a, a, a, a, 0, w, a, weight, 1e-6, turns, 1.0, 0, type_, _lib.long_array(list({**sizes, **change}.values())), None)

    def backward(type_=0, weight=0, q=a, turns=a, w=a, **change):
        d = {**sizes, "gb": 0, "gl": 1024, "gh": 128, "hb": 0, "hl": 256, "hh": 128, **change}
        return lib.rda_norm_rotate_back(q, a, a, a, a, a, a, a, a, 0, w, a, weight, 1e-6, turns, 1.0, 0, a, type_, _lib.long_array(list(d.values())), None)

    for bad in (dict(B=0), dict(L=0), dict(H=0), dict(Hkv=0), dict(Hkv=65536), dict(D=120), dict(D=272, R=16), dict(R=0), dict(R=144), dict(type_=3), dict(weight=3), dict(weight=-1),
                dict(q=a + 2), dict(w=a + 4), dict(ql=1028), dict(kh=4), dict(turns=None), dict(L=rotary.MAX_TOKENS + 1)):
        assert forward(**bad) == 1 and backward(**bad) == 1, bad
    assert backward(gl=1028) == 1 and backward(hh=4) == 1
    assert lib.rda_norm_rotate_back_workspace(0, 8, 2, 128) == 0 and lib.rda_norm_rotate_back_workspace(4, 8, 2, 120) == 0
    assert lib.rda_norm_rotate_back_workspace(4, 16, 2, 128) == 1 * 2 * 128 * 4  # a workgroup of four tokens, a slice of each tensor's heads
    assert lib.rda_norm_rotate_back_workspace(1 << 20, 32, 8, 128) == 256 * 3 * 128 * 4


SHAPES = [(1, 1, 1, 16, 16), (1, 32, 8, 128, 128), (5, 3, 1, 64, 32), (130, 7, 7, 128, 64), (33, 40, 8, 128, 128), (9, 5, 5, 80, 48), (4, 33, 3, 256, 256), (3, 2, 2, 240, 16),
          (70, 66, 11, 96, 96), (2, 300, 100, 32, 32)]


def run(dev, type_, weights, layout, tokens, heads, kv, D, R, seed, wide=False, arrange=lambda t: t):
    """(inputs on the CPU; outputs and gradients) of a call and its backward pass."""
    g = gen(seed)
    t = TYPES[type_]
    q, k, gq, gk = ((torch.randn(tokens, h, D, generator=g) * 2).to(t) for h in (heads, kv, heads, kv))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(TYPES[weights]) for _ in range(2))
    positions = torch.randint(0, 5000, (tokens,), generator=g, dtype=torch.int64 if wide else torch.int32)
    rot = rotary.Rotary(R, layout=layout, scaling="yarn", factor=2.0, original=512, device=dev)
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    norm = rotary.HeadNorm(leaves[2], leaves[3], eps=1e-5)
    y = rotary.norm_rotate(arrange(leaves[0]), arrange(leaves[1]), positions.to(dev), rot, norm)
    grads = torch.autograd.grad(y, leaves, [gq.to(dev), gk.to(dev)])
    return (q, k, gq, gk, wq, wk, positions, rot), y, grads


def compare(inputs, y, grads):
    q, k, gq, gk, wq, wk, positions, rot = inputs
    for i, (x, w, grad) in enumerate(((q, wq, gq), (k, wk, gk))):
        close(y[i], *norm_turned(x, w, positions, rot, 1e-5), x.dtype, f"output {i}")
        (gx, gx_off), (gw, gw_off) = norm_turned_back(x, w, grad, positions, rot, 1e-5)
        close(grads[i], gx, gx_off, x.dtype, f"gradient {i}")
        close(grads[2 + i], gw, gw_off, w.dtype, f"weights' gradient {i}")
        assert y[i].dtype == grads[i].dtype == x.dtype and y[i].is_contiguous() and grads[2 + i].dtype == w.dtype


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv,D,R", SHAPES)
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("type_,weights", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32"), ("fp32", "bf16")])
def test_values_and_gradients(dev, type_, weights, layout, tokens, heads, kv, D, R):
    print(f"norm_rotate {type_} {weights} {layout} {tokens} x {heads}/{kv} x {D} ({R})", flush=True)
    compare(*run(dev, type_, weights, layout, tokens, heads, kv, D, R, seed=tokens + D, wide=heads % 2 == 0))


@pytest.mark.gpu
def test_many_tokens(dev):
    """More tokens than the backward pass has workgroups: each takes several; twice the same bits."""
    a = run(dev, "fp32", "fp32", "half", 3500, 9, 2, 64, 64, seed=3)
    compare(*a)
    b = run(dev, "fp32", "fp32", "half", 3500, 9, 2, 64, 64, seed=3)
    assert all(torch.equal(x, y) for x, y in zip((*a[1], *a[2]), (*b[1], *b[2])))


@pytest.mark.gpu
def test_strides_and_sizes(dev):
    """Heads before tokens, parts of one projection, unaligned views, batches, expanded gradients, no tokens, rows of zeros."""
    compare(*run(dev, "bf16", "bf16", "half", 21, 6, 2, 64, 64, seed=4, arrange=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)))
    compare(*run(dev, "fp16", "fp32", "half", 21, 6, 2, 64, 32, seed=5, arrange=lambda t: torch.cat((t, t), 2)[..., :64]))
    compare(*run(dev, "fp16", "fp16", "half", 21, 6, 2, 64, 64, seed=6, arrange=lambda t: torch.cat((t.flatten(), t.flatten()[:1]))[:-1].view(t.shape)))
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)  # noqa: E731
    compare(*run(dev, "bf16", "fp32", "interleaved", 21, 6, 2, 64, 64, seed=7, arrange=odd))
    g = gen(8)
    rot = rotary.Rotary(64, device=dev)
    w = [(1 + 0.3 * torch.randn(64, generator=g)).to(dev).requires_grad_() for _ in range(2)]
    norm = rotary.HeadNorm(*w)
    q, k = torch.randn(3, 5, 4, 64, generator=g).half().to(dev), torch.randn(3, 5, 2, 64, generator=g).half().to(dev)
    positions = torch.arange(15, device=dev).view(3, 5)
    batched = rotary.norm_rotate(q, k, positions, rot, norm)
    flat = rotary.norm_rotate(q.view(15, 4, 64), k.view(15, 2, 64), positions.view(15), rot, norm)
    assert batched[0].shape == q.shape and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(batched, flat))
    one = torch.autograd.grad(sum(x.float().sum() for x in batched), w)  # gradients of one value everywhere, expanded
    two = torch.autograd.grad(flat, w, [torch.ones_like(x) for x in flat])
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    empty = rotary.norm_rotate(q[:0], k[:0], positions[:0], rot, norm)
    assert empty[0].shape == (0, 5, 4, 64) and not any(x.any() for x in torch.autograd.grad(empty, w, [torch.zeros_like(x) for x in empty]))
    zero = rotary.norm_rotate(q * 0, k * 0, positions, rot, norm)
    assert not zero[0].any() and not zero[1].any()


@pytest.mark.gpu
def test_far_positions_and_far_values(dev):
    """Positions past 2^31; heads whose squares are near the ends of fp32's range."""
    g = gen(9)
    rot = rotary.Rotary(128, base=5e5, device=dev)
    q, k = torch.randn(9, 2, 128, generator=g), torch.randn(9, 1, 128, generator=g)
    q[1], q[2] = q[1] * 1e17, q[2] * 1e-12
    positions = torch.randint(-10 ** 6, 10 ** 6, (9,), generator=g)
    positions[0] = 2 ** 31 + 5
    w = torch.ones(128)
    y = rotary.norm_rotate(q.to(dev), k.to(dev), positions.to(dev), rot, rotary.HeadNorm(w.to(dev), w.to(dev), eps=1e-5))
    for got, x in zip(y, (q, k)):
        close(got, *norm_turned(x, w, positions, rot, 1e-5), torch.float32)


@pytest.mark.gpu
def test_recording(dev):
    """Gradients are carried where anything requires one; weights changed in place are seen by later calls and stop an earlier one's backward pass; the
    gradient has none itself."""
    g = gen(10)
    rot, positions = rotary.Rotary(64, device=dev), torch.arange(6, device=dev)
    q, k = torch.randn(6, 4, 64, generator=g).to(dev), torch.randn(6, 2, 64, generator=g).to(dev)
    w = [torch.ones(64, device=dev) for _ in range(2)]
    norm = rotary.HeadNorm(*w)
    a = rotary.norm_rotate(q, k, positions, rot, norm)
    assert not a[0].requires_grad
    w[0] *= 2
    b = rotary.norm_rotate(q, k, positions, rot, norm)
    assert torch.equal(b[0], a[0] * 2) and torch.equal(b[1], a[1])
    w[1].requires_grad_()
    y = rotary.norm_rotate(q, k, positions, rot, norm)
    assert y[0].requires_grad
    with torch.no_grad():
        assert not rotary.norm_rotate(q, k, positions, rot, norm)[0].requires_grad
        w[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y[1].sum().backward()
    y = rotary.norm_rotate(q, k, positions, rot, norm)
    grad, = torch.autograd.grad(y[1].sum(), w[1], create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.gpu
def test_captured(dev):
    """Forward and backward captured together and replayed while values, gradients, weights and positions change: the eager bits each time, and on a side
    stream."""
    g = gen(11)
    rot = rotary.Rotary(64, device=dev)
    leaves = [torch.randn(*s, generator=g).bfloat16().to(dev).requires_grad_() for s in ((37, 4, 64), (37, 2, 64), (64,), (64,))]
    grads = [torch.randn(37, h, 64, generator=g).bfloat16().to(dev) for h in (4, 2)]
    positions, norm = torch.arange(37, dtype=torch.int32, device=dev), rotary.HeadNorm(leaves[2], leaves[3])

    def step():
        y = rotary.norm_rotate(leaves[0], leaves[1], positions, rot, norm)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, grads))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for t in leaves + grads:
                t.copy_(torch.randn(t.shape, generator=g).bfloat16())
            positions += 1000
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        with torch.cuda.stream(side):
            again = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want)), i
