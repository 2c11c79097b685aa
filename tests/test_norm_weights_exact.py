"""The weights' gradients of norm_rotate as exact sums: heads whose values are one power of two, quarter turns and small whole gradients make every term a whole number
and every sum of them one that 32 bits hold, in any order, so that no token or head may be left out or counted twice."""
import math

import pytest
import torch

from comfyui_rdna2_attention_amd import rotary
from helpers import gen
from paged_reference import turned

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def terms(x, grad, positions, rot):
    """g u of every token and head, in 64 bits: g the gradient turned back, u the values' signs."""
    back, _ = turned(grad, positions, rot, inverse=True)
    whole = back.round()
    assert (back - whole).abs().max() < 1e-6 and (whole != 0).all()
    return whole * x.double().sign()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv,D,R", [(1, 1, 1, 16, 16), (7, 33, 5, 64, 32), (3500, 9, 2, 64, 64), (3077, 16, 8, 128, 128), (13001, 32, 8, 128, 64), (777, 40, 7, 256, 256), (9001, 3, 1, 32, 32)])
@pytest.mark.parametrize("layout", rotary.LAYOUTS)
@pytest.mark.parametrize("type_,weights", [("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp32"), ("bf16", "bf16")])
def test_sums_of_whole_numbers(dev, type_, weights, layout, tokens, heads, kv, D, R):
    g = gen(tokens + D)
    t = TYPES[type_]
    rot = rotary.Rotary(R, radians=[math.pi / 2] * (R // 2), layout=layout, device=dev)
    assert (rot.turns == 0.25).all()  # cosines and sines of whole positions are 0, 1 and -1
    signs = lambda *s: torch.randint(0, 2, s, generator=g) * 2.0 - 1  # noqa: E731
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g, dtype=torch.int32)
    x, grads = [], []
    for h in (heads, kv):
        x.append((signs(tokens, h, D) * 2.0 ** torch.randint(-2, 3, (tokens, h, 1), generator=g)).to(t))
        grads.append((signs(tokens, h, D) * torch.randint(1, 9, (tokens, h, D), generator=g)).to(t))
        assert tokens * h * 8 < 2 ** 24
    leaves = [torch.ones(D, dtype=TYPES[weights], device=dev).requires_grad_() for _ in range(2)]
    norm = rotary.HeadNorm(*leaves, eps=0.0)
    y = rotary.norm_rotate(x[0].to(dev), x[1].to(dev), positions.to(dev), rot, norm)
    got = torch.autograd.grad(y, leaves, [z.to(dev) for z in grads])
    for i in range(2):
        want = terms(x[i], grads[i], positions, rot).sum((0, 1))
        assert torch.equal(got[i].cpu(), want.to(TYPES[weights])), (i, (got[i].cpu().double() - want).abs().max())
