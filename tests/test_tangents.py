"""Forward-mode tangents (torch.autograd.forward_ad): no operator of rotary and paged_kv makes its outputs' ones, so tensors that carry one are refused, not silently
cut off. On the CPU: the calls refuse before any launch."""
import pytest
import torch
from torch.autograd import forward_ad

from comfyui_rdna2_attention_amd import paged_kv, rotary

CALLS = ["rotate x", "rotate out", "norm_rotate q", "norm_rotate k", "norm_rotate norm.q", "norm_rotate norm.k", "append k", "append v", "append q", "append q_out", "append pages",
         "append quantized k", "append norm.k", "append k_scales", "read v_scales", "attention q", "attention slopes", "attention out", "attention pages", "attention quantized q",
         "attention k_scales"]


def call(name, change):
    """Makes the call, `change` applied to the tensor that its name ends with."""
    operator, *rest = name.split()
    which = rest[-1]
    put = lambda n, t: change(t) if n == which else t  # noqa: E731
    rot, n = rotary.Rotary(64, device="cpu"), torch.arange(3)
    q, k = torch.ones(3, 4, 64), torch.ones(3, 2, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    batch = paged_kv.Batch(i32(0, 1).view(1, 2), i32(0, 3), i32(9))
    codes = [torch.zeros(4, 32, 2, 64, dtype=torch.int8) for _ in range(2)]
    if operator == "rotate":
        return rotary.rotate(put("x", q), n, rot, out=put("out", torch.ones(3, 4, 64)) if which == "out" else None)
    norm = rotary.HeadNorm(put("norm.q", torch.ones(64)), put("norm.k", torch.ones(64)))
    if operator == "norm_rotate":
        return rotary.norm_rotate(put("q", q), put("k", k), n, rot, norm)
    quantized = operator == "read" or "quantized" in rest or which in ("k_scales", "norm.k")
    cache = paged_kv.QuantizedCache(*codes, put("k_scales", torch.zeros(4, 2, 2)), put("v_scales", torch.zeros(4, 2, 2))) if quantized else \
        paged_kv.Cache(torch.zeros(4, 32, 2, 64), put("pages", torch.zeros(4, 32, 2, 64)))
    if operator == "append":
        return paged_kv.append(cache, batch, put("k", k), put("v", k), q=put("q", q), q_out=put("q_out", torch.ones(3, 4, 64, dtype=torch.float16 if quantized else torch.float32)),
                               norm=norm if which == "norm.k" else None)
    if operator == "read":
        return paged_kv.read(cache, batch, 3)
    q = q.half() if quantized else q
    return paged_kv.attention(cache, batch, put("q", q), slopes=put("slopes", torch.ones(4)), out=put("out", torch.ones_like(q)))


@pytest.mark.parametrize("name", CALLS)
def test_refused(name):
    with forward_ad.dual_level():
        for context in (torch.enable_grad, torch.no_grad):  # which forward mode does not go by
            with context(), pytest.raises(ValueError, match="tangent"):
                call(name, lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="current GPU"):  # as without a level
            call(name, lambda t: t)
        with pytest.raises(ValueError, match="current GPU"):
            call(name, lambda t: forward_ad.unpack_dual(forward_ad.make_dual(t, torch.ones_like(t))).primal)
    with pytest.raises(ValueError, match="current GPU"):
        call(name, lambda t: t)


@pytest.mark.parametrize("name", ["rotate x", "norm_rotate q", "norm_rotate norm.k"])
def test_refused_where_gradients_are_recorded(name):
    with forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        call(name, lambda t: forward_ad.make_dual(t.requires_grad_(), torch.ones_like(t)))


def test_gradients_that_carry_a_tangent():
    """Backward passes under a dual level: their own inputs are looked at too."""
    rot, n, w = rotary.Rotary(64, device="cpu"), torch.arange(3), torch.ones(64)
    q, k = torch.ones(3, 4, 64), torch.ones(3, 2, 64)
    with forward_ad.dual_level():
        for i in range(2):
            grads = [q.clone(), k.clone()]
            grads[i] = forward_ad.make_dual(grads[i], grads[i].clone())
            with pytest.raises(ValueError, match="tangent"):
                rotary._norm_rotate_back(q, k, *grads, n, rot, w, w, 1e-6)


def test_functional_jvp():
    """torch.func.jvp gives an error too, not a result without a tangent."""
    rot, n = rotary.Rotary(64, device="cpu"), torch.arange(3)
    norm, k = rotary.HeadNorm(torch.ones(64), torch.ones(64)), torch.ones(3, 2, 64)
    q = torch.ones(3, 4, 64)
    for f in (lambda x: rotary.rotate(x, n, rot), lambda x: rotary.norm_rotate(x, k, n, rot, norm)):
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(f, (q,), (torch.ones_like(q),))
