"""append and attention have no backward pass: where gradients are recorded, tensors that require one are refused, not silently cut off."""
import pytest
import torch

from comfyui_rdna2_attention_amd import paged_kv
from test_paged_writes import launches, world  # noqa: F401


def test_cache_takes_no_leaves():
    k = torch.zeros(4, 8, 2, 64)
    for bad in ((k.clone().requires_grad_(), k), (k, k.clone().requires_grad_())):
        with pytest.raises(ValueError, match="gradient"):
            paged_kv.Cache(*bad)


def test_append(launches):  # noqa: F811
    cache, batch = world()
    k, q = torch.ones(3, 2, 64), torch.ones(3, 4, 64)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    for bad in (dict(k=grad(k), v=k), dict(k=k, v=grad(k)), dict(k=k, v=k, q=grad(q)), dict(k=k, v=k, q=grad(q), q_out=q), dict(k=k, v=k, q=q, q_out=grad(q))):
        with pytest.raises(ValueError, match="gradient"):
            paged_kv.append(cache, batch, **bad)
        assert launches == []
        with torch.no_grad():
            paged_kv.append(cache, batch, **bad)
        assert launches.pop() == "append"
    paged_kv.append(cache, batch, k, k, q=q)
    with torch.inference_mode():
        paged_kv.append(cache, batch, grad(k), k)


def test_attention(launches):  # noqa: F811
    cache, batch = world()
    q, slopes = torch.ones(3, 4, 64), torch.ones(4)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    for bad in (dict(q=grad(q)), dict(q=q, slopes=grad(slopes)), dict(q=q, out=grad(q))):
        with pytest.raises(ValueError, match="gradient"):
            paged_kv.attention(cache, batch, **bad)
        assert launches == []
        with torch.no_grad():
            paged_kv.attention(cache, batch, **bad)
        assert launches.pop() == "attention"
    assert not paged_kv.attention(cache, batch, q, slopes=slopes).requires_grad
