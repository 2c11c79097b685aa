"""What rotary and paged_kv write in place counts as a write in the tensors' version counters, as torch's own in-place operations do: by them
int8_gemv's sibling linears (and autograd) know that a tensor changed. On the CPU, with stand-ins for the launches."""
import ctypes
import types

import pytest
import torch

from comfyui_rdna2_attention_amd import _lib, int8_gemv, paged_kv, rotary
from test_patch_glue import _gemv_layer, _record_gemv_kernels, cast_context


@pytest.fixture
def launches(monkeypatch):
    """Launches that only note that they ran; rotate_positions clears y (fp32, contiguous)."""
    ran = []

    def rotate_positions(x, y, positions, wide, turns, factor, flags, type_, dims, stream):
        ran.append("rotate")
        ctypes.memset(y, 0, 4 * dims[0] * dims[1] * dims[2] * dims[3])
        return 0

    paged = types.SimpleNamespace(paged_append=lambda *a: ran.append("append") or 0, paged_attn=lambda *a: ran.append("attention") or 0,
                                  paged_attn_workspace=lambda *a: 64)
    for module in (rotary, paged_kv):
        monkeypatch.setattr(module, "same_device", lambda *a: None)
    monkeypatch.setattr(rotary, "get_kernels", lambda: types.SimpleNamespace(rotate_positions=rotate_positions))
    monkeypatch.setattr(paged_kv, "get_kernels", lambda: paged)
    monkeypatch.setattr(_lib, "raw_stream", lambda: 0)
    return ran


def world():
    cache = paged_kv.Cache(torch.zeros(4, 8, 2, 64), torch.zeros(4, 8, 2, 64))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return cache, paged_kv.Batch(i32(0, 1, 2, 3).view(1, 4), i32(0, 3), i32(9))


def test_versions(launches):
    x, rot = torch.ones(3, 4, 64), rotary.Rotary(64, device="cpu")
    out, whole = torch.ones(3, 4, 64), torch.ones(3, 6, 64)
    rotary.rotate(x, torch.arange(3), rot, out=out)
    rotary.rotate(x, torch.arange(3), rot)
    assert out._version == 1 and x._version == 0
    rotary.rotate(x, torch.arange(3), rot, out=x)
    assert x._version == 1
    cache, batch = world()
    k, v, q, q_out = torch.ones(3, 2, 64), torch.ones(3, 2, 64), torch.ones(3, 4, 64), torch.ones(3, 4, 64)
    paged_kv.append(cache, batch, k, v)
    assert cache.k._version == 1 and cache.v._version == 1
    paged_kv.append(cache, batch, k, v, q=q, q_out=q_out)
    assert cache.k._version == 2 and cache.v._version == 2 and q_out._version == 1 and q._version == 0
    paged_kv.append(cache, batch, k, v, q=q)
    assert q._version == 1 and k._version == 0 and v._version == 0
    paged_kv.attention(cache, batch, q, out=whole[:, 1:5])  # a view: its base counts
    paged_kv.attention(cache, batch, q)
    assert whole._version == 1 and q._version == 1 and cache.k._version == 3 and batch.lengths._version == 0
    assert launches == ["rotate"] * 3 + ["append"] * 3 + ["attention"] * 2
    with torch.inference_mode():  # tensors without counters
        rotary.rotate(x, torch.arange(3), rot, out=torch.ones(3, 4, 64))


def test_sibling_linears_see_a_turn_in_place(launches, monkeypatch):
    """q's launch computes k's output too, from the values of then; a turn of that input in place makes k compute from the new ones."""
    cast_context(monkeypatch)
    calls = []
    _record_gemv_kernels(monkeypatch, calls)
    int8_gemv.forget_siblings()
    K = 4096
    q, k = _gemv_layer(K, K), _gemv_layer(K, K)
    int8_gemv.register_siblings([(m, K, K, torch.int8, 256) for m in (q, k)])
    x = torch.ones(1, K)
    int8_gemv.linear_forward(q, K, K, torch.int8, 256, x)
    rotary.rotate(x.view(1, 32, 128), torch.arange(1), rotary.Rotary(128, device="cpu"), out=x.view(1, 32, 128))
    got = int8_gemv.linear_forward(k, K, K, torch.int8, 256, x)
    int8_gemv.forget_siblings()
    assert [c[2] for c in calls] == [4096.0, 0.0] and float(got[0]) == 2


def test_saved_tensors_see_a_turn_in_place(launches):
    """autograd refuses a backward pass over a value that rotate has replaced."""
    x, w = torch.ones(3, 4, 64), torch.ones(3, 4, 64, requires_grad=True)
    y = (x * w).sum()
    with torch.no_grad():
        rotary.rotate(x, torch.arange(3), rotary.Rotary(64, device="cpu"), out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
