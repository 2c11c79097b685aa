"""Rotary positions for text models on MI355X: pairs of a head's values turned by angles that grow with the token's position, in the
half and the interleaved layout, over all or part of the head, with the frequency scalings of long contexts. The RoPE of a Krea 2
block, whose matrices the model makes (rms_norm.rms_norm_rope), is another operator; paged_kv.append turns queries and keys on the
way into the cache with the same arithmetic as `rotate`. `norm_rotate` norms queries and keys head by head first, in the same pass.
"""
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .hip_attention import Kernels

MAX_HEAD = 256
MAX_TOKENS = 2 ** 26 - 64  # of a call
LAYOUTS = ("half", "interleaved")
TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # the library's type codes

kernels = None


def get_kernels():
    global kernels
    if kernels is None:
        kernels = Kernels("rotary", ("rotate_positions", "norm_rotate", "norm_rotate_back", "norm_rotate_back_workspace"))
    return kernels


def frequencies(dim, base=10000.0, scaling=None, factor=1.0, original=None, low=1.0, high=4.0, fast=32.0, slow=1.0):
    """(radians per position of each of the dim / 2 pairs, the factor on their cosines and sines), in 64 bits. Pair i turns by
    base^(-2 i / dim) radians a position, and with `scaling`

    * "linear": by 1 / factor of it;
    * "ntk": by that of the base times factor^(dim / (dim - 2)), which divides the slowest pair's frequency by factor;
    * "bands": pairs that turn less than `low` times over the `original` context by 1 / factor of it, those of more than `high`
      turns as without scaling, those between by a mix, linear in the turns;
    * "yarn": pairs of fewer than `slow` turns over the original context by 1 / factor of it, those of more than `fast` turns
      as without, those between by a mix, linear in the pair's index (the two bounds rounded outwards to whole
      pairs); cosines and sines times 0.1 ln(factor) + 1."""
    if dim < 2 or dim % 2 or base <= 0 or factor <= 0:
        raise ValueError("frequencies takes an even dim, a positive base and a positive factor")
    if scaling not in (None, "linear", "ntk", "bands", "yarn"):
        raise ValueError(f"scaling is None, 'linear', 'ntk', 'bands' or 'yarn', not {scaling!r}")
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling takes more than one pair")
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling in ("bands", "yarn"):
        if original is None or original <= 0:
            raise ValueError(f"{scaling} scaling takes the original context's length")
        if scaling == "bands":
            if not 0 < low < high:
                raise ValueError("bands scaling takes 0 < low < high")
            kept = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        else:
            if not 0 < slow < fast or base == 1.0:
                raise ValueError("yarn scaling takes 0 < slow < fast and a base other than 1")
            first, last = (dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow))
            first, last = max(math.floor(first), 0), min(math.ceil(last), dim - 1)
            kept = [1.0 - min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0) for i in range(dim // 2)]
        f = [x * k + x / factor * (1.0 - k) for x, k in zip(f, kept)]
    return f, 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1.0 else 1.0


class Rotary:
    """How a model's heads turn: `dim` rotated values at the head's start (a multiple of 16), the layout of their pairs -- "half":
    values i and i + dim / 2, "interleaved": 2 i and 2 i + 1 -- and their frequencies, by the arguments of `frequencies`, or
    given as radians per position (dim / 2 numbers). `attention` replaces the factor on cosines and sines. Kept on `device`
    as dim / 2 numbers of 64 bits; a program makes it once."""

    def __init__(self, dim, base=10000.0, layout="half", scaling=None, attention=None, radians=None, device="cuda", **options):
        if dim <= 0 or dim % 16 or dim > MAX_HEAD:
            raise ValueError(f"Rotary takes a dim that is a multiple of 16, at most {MAX_HEAD}, not {dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"layout is 'half' or 'interleaved', not {layout!r}")
        if radians is None:
            radians, factor = frequencies(dim, base, scaling, **options)
        else:
            if scaling is not None or options:
                raise ValueError("Rotary takes radians, or the arguments that they are made from")
            radians, factor = [float(x) for x in radians], 1.0
            if len(radians) != dim // 2:
                raise ValueError(f"Rotary takes {dim // 2} radians per position, not {len(radians)}")
        self.dim, self.layout, self.factor = dim, layout, float(factor if attention is None else attention)
        self.interleaved = int(layout == "interleaved")
        self.turns = torch.tensor([x / (2 * math.pi) for x in radians], dtype=torch.float64, device=device)


def vector_rows(t):
    """t as the kernels address it -- a contiguous last dimension, rows on 16-byte boundaries -- copied if it is not."""
    if rows_ready(t):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def rows_ready(t):
    strides, vector = t.stride(), 16 // t.element_size()
    if strides[-1] != 1 or t.data_ptr() % 16:
        return False
    for s in strides[:-1]:
        if s % vector:
            return False
    return True


def distinct(t):
    """Whether no dimension of t repeats one address (expanded views): what a kernel writes has to."""
    return all(s != 0 or n == 1 for s, n in zip(t.stride(), t.shape))


def same_device(what, *tensors):
    """Raises ValueError unless every tensor (None: none) is on the current GPU: the kernels run on its current stream."""
    device = -1
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if device == -1:
                device = d if d >= 0 and d == torch._C._cuda_getDevice() else -2
            if d != device:
                raise ValueError(f"{what} runs on the current GPU; its tensors are on {', '.join(sorted({str(x.device) for x in tensors if x is not None}))}")


def written(*tensors):
    """Counts a write in the tensors' versions, as torch's own in-place operations do: a kernel's write through an address counts none, and
    int8_gemv's sibling linears and autograd would take the tensors for unchanged."""
    torch._C._increment_version(tensors)


def no_tangents(what, *tensors):
    """Raises ValueError if any of the tensors (None: none) carries a forward-mode tangent: the kernels would drop it. (torch.no_grad() does not end forward mode.) Called
    where a level of it is open: that look is all that a call without one pays."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what} has no forward mode and would drop its tensors' tangents: call it with the primals of torch.autograd.forward_ad.unpack_dual")


class Sizes(dict):
    """The size arguments (and bytes of workspace) of an operator's calls by their tensors' types, shapes and strides: checked and packed once for each."""

    def keep(self, key, values, workspace=None):
        if len(self) >= 4096:
            self.clear()
        self[key] = value = _lib.long_array(values) if workspace is None else (_lib.long_array(values), workspace)
        return value


class _Turn(torch.autograd.Function):
    """rotate where gradients are recorded: linear in x, so that its gradient is the turn back (times the factor), and that one's the turn."""

    @staticmethod
    def forward(ctx, x, positions, rotary, inverse):
        ctx.save_for_backward(positions, rotary.turns)
        ctx.rotary, ctx.inverse = rotary, inverse
        return rotate(x, positions, rotary, inverse=inverse)

    @staticmethod
    def backward(ctx, grad):
        return rotate(grad, ctx.saved_tensors[0], ctx.rotary, inverse=not ctx.inverse), None, None, None


_rotate_sizes = Sizes()


def rotate(x, positions, rotary, out=None, inverse=False):
    """x (tokens, heads, D) or (batch, length, heads, D) in fp16, bf16 or fp32, D a multiple of 16 up to 256, turned by `positions`
    (tokens) or (batch, length), int32 or int64: a pair's angle is its frequency times the position, the product in 64 bits, the
    turn in 32, rounded once. Values past rotary.dim are copied. inverse turns back: the gradient of x for a gradient of the result
    (and, where rotary.factor is 1, x itself). Any strides of x with a contiguous last dimension (other heads-first
    layouts are views of these shapes); out, if given, is x itself or does not overlap it. Returns out, or a new contiguous tensor, which
    carries x's gradient where gradients are recorded (an out carries none, and is refused there if x or out requires one). Forward-mode tangents are refused."""
    made = out is None
    if forward_ad._current_level >= 0:
        no_tangents("rotate", x, out)
    if (x.requires_grad or (not made and out.requires_grad)) and torch.is_grad_enabled():
        if not made:
            raise ValueError("rotate records no gradient through out: leave it, or call under torch.no_grad()")
        return _Turn.apply(x, positions, rotary, inverse)
    if made:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    positions = positions.contiguous()
    key = (x.dtype, x.shape, x.stride(), out.dtype, out.shape, out.stride(), positions.dtype, positions.shape, rotary.dim)
    dims = _rotate_sizes.get(key)
    if dims is None:
        x, dims = _check_rotate(x, positions, rotary, out, key)
    same_device("rotate", x, positions, rotary.turns, out)
    if out.data_ptr() % 16:
        raise ValueError(OUT_ERROR)
    if x.numel() == 0:
        return out
    _lib.check(get_kernels().rotate_positions(x.data_ptr(), out.data_ptr(), positions.data_ptr(), positions.dtype is torch.int64, rotary.turns.data_ptr(),
                                              rotary.factor, rotary.interleaved + 2 * bool(inverse), TYPES[x.dtype], dims, _lib.raw_stream()))
    if not made:
        written(out)
    return out


OUT_ERROR = "rotate's out has x's shape and type, a contiguous last dimension and rows on 16-byte boundaries, each its own"


def _check_rotate(x, positions, rotary, out, key):
    """(x, copied where the kernel cannot address it; the size arguments) of a rotate call, or ValueError."""
    if x.dim() not in (3, 4) or x.dtype not in TYPES or x.shape[-1] % 16 or not rotary.dim <= x.shape[-1] <= MAX_HEAD or x.shape[-2] > 65535:
        raise ValueError(f"rotate takes (tokens, heads, D) or (batch, length, heads, D) in fp16, bf16 or fp32, D a multiple of 16 from {rotary.dim} "
                         f"to {MAX_HEAD}, at most 65535 heads, not {tuple(x.shape)} {x.dtype}")
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != x.shape[:-2]:
        raise ValueError(f"rotate takes int32 or int64 positions of shape {tuple(x.shape[:-2])}, not {tuple(positions.shape)} {positions.dtype}")
    if positions.numel() > MAX_TOKENS:
        raise ValueError(f"rotate takes at most {MAX_TOKENS} tokens")
    if out.shape != x.shape or out.dtype != x.dtype or not (out.numel() == 0 or (rows_ready(out) and distinct(out))):
        raise ValueError(OUT_ERROR)
    ready = x.numel() == 0 or rows_ready(x)
    if not ready:
        x = x.clone(memory_format=torch.contiguous_format)
    B, L = (1, x.shape[0]) if x.dim() == 3 else x.shape[:2]
    sx, so = x.stride(), out.stride()
    values = [B, L, x.shape[-2], x.shape[-1], rotary.dim, *(sx[:3] if x.dim() == 4 else (0, *sx[:2])), *(so[:3] if x.dim() == 4 else (0, *so[:2]))]
    return x, _rotate_sizes.keep(key, values) if ready else _lib.long_array(values)


WEIGHTS_ERROR = "HeadNorm takes contiguous weights on 16-byte boundaries"


class HeadNorm:
    """RMS norms of a layer's query and key heads: q and k are their weights, (D,) each, contiguous, of one type (fp16, bf16 or fp32), kept as they are -- a
    training step's updates of them are seen --, eps what is added to a head's mean square."""

    def __init__(self, q, k, eps=1e-6):
        if q.dim() != 1 or q.shape != k.shape or q.dtype not in TYPES or k.dtype != q.dtype or q.device != k.device or q.numel() == 0 or q.numel() % 16:
            raise ValueError("HeadNorm takes weights q and k as (D,) of one type (fp16, bf16 or fp32) on one device, D a multiple of 16")
        if not (rows_ready(q) and rows_ready(k)):
            raise ValueError(WEIGHTS_ERROR)
        if not 0.0 <= eps < 1e30:
            raise ValueError("HeadNorm takes an eps that is not negative")
        self._q, self._k, self.eps = q, k, float(eps)

    q = property(lambda self: self._q, doc="The weights of the query heads.")
    k = property(lambda self: self._k, doc="The weights of the key heads.")


_norm_sizes, _norm_back_sizes = Sizes(), Sizes()


class _NormTurn(torch.autograd.Function):
    """norm_rotate where gradients are recorded; the gradient has none itself."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, rotary, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, rotary.turns)
        ctx.rotary, ctx.eps = rotary, eps
        return _norm_rotate(q, k, positions, rotary, q_weight, k_weight, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, q_grad, k_grad):
        q, k, q_weight, k_weight, positions, _ = ctx.saved_tensors
        return (*_norm_rotate_back(q, k, q_grad, k_grad, positions, ctx.rotary, q_weight, k_weight, ctx.eps), None, None, None)


def norm_rotate(q, k, positions, rotary, norm):
    """q (tokens, heads, D) and k (tokens, KV heads, D), or both with a batch dimension before them as rotate takes, normed head by head and turned by
    `positions`, in one launch: (q, k), new contiguous tensors of their type. A head x becomes the turn of w x / sqrt(mean(x^2) + norm.eps), w norm.q or
    norm.k, in 32 bits, rounded once. Any strides with a contiguous last dimension. Gradients of q, k and the weights are carried where they are
    recorded, those of the weights summed in 32 bits and rounded once; the same inputs give the same bits. (A backward pass is captured as torch's own are: with
    no graph of the same leaves alive that was recorded outside of the capture.) Forward-mode tangents are refused."""
    if forward_ad._current_level >= 0:
        no_tangents("norm_rotate", q, k, norm.q, norm.k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or norm.q.requires_grad or norm.k.requires_grad):
        return _NormTurn.apply(q, k, norm.q, norm.k, positions, rotary, norm.eps)
    return _norm_rotate(q, k, positions, rotary, norm.q, norm.k, norm.eps)


def _norm_rotate(q, k, positions, rotary, q_weight, k_weight, eps):
    q, k, positions = _aligned(q), _aligned(k), positions.contiguous()
    if (q_weight.data_ptr() | k_weight.data_ptr()) % 16:  # (their data may have been replaced)
        raise ValueError(WEIGHTS_ERROR)
    key = (q.dtype, q.shape, q.stride(), k.dtype, k.shape, k.stride(), positions.dtype, positions.shape, rotary.dim,
           q_weight.dtype, q_weight.shape, q_weight.stride(), k_weight.dtype, k_weight.shape, k_weight.stride())
    dims = _norm_sizes.get(key)
    if dims is None:
        q, k, dims = _check_norm_rotate(q, k, positions, rotary, q_weight, k_weight, key)
    same_device("norm_rotate", q, k, positions, q_weight, k_weight, rotary.turns)
    q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
    if positions.numel() == 0:
        return q_out, k_out
    _lib.check(get_kernels().norm_rotate(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), positions.data_ptr(), positions.dtype is torch.int64,
                                         q_weight.data_ptr(), k_weight.data_ptr(), TYPES[q_weight.dtype], eps, rotary.turns.data_ptr(), rotary.factor,
                                         rotary.interleaved, TYPES[q.dtype], dims, _lib.raw_stream()))
    return q_out, k_out


def _norm_rotate_back(q, k, q_grad, k_grad, positions, rotary, q_weight, k_weight, eps):
    """The gradients of q, k and the weights."""
    if forward_ad._current_level >= 0:
        no_tangents("norm_rotate's gradient", q, k, q_grad, k_grad, q_weight, k_weight)
    positions = positions.contiguous()
    key = (q.dtype, q.shape, q.stride(), k.dtype, k.shape, k.stride(), q_grad.shape, q_grad.stride(), k_grad.shape, k_grad.stride(), positions.shape, rotary.dim,
           q_weight.dtype, q_weight.shape, q_weight.stride(), k_weight.dtype, k_weight.shape, k_weight.stride())
    sizes = _norm_back_sizes.get(key)
    if sizes is None or (q.data_ptr() | k.data_ptr() | q_grad.data_ptr() | k_grad.data_ptr()) % 16:
        if not (q_weight.shape == k_weight.shape == q.shape[-1:] and q_weight.dtype == k_weight.dtype and rows_ready(q_weight) and rows_ready(k_weight)):
            raise ValueError("norm_rotate's gradient takes the weights that its call took: their data has been replaced")
        if q_grad.shape != q.shape or k_grad.shape != k.shape or q.dtype != k.dtype or positions.shape != q.shape[:-2] or positions.shape != k.shape[:-2]:
            raise ValueError("norm_rotate's gradient takes the q, k and positions that its call took: their data has been replaced")
        ready = all(rows_ready(t) for t in (q, k, q_grad, k_grad))
        q, k, q_grad, k_grad = vector_rows(q), vector_rows(k), vector_rows(q_grad), vector_rows(k_grad)
        sizes = _norm_back_dims(q, k, q_grad, k_grad, rotary, key if ready else None)
    q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
    if positions.numel() == 0:
        return q_out, k_out, torch.zeros_like(q_weight), torch.zeros_like(k_weight)
    q_weight_out, k_weight_out = torch.empty_like(q_weight), torch.empty_like(k_weight)
    same_device("norm_rotate's gradient", q, k, q_grad, k_grad, positions, q_weight, k_weight, rotary.turns)
    dims, size = sizes
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    kernels = get_kernels()
    _lib.check(kernels.norm_rotate_back(q.data_ptr(), k.data_ptr(), q_grad.data_ptr(), k_grad.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                                        q_weight_out.data_ptr(), k_weight_out.data_ptr(), positions.data_ptr(), positions.dtype is torch.int64,
                                        q_weight.data_ptr(), k_weight.data_ptr(), TYPES[q_weight.dtype], eps, rotary.turns.data_ptr(), rotary.factor,
                                        rotary.interleaved, workspace.data_ptr(), TYPES[q.dtype], dims, _lib.raw_stream()))
    return q_out, k_out, q_weight_out, k_weight_out


def _aligned(t):
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


def _strides(t):
    return t.stride()[:3] if t.dim() == 4 else (0, *t.stride()[:2])


def _norm_dims(q, k, rotary):
    B, L = (1, q.shape[0]) if q.dim() == 3 else q.shape[:2]
    return [B, L, q.shape[-2], k.shape[-2], q.shape[-1], rotary.dim, *_strides(q), *_strides(k)]


def _norm_back_dims(q, k, q_grad, k_grad, rotary, key):
    """(the size arguments, bytes of workspace) of a gradient; kept for the key (None: not)."""
    values = _norm_dims(q, k, rotary) + [s for t in (q_grad, k_grad) for s in _strides(t)]
    B, L, H, Hkv, D = values[:5]
    size = get_kernels().norm_rotate_back_workspace(B * L, H, Hkv, D) if B * L else 0
    return (_lib.long_array(values), size) if key is None else _norm_back_sizes.keep(key, values, size)


def _check_norm_rotate(q, k, positions, rotary, weight, k_weight, key):
    """(q and k, copied where the kernel cannot address them; the size arguments) of a norm_rotate call, or ValueError."""
    if weight.dtype not in TYPES or k_weight.dtype != weight.dtype or k_weight.shape != weight.shape or weight.dim() != 1:
        raise ValueError("norm_rotate takes weights of one type (fp16, bf16 or fp32) and size")
    if not (weight.is_contiguous() and k_weight.is_contiguous()):
        raise ValueError(WEIGHTS_ERROR)
    D = weight.shape[0]
    if q.dim() not in (3, 4) or q.dtype not in TYPES or q.shape[-1] != D or not 0 < q.shape[-2] <= 65535 or not rotary.dim <= D <= MAX_HEAD:
        raise ValueError(f"norm_rotate takes q as (tokens, heads, D) or (batch, length, heads, D) in fp16, bf16 or fp32, D the weights' {D}, from {rotary.dim} "
                         f"to {MAX_HEAD}, 1 to 65535 heads, not {tuple(q.shape)} {q.dtype}")
    if k.dtype != q.dtype or k.shape[:-2] != q.shape[:-2] or k.dim() != q.dim() or k.shape[-1] != D or not 0 < k.shape[-2] <= 65535:
        raise ValueError(f"norm_rotate takes k of q's type, tokens and D, not {tuple(k.shape)} {k.dtype}")
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != q.shape[:-2]:
        raise ValueError(f"norm_rotate takes int32 or int64 positions of shape {tuple(q.shape[:-2])}, not {tuple(positions.shape)} {positions.dtype}")
    if positions.numel() > MAX_TOKENS:
        raise ValueError(f"norm_rotate takes at most {MAX_TOKENS} tokens")
    ready = q.numel() == 0 or (rows_ready(q) and rows_ready(k))
    if not ready:
        q, k = vector_rows(q), vector_rows(k)
    values = _norm_dims(q, k, rotary)
    return q, k, _norm_sizes.keep(key, values) if ready else _lib.long_array(values)
