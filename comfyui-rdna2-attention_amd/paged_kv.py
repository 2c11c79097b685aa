"""A key/value cache in pages, on MI355X: sequences of any lengths share one pool of fixed-size pages, a step appends its new tokens'
keys and values (rotated on the way), and attention reads them for one new token of each sequence or for chunks of prompts. Next to
int8_gemv.attention_decode, whose cache is one contiguous fp32 block per sequence.

A step of a serving loop: write the batch's page table, starts and lengths; `append`; `attention` with the rotated queries. All three
are device tensors that the kernels read: a captured graph of the two calls stays valid while their contents change.

There is no backward pass: where gradients are recorded, tensors that require one are refused.
"""
import torch

from . import _lib
from .hip_attention import Kernels
from .rotary import MAX_TOKENS, TYPES, Sizes, distinct, rows_ready, same_device, vector_rows, written

HEADS = (64, 128)  # head dims of `attention`
MAX_SEQUENCES = 8192
MAX_KEYS = 2 ** 31 - 2 ** 16  # tokens that a row of a page table holds

kernels = None


def get_kernels():
    global kernels
    if kernels is None:
        kernels = Kernels("paged_kv", ("paged_append", "paged_attn", "paged_attn_workspace"))
    return kernels


def _no_gradient(what, *tensors):
    """Raises ValueError if any of the tensors (None: none) requires a gradient and gradients are recorded."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what} has no backward pass and would drop the gradient of its inputs: call it under torch.no_grad(), or with detached tensors")


class Cache:
    """The pages of a layer's keys and values: k and v (pages, page size, KV heads, D), fp16, bf16 or fp32, in any order of
    dimensions in memory but the last, which is contiguous (a (pages, KV heads, page size, D) pool is passed as its
    transpose(1, 2)); rows on 16-byte boundaries, no gradient required. Any page size; multiples of 8 tokens (fp32: 4) are read fastest."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype not in TYPES or v.dtype != k.dtype or k.numel() == 0 or k.shape[3] % 16:
            raise ValueError("Cache takes k and v as (pages, page size, KV heads, D) of one shape, none of it zero, in fp16, bf16 or fp32, D a multiple of 16")
        if not (rows_ready(k) and rows_ready(v)):
            raise ValueError("Cache takes k and v with a contiguous last dimension and rows on 16-byte boundaries")
        if k.device != v.device:
            raise ValueError("Cache takes k and v on one device")
        if k.requires_grad or v.requires_grad:
            raise ValueError("Cache takes k and v that require no gradient: append writes them")
        self._k, self._v = k, v
        self.sizes = (k.dtype, k.shape, k.stride(), v.stride())

    k = property(lambda self: self._k, doc="The pages of the keys.")
    v = property(lambda self: self._v, doc="The pages of the values.")


class Batch:
    """The sequences of a step, all int32 on the device: table (sequences, pages per sequence) -- a sequence's page ids in
    order, entries past its length unread --, starts (sequences + 1) -- its new tokens are rows starts[b] .. starts[b + 1] - 1 of q, k
    and v --, and lengths (sequences) -- its cached tokens, the new ones included. starts does not fall and ends within those rows; rows behind
    the last sequence (a padded batch) belong to none. Of a length past the table's capacity only the keys that the table holds are there;
    positions, and windows with them, follow the length. Keys on pages that the cache does not have are masked."""

    def __init__(self, table, starts, lengths):
        if table.dim() != 2 or starts.dim() != 1 or lengths.dim() != 1 or any(t.dtype != torch.int32 for t in (table, starts, lengths)):
            raise ValueError("Batch takes int32 table (sequences, pages), starts (sequences + 1) and lengths (sequences)")
        B = table.shape[0]
        if B == 0 or table.shape[1] == 0 or starts.shape[0] != B + 1 or lengths.shape[0] != B or B > MAX_SEQUENCES:
            raise ValueError(f"Batch takes 1 to {MAX_SEQUENCES} sequences of at least a page: table (B, pages), starts (B + 1), lengths (B)")
        if table.stride(1) != 1 or not (starts.is_contiguous() and lengths.is_contiguous()):
            raise ValueError("Batch takes a table with contiguous rows, and contiguous starts and lengths")
        if not table.device == starts.device == lengths.device:
            raise ValueError("Batch takes its tensors on one device")
        self._table, self._starts, self._lengths = table, starts, lengths
        self.sizes = (table.shape, table.stride(0))

    def _replace(name):
        def put(self, t):  # also what batch.lengths += 1 does, with the tensor itself
            old = getattr(self, name)
            if t is not old and (t.dtype != old.dtype or t.shape != old.shape or t.stride() != old.stride() or t.device != old.device):
                raise ValueError(f"Batch keeps the type, shape, strides and device of its {name[1:]}")
            setattr(self, name, t)
        return property(lambda self: getattr(self, name), put)

    table, starts, lengths = _replace("_table"), _replace("_starts"), _replace("_lengths")
    del _replace


def _sizes(what, cache, batch):
    """(sequences, pages per sequence, table pitch, pages, page size), checked."""
    (B, N), pitch = batch.sizes
    P, S = cache.k.shape[:2]
    if N * S > MAX_KEYS:
        raise ValueError(f"{what} takes tables of at most {MAX_KEYS} tokens a sequence")
    return B, N, pitch, P, S


_append_sizes, _attention_sizes = Sizes(), Sizes()
_workspaces = {}  # bytes by sizes


def append(cache, batch, k, v, rotary=None, q=None, q_out=None):
    """Writes k and v (tokens, KV heads, D) of the batch's new tokens to their pages, k turned by its position first (`rotary`, as
    rotary.rotate turns it; None: not). The i-th new token of sequence b has position lengths[b] - (starts[b + 1] - starts[b]) + i. k
    and v are fp16, bf16 or fp32, of the cache's type or another: rounded to it once, after the turn. q (tokens, heads, D), if
    given, is turned in the same launch into q_out (the cache's type; None: in place) -- what attention takes. Rows of no
    sequence are left as they were in q_out, as is the cache where a position is negative, past the table or on a page that it does not
    have. Two tokens on one row of one page: either's values may remain, or
    some of each. q_out is q itself or does not overlap q, k and v, and
    none of them overlaps the pages. Returns q_out."""
    kc, vc = cache._k, cache._v
    _no_gradient("append", k, v, q, q_out)
    if q is not None:
        if q_out is None:
            q_out = q
        if q.data_ptr() % 16 and q_out is not q:
            q = q.clone(memory_format=torch.contiguous_format)
    if k.data_ptr() % 16 or v.data_ptr() % 16:
        k, v = k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format)
    key = (cache.sizes, batch.sizes, k.dtype, k.shape, k.stride(), v.dtype, v.shape, v.stride(), 0 if rotary is None else rotary.dim,
           None if q is None else (q.dtype, q.shape, q.stride()), None if q_out is None else (q_out.dtype, q_out.shape, q_out.stride()))
    dims = _append_sizes.get(key)
    if dims is None:
        k, v, q, dims = _check_append(cache, batch, k, v, rotary, q, q_out, key)
    same_device("append", kc, batch._table, k, v, q, q_out, None if rotary is None else rotary.turns)
    if q_out is not None and q_out.data_ptr() % 16:
        raise ValueError(Q_OUT_ERROR)
    if k.shape[0] == 0:
        return q_out
    _lib.check(get_kernels().paged_append(None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), None if q is None else q_out.data_ptr(),
                                          kc.data_ptr(), vc.data_ptr(), batch._table.data_ptr(), batch._starts.data_ptr(), batch._lengths.data_ptr(),
                                          None if rotary is None else rotary.turns.data_ptr(), 1.0 if rotary is None else rotary.factor,
                                          0 if rotary is None else rotary.interleaved, TYPES[k.dtype], TYPES[kc.dtype], dims, _lib.raw_stream()))
    if q is None:
        written(kc, vc)
    else:
        written(kc, vc, q_out)
    return q_out


Q_OUT_ERROR = "append's q_out has q's shape and the cache's type, a contiguous last dimension and rows on 16-byte boundaries, each its own"


def _check_append(cache, batch, k, v, rotary, q, q_out, key):
    """(k, v and q, copied where the kernel cannot address them; the size arguments) of an append call, or ValueError."""
    kc, vc = cache.k, cache.v
    _, _, Hkv, D = kc.shape
    if k.dim() != 3 or k.dtype not in TYPES or k.shape[1:] != (Hkv, D) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"append takes k and v as (tokens, {Hkv}, {D}) of one type: fp16, bf16 or fp32")
    if D > 256 or (rotary is not None and rotary.dim > D):
        raise ValueError("append takes heads of at most 256 values, and no more rotated ones than these")
    T, H = k.shape[0], 0
    if q is not None:
        H = q.shape[1] if q.dim() == 3 else 0
        if q.dim() != 3 or q.dtype != k.dtype or q.shape[0] != T or q.shape[2] != D or H == 0:
            raise ValueError(f"append takes q as ({T}, heads, {D}) of k's type")
        if q_out.shape != q.shape or q_out.dtype != kc.dtype or not (T == 0 or (rows_ready(q_out) and distinct(q_out))):
            raise ValueError(Q_OUT_ERROR)
    elif q_out is not None:
        raise ValueError("append takes q_out with q only")
    B, N, pitch, P, S = _sizes("append", cache, batch)
    if not (distinct(kc) and distinct(vc)):
        raise ValueError("append takes a cache whose pages, rows and heads are not one memory (an expanded view)")
    if T > MAX_TOKENS:
        raise ValueError(f"append takes at most {MAX_TOKENS} tokens")
    if H + 2 * Hkv > 65535:
        raise ValueError("append takes at most 65535 heads")
    ready = T == 0 or all(rows_ready(t) for t in (k, v) + (() if q is None else (q,)))
    if not ready:
        k, v, q = vector_rows(k), vector_rows(v), None if q is None else vector_rows(q)
    none = (0, 0)
    values = [T, H, Hkv, D, 0 if rotary is None else rotary.dim, B, N, pitch, P, S, *(none if q is None else q.stride()[:2]), *k.stride()[:2], *v.stride()[:2],
              *(none if q is None else q_out.stride()[:2]), *kc.stride()[:3], *vc.stride()[:3]]
    return k, v, q, _append_sizes.keep(key, values) if ready else _lib.long_array(values)


def attention(cache, batch, q, out=None, scale=None, softcap=0.0, window=0, slopes=None, prefix=None):
    """Attention of the batch's new tokens q (tokens, heads, D), the cache's type, D 64 or 128, over the cached keys of their sequences.
    A token at position n (its own key included) sees the keys j <= n; with window > 0 those with n - j < window; with prefix (int32,
    one per sequence) also those j < prefix[b], ahead of it or behind the window. Scores are scale q.k (scale None: D^-0.5); with
    softcap > 0, softcap tanh(scale q.k / softcap), to 7e-7 of softcap, or, in fp32 and from a softcap of 1420 on, to 2e-6 of the score (so a cap
    far above the scores changes nothing); with slopes (fp32, one per head, finite), less slopes[h] |n - j|. heads is a multiple of the
    cache's KV heads, which they share in order. A token that sees nothing gets 0. Returns out (q's shape, not overlapping q; rows of no
    sequence left as they were), or a new tensor, with those rows 0. Keys between a prefix and the window cost time as if they were seen. A call takes
    up to 102 MB of workspace from torch's allocator."""
    kc, vc = cache._k, cache._v
    _no_gradient("attention", q, slopes, out)
    fill = out is None
    if fill:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    key = (cache.sizes, batch.sizes, q.dtype, q.shape, q.stride(), out.dtype, out.shape, out.stride(),
           None if slopes is None else (slopes.dtype, slopes.shape, slopes.stride()), None if prefix is None else (prefix.dtype, prefix.shape, prefix.stride()))
    dims = _attention_sizes.get(key)
    if dims is None:
        q, dims = _check_attention(cache, batch, q, out, slopes, prefix, key)
    if scale is None:
        scale = cache._k.shape[3] ** -0.5
    if not 0.0 <= softcap < 1e30 or not 1e-30 < (scale / softcap if softcap else scale) < 1e30 or not 0 <= window < 2 ** 31:
        raise ValueError("attention takes a positive scale, softcap >= 0 (0: none), neither beyond 1e30, and 0 <= window < 2^31 (0: none)")
    same_device("attention", kc, batch._table, q, out, slopes, prefix)
    if q.numel() == 0:
        return out
    address = out.data_ptr()
    if address % 16:
        raise ValueError(OUT_ERROR)
    if address == q.data_ptr():
        raise ValueError("attention's out is not q: rows are written while others' queries are still read")
    T, H, Hkv, D, B = dims[:5]
    type_ = TYPES[q.dtype]
    k = get_kernels()
    sizes = (T, B, H, Hkv, D, type_)
    size = _workspaces.get(sizes)
    if size is None:
        if len(_workspaces) >= 4096:
            _workspaces.clear()
        size = _workspaces[sizes] = k.paged_attn_workspace(*sizes)
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    _lib.check(k.paged_attn(q.data_ptr(), address, kc.data_ptr(), vc.data_ptr(), batch._table.data_ptr(), batch._starts.data_ptr(), batch._lengths.data_ptr(),
                            None if prefix is None else prefix.data_ptr(), None if slopes is None else slopes.data_ptr(), workspace.data_ptr(),
                            scale, softcap, window, fill, type_, dims, _lib.raw_stream()))
    if not fill:
        written(out)
    return out


OUT_ERROR = "attention's out has q's shape and type, a contiguous last dimension and rows on 16-byte boundaries, each its own"


def _check_attention(cache, batch, q, out, slopes, prefix, key):
    """(q, copied where the kernel cannot address it; the size arguments) of an attention call, or ValueError."""
    kc, vc = cache.k, cache.v
    _, _, Hkv, D = kc.shape
    if q.dim() != 3 or q.dtype != kc.dtype or D not in HEADS or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % Hkv:
        raise ValueError(f"attention takes q as (tokens, a multiple of {Hkv} heads, {D}) of the cache's type {kc.dtype}, head dim 64 or 128")
    T, H = q.shape[:2]
    B, N, pitch, P, S = _sizes("attention", cache, batch)
    if out.shape != q.shape or out.dtype != q.dtype or not (T == 0 or (rows_ready(out) and distinct(out))):
        raise ValueError(OUT_ERROR)
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.numel() != H or not slopes.is_contiguous()):
        raise ValueError(f"attention takes slopes as {H} contiguous fp32 values")
    if prefix is not None and (prefix.dtype != torch.int32 or prefix.numel() != B or not prefix.is_contiguous()):
        raise ValueError(f"attention takes prefix as {B} contiguous int32 values")
    if max(*kc.stride()[:2], *vc.stride()[:2]) >= 2 ** 32:
        raise ValueError("attention takes a cache whose pages and rows are less than 2^32 values apart")
    if T * (H // Hkv) >= 2 ** 31:
        raise ValueError("attention takes fewer than 2^31 rows of tokens and heads per KV head")
    ready = T == 0 or rows_ready(q)
    if not ready:
        q = vector_rows(q)
    values = [T, H, Hkv, D, B, N, pitch, P, S, *q.stride()[:2], *out.stride()[:2], *kc.stride()[:3], *vc.stride()[:3]]
    return q, _attention_sizes.keep(key, values) if ready else _lib.long_array(values)
