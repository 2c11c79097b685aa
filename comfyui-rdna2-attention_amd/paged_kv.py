"""A key/value cache in pages, on MI355X: sequences of any lengths share one pool of fixed-size pages, a step appends its new tokens'
keys and values (rotated on the way), and attention reads them for one new token of each sequence or for chunks of prompts. Next to
int8_gemv.attention_decode, whose cache is one contiguous fp32 block per sequence.

The pages hold 16- or 32-bit values (`Cache`), or int8 codes with a scale for each block of tokens and KV head (`QuantizedCache`: half the memory, and half
the time where attention waits for it: single tokens and short chunks. Long chunks and prompts wait for arithmetic, and take from the same time to a fifth
more, with heads of 64 values up to a third); `append` and `attention` take either, `read` gives a quantized cache's values back.

A step of a serving loop: write the batch's page table, starts and lengths; `append`; `attention` with the rotated queries. All three
are device tensors that the kernels read: a captured graph of the two calls stays valid while their contents change.

There is no backward pass: where gradients are recorded, tensors that require one are refused, as tensors with a forward-mode tangent always are.
"""
import torch
from torch.autograd import forward_ad

from . import _lib
from .hip_attention import Kernels
from .rotary import MAX_HEAD, MAX_TOKENS, TYPES, WEIGHTS_ERROR, Sizes, distinct, no_tangents, rows_ready, same_device, vector_rows, written

HEADS = (64, 128)  # head dims of `attention`
MAX_SEQUENCES = 8192
MAX_KEYS = 2 ** 31 - 2 ** 16  # tokens that a row of a page table holds
BLOCKS = (16, 32, 64)  # tokens that share a scale of a quantized cache
OUT_TYPES = (torch.float16, torch.bfloat16)  # of queries over a quantized cache

kernels = None


def get_kernels():
    global kernels
    if kernels is None:
        kernels = Kernels("paged_kv", ("paged_append", "paged_attn", "paged_attn_workspace", "paged_append_i8", "paged_read_i8", "paged_attn_i8", "paged_attn_i8_workspace"))
    return kernels


def _no_gradient(what, *tensors, cache=()):
    """Raises ValueError if any of the tensors (None: none) requires a gradient and gradients are recorded, or if one of them or of the cache's carries a forward-mode
    tangent."""
    if forward_ad._current_level >= 0:
        no_tangents(what, *tensors, *cache)
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
        self._k, self._v = self._tensors = k, v
        self.sizes = (k.dtype, k.shape, k.stride(), v.stride())

    k = property(lambda self: self._k, doc="The pages of the keys.")
    v = property(lambda self: self._v, doc="The pages of the values.")


class QuantizedCache:
    """The pages of a layer's keys and values in 8 bits: k and v int8 codes (pages, page size, KV heads, D), D a multiple of 16, in any order of dimensions in
    memory but the last, which is contiguous, rows on 16-byte boundaries; k_scales and v_scales fp32 (pages, page size / block, KV heads), any strides: a value is
    its code times the scale of its block of 16, 32 or 64 consecutive tokens and KV head. Scales are not negative; one that is not finite stands for
    a block of NaN (to attention, of V, one above 2^126 may; append's are below 2^122). `empty` makes the four tensors.

    append sets a block's scale to the largest magnitude of its new values / 127. A block that is filled by several appends keeps the largest scale so far:
    where it grows, the older codes are rounded to it once more, so that a value written once is off by half a scale at most (and 2^-16 of it), each
    later growth adding at most half of the scale after it. Small blocks follow their tokens' sizes more closely; all cost attention the same. (An append whose
    sequences have fewer than 4 new tokens on average is laid out for single tokens: a long chunk among them takes some 70 us, with blocks of 64 tokens 140.)"""

    def __init__(self, k, v, k_scales, v_scales):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != torch.int8 or v.dtype != torch.int8 or k.numel() == 0 or k.shape[3] % 16:
            raise ValueError("QuantizedCache takes k and v as int8 (pages, page size, KV heads, D) of one shape, none of it zero, D a multiple of 16")
        P, S, heads, _ = k.shape
        block = S // k_scales.shape[1] if k_scales.dim() == 3 and k_scales.shape[1] else 0
        if block not in BLOCKS or k_scales.shape != (P, S // block, heads) or S % block or v_scales.shape != k_scales.shape or \
                k_scales.dtype != torch.float32 or v_scales.dtype != torch.float32:
            raise ValueError("QuantizedCache takes k_scales and v_scales as fp32 (pages, page size / block, KV heads), block 16, 32 or 64")
        for t in (k, v):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(x % 16 for x in t.stride()[:3]):
                raise ValueError("QuantizedCache takes k and v with a contiguous last dimension and rows on 16-byte boundaries")
        if not k.device == v.device == k_scales.device == v_scales.device:
            raise ValueError("QuantizedCache takes its tensors on one device")
        if k_scales.requires_grad or v_scales.requires_grad:
            raise ValueError("QuantizedCache takes scales that require no gradient: append writes them")
        self._k, self._v, self._k_scales, self._v_scales = self._tensors = k, v, k_scales, v_scales
        self.block = block
        self.sizes = (k.dtype, k.shape, k.stride(), v.stride(), block, k_scales.stride(), v_scales.stride())

    @classmethod
    def empty(cls, pages, page_size, kv_heads, dim, block=32, device="cuda"):
        """A cache of `pages` pages of nothing yet, each head's tokens of a page together in memory, which attention reads fastest."""
        if block not in BLOCKS or page_size <= 0 or page_size % block:
            raise ValueError(f"QuantizedCache takes blocks of 16, 32 or 64 tokens, pages of whole blocks, not {block} and {page_size}")
        codes = torch.zeros(2, pages, kv_heads, page_size, dim, dtype=torch.int8, device=device).transpose(2, 3)
        scales = torch.zeros(2, pages, page_size // block, kv_heads, dtype=torch.float32, device=device)
        return cls(codes[0], codes[1], scales[0], scales[1])

    k = property(lambda self: self._k, doc="The codes of the keys.")
    v = property(lambda self: self._v, doc="The codes of the values.")
    k_scales = property(lambda self: self._k_scales, doc="The scales of the keys' blocks.")
    v_scales = property(lambda self: self._v_scales, doc="The scales of the values' blocks.")


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


def append(cache, batch, k, v, rotary=None, q=None, q_out=None, norm=None):
    """Writes k and v (tokens, KV heads, D) of the batch's new tokens to their pages, k turned by its position first (`rotary`, as
    rotary.rotate turns it; None: not). The i-th new token of sequence b has position lengths[b] - (starts[b + 1] - starts[b]) + i. k
    and v are fp16, bf16 or fp32, of the cache's type or another: rounded to it once, after the turn. q (tokens, heads, D), if
    given, is turned in the same launch into q_out (the cache's type; None: in place) -- what attention takes. Rows of no
    sequence are left as they were in q_out, as is the cache where a position is negative, past the table or on a page that it does not
    have. Two tokens on one row of one page: either's values may remain, or
    some of each. q_out is q itself or does not overlap q, k and v, and
    none of them overlaps the pages. Returns q_out.

    A QuantizedCache gets codes, and new scales of the blocks that are written (see there); two tokens of one block belong to one sequence, or either's scale
    may remain for both. q_out is fp16 or bf16 there (None: in place, q in one of them), and `norm` (a rotary.HeadNorm of D weights) norms k and
    q ahead of their turn as rotary.norm_rotate does. (With a Cache, call rotary.norm_rotate first and append its result.)"""
    kc, vc = cache._k, cache._v
    _no_gradient("append", k, v, q, q_out, cache=cache._tensors)
    if isinstance(cache, QuantizedCache):
        return _append_quantized(cache, batch, k, v, rotary, q, q_out, norm)
    if norm is not None:
        raise ValueError("append takes norm with a QuantizedCache; for a Cache, rotary.norm_rotate gives the k and q to append without rotary")
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


_append_quantized_sizes, _read_sizes = Sizes(), Sizes()


def _append_quantized(cache, batch, k, v, rotary, q, q_out, norm):
    """append to a QuantizedCache."""
    kc, vc, ks, vs = cache._k, cache._v, cache._k_scales, cache._v_scales
    if q is not None:
        if q_out is None:
            q_out = q
        if q.data_ptr() % 16 and q_out is not q:
            q = q.clone(memory_format=torch.contiguous_format)
    if k.data_ptr() % 16 or v.data_ptr() % 16:
        k, v = k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format)
    qw, kw = (None, None) if norm is None else (norm.q, norm.k)
    _no_gradient("append", qw, kw)
    if kw is not None and (qw.data_ptr() | kw.data_ptr()) % 16:  # (their data may have been replaced)
        raise ValueError(WEIGHTS_ERROR)
    key = (cache.sizes, batch.sizes, k.dtype, k.shape, k.stride(), v.dtype, v.shape, v.stride(), 0 if rotary is None else rotary.dim,
           None if kw is None else (qw.dtype, qw.shape, qw.stride(), kw.dtype, kw.shape, kw.stride()),
           None if q is None else (q.dtype, q.shape, q.stride()), None if q_out is None else (q_out.dtype, q_out.shape, q_out.stride()))
    dims = _append_quantized_sizes.get(key)
    if dims is None:
        k, v, q, dims = _check_append_quantized(cache, batch, k, v, rotary, q, q_out, norm, key)
    same_device("append", kc, ks, batch._table, k, v, q, q_out, qw, kw, None if rotary is None else rotary.turns)
    if q_out is not None and q_out.data_ptr() % 16:
        raise ValueError(QUANTIZED_Q_OUT_ERROR)
    if k.shape[0] == 0:
        return q_out
    _lib.check(get_kernels().paged_append_i8(
        None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), None if q is None else q_out.data_ptr(), kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(),
        batch._table.data_ptr(), batch._starts.data_ptr(), batch._lengths.data_ptr(), None if rotary is None else rotary.turns.data_ptr(),
        1.0 if rotary is None else rotary.factor, 0 if rotary is None else rotary.interleaved, None if qw is None else qw.data_ptr(),
        None if kw is None else kw.data_ptr(), 2 if kw is None else TYPES[kw.dtype], 0.0 if norm is None else norm.eps, TYPES[k.dtype],
        0 if q is None else TYPES[q_out.dtype], dims, _lib.raw_stream()))
    if q is None:
        written(kc, vc, ks, vs)
    else:
        written(kc, vc, ks, vs, q_out)
    return q_out


QUANTIZED_Q_OUT_ERROR = "append's q_out has q's shape, is fp16 or bf16 over a QuantizedCache, with a contiguous last dimension and rows on 16-byte boundaries, each its own"


def _check_append_quantized(cache, batch, k, v, rotary, q, q_out, norm, key):
    """(k, v and q, copied where the kernel cannot address them; the size arguments) of an append to a QuantizedCache, or ValueError."""
    kc, vc, ks, vs = cache.k, cache.v, cache.k_scales, cache.v_scales
    _, _, Hkv, D = kc.shape
    if k.dim() != 3 or k.dtype not in TYPES or k.shape[1:] != (Hkv, D) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"append takes k and v as (tokens, {Hkv}, {D}) of one type: fp16, bf16 or fp32")
    if D > MAX_HEAD or (rotary is not None and rotary.dim > D):
        raise ValueError(f"append takes heads of at most {MAX_HEAD} values, and no more rotated ones than these")
    if norm is not None and not (norm.q.shape == norm.k.shape == (D,) and norm.q.dtype == norm.k.dtype and norm.k.dtype in TYPES):
        raise ValueError(f"append takes a norm of {D} weights, of one type: fp16, bf16 or fp32")
    if norm is not None and not (norm.q.is_contiguous() and norm.k.is_contiguous()):
        raise ValueError(WEIGHTS_ERROR)
    T, H = k.shape[0], 0
    if q is not None:
        H = q.shape[1] if q.dim() == 3 else 0
        if q.dim() != 3 or q.dtype != k.dtype or q.shape[0] != T or q.shape[2] != D or H == 0:
            raise ValueError(f"append takes q as ({T}, heads, {D}) of k's type")
        if q_out.shape != q.shape or q_out.dtype not in OUT_TYPES or not (T == 0 or (rows_ready(q_out) and distinct(q_out))):
            raise ValueError(QUANTIZED_Q_OUT_ERROR)
    elif q_out is not None:
        raise ValueError("append takes q_out with q only")
    B, N, pitch, P, S = _sizes("append", cache, batch)
    if not all(distinct(t) for t in (kc, vc, ks, vs)):
        raise ValueError("append takes a cache whose pages, rows, heads and scales are not one memory (an expanded view)")
    if T > MAX_TOKENS:
        raise ValueError(f"append takes at most {MAX_TOKENS} tokens")
    if H + 2 * Hkv > 65535:
        raise ValueError("append takes at most 65535 heads")
    ready = T == 0 or all(rows_ready(t) for t in (k, v) + (() if q is None else (q,)))
    if not ready:
        k, v, q = vector_rows(k), vector_rows(v), None if q is None else vector_rows(q)
    none = (0, 0)
    values = [T, H, Hkv, D, 0 if rotary is None else rotary.dim, B, N, pitch, P, S, cache.block, *(none if q is None else q.stride()[:2]), *k.stride()[:2],
              *v.stride()[:2], *(none if q is None else q_out.stride()[:2]), *kc.stride()[:3], *vc.stride()[:3], *ks.stride(), *vs.stride()]
    return k, v, q, _append_quantized_sizes.keep(key, values) if ready else _lib.long_array(values)


def read(cache, batch, tokens, dtype=torch.bfloat16):
    """The values that a QuantizedCache holds for a batch's rows: (k, v), new tensors (tokens, KV heads, D) of dtype (fp16, bf16 or fp32), rounded to it once.
    Row i of sequence b is the token at the position that append would write it to: with starts that step by the lengths, whole sequences. Rows of no
    sequence, and of positions or pages that do not exist, are 0."""
    if not isinstance(cache, QuantizedCache):
        raise ValueError("read takes a QuantizedCache: a Cache's pages hold their values as they are")
    kc, vc, ks, vs = cache._k, cache._v, cache._k_scales, cache._v_scales
    _, _, Hkv, D = kc.shape
    _no_gradient("read", cache=cache._tensors)
    key = (cache.sizes, batch.sizes, tokens, dtype)
    dims = _read_sizes.get(key)
    if dims is None:
        if dtype not in TYPES or not 0 <= tokens <= MAX_TOKENS or D > MAX_HEAD or Hkv > 65535:
            raise ValueError(f"read takes 0 to {MAX_TOKENS} tokens and a dtype of fp16, bf16 or fp32, of a cache of heads of at most {MAX_HEAD} values")
        B, N, pitch, P, S = _sizes("read", cache, batch)
        dims = _read_sizes.keep(key, [tokens, Hkv, D, B, N, pitch, P, S, cache.block, *kc.stride()[:3], *vc.stride()[:3], *ks.stride(), *vs.stride()])
    same_device("read", kc, batch._table)
    k, v = (torch.empty((tokens, Hkv, D), dtype=dtype, device=kc.device) for _ in range(2))
    if tokens:
        _lib.check(get_kernels().paged_read_i8(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), batch._table.data_ptr(), batch._starts.data_ptr(),
                                               batch._lengths.data_ptr(), k.data_ptr(), v.data_ptr(), TYPES[dtype], dims, _lib.raw_stream()))
    return k, v


def attention(cache, batch, q, out=None, scale=None, softcap=0.0, window=0, slopes=None, prefix=None):
    """Attention of the batch's new tokens q (tokens, heads, D), the cache's type (over a QuantizedCache fp16 or bf16), D 64 or 128, over the cached keys of their sequences.
    A token at position n (its own key included) sees the keys j <= n; with window > 0 those with n - j < window; with prefix (int32,
    one per sequence) also those j < prefix[b], ahead of it or behind the window. Scores are scale q.k (scale None: D^-0.5); with
    softcap > 0, softcap tanh(scale q.k / softcap), to 7e-7 of softcap, or, in fp32 and from a softcap of 1420 on, to 2e-6 of the score (so a cap
    far above the scores changes nothing); with slopes (fp32, one per head, finite), less slopes[h] |n - j|. heads is a multiple of the
    cache's KV heads, which they share in order. A token that sees nothing gets 0. Weighted sums are held in fp32 before they are divided: values that pass its range when
    added up over the keys seen give infinities. Weights are rounded before they meet V: over a 16-bit Cache to its type, over a QuantizedCache to fp16, where each weighted value is off by at
    most 2^-11 of itself or 2^-32 of 127 times the largest scale of V that the row sees, whichever is more; and there values of a bf16 query below 2^-28 of their row's
    largest may lose bits. Returns out (q's shape, not overlapping q; rows of no sequence left as they were), or a new tensor, with those rows 0. Keys between a prefix and the window cost time as if they were seen (over a
    QuantizedCache none). A call takes up to 102 MB of workspace from torch's allocator."""
    kc, vc = cache._k, cache._v
    _no_gradient("attention", q, slopes, out, cache=cache._tensors)
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
    quantized = isinstance(cache, QuantizedCache)
    sizes = (T, B, H, Hkv, D, type_, quantized)
    size = _workspaces.get(sizes)
    if size is None:
        if len(_workspaces) >= 4096:
            _workspaces.clear()
        size = _workspaces[sizes] = (k.paged_attn_i8_workspace if quantized else k.paged_attn_workspace)(*sizes[:6])
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    if quantized:
        _lib.check(k.paged_attn_i8(q.data_ptr(), address, kc.data_ptr(), vc.data_ptr(), cache._k_scales.data_ptr(), cache._v_scales.data_ptr(), batch._table.data_ptr(),
                                   batch._starts.data_ptr(), batch._lengths.data_ptr(), None if prefix is None else prefix.data_ptr(),
                                   None if slopes is None else slopes.data_ptr(), workspace.data_ptr(), scale, softcap, window, fill, type_, dims, _lib.raw_stream()))
    else:
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
    quantized = isinstance(cache, QuantizedCache)
    if quantized and (q.dim() != 3 or q.dtype not in OUT_TYPES or D not in HEADS or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % Hkv):
        raise ValueError(f"attention over a QuantizedCache takes q as (tokens, a multiple of {Hkv} heads, {D}) in fp16 or bf16, head dim 64 or 128")
    if not quantized and (q.dim() != 3 or q.dtype != kc.dtype or D not in HEADS or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % Hkv):
        raise ValueError(f"attention takes q as (tokens, a multiple of {Hkv} heads, {D}) of the cache's type {kc.dtype}, head dim 64 or 128")
    T, H = q.shape[:2]
    B, N, pitch, P, S = _sizes("attention", cache, batch)
    if out.shape != q.shape or out.dtype != q.dtype or not (T == 0 or (rows_ready(out) and distinct(out))):
        raise ValueError(OUT_ERROR)
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.numel() != H or not slopes.is_contiguous()):
        raise ValueError(f"attention takes slopes as {H} contiguous fp32 values")
    if prefix is not None and (prefix.dtype != torch.int32 or prefix.numel() != B or not prefix.is_contiguous()):
        raise ValueError(f"attention takes prefix as {B} contiguous int32 values")
    scales = (*cache.k_scales.stride(), *cache.v_scales.stride()) if quantized else ()
    if max(*kc.stride()[:2], *vc.stride()[:2], *scales) >= 2 ** 32 or (quantized and max(kc.stride(1), vc.stride(1)) >= 2 ** 28):
        raise ValueError("attention takes a cache whose pages and rows (of a QuantizedCache: rows 2^28) are less than 2^32 values apart")
    if T * (H // Hkv) >= 2 ** 31:
        raise ValueError("attention takes fewer than 2^31 rows of tokens and heads per KV head")
    ready = T == 0 or rows_ready(q)
    if not ready:
        q = vector_rows(q)
    values = [T, H, Hkv, D, B, N, pitch, P, S, *((cache.block,) if quantized else ()), *q.stride()[:2], *out.stride()[:2], *kc.stride()[:3], *vc.stride()[:3], *scales]
    return q, _attention_sizes.keep(key, values) if ready else _lib.long_array(values)
