"""A key/value cache in pages, and the decode steps that read it.

What a serving program does after the prompt, for which the reference has no operator of its own (its decode steps go to
``flash_attn_func`` over a contiguous cache, anchor_attn/src/modules/llama/anchor_attention.py:101-109): keys and values lie in pages of 16 to
256 rows anywhere in a pool, a table names the pages of each sequence in order, and lengths say how many keys it has.

* :func:`append_to_pages` rotates new queries and keys by their positions and stores keys and values in their pages;
* :func:`paged_decode_attention` is attention of one new token per sequence over all its keys;
* :func:`paged_sparse_decode_attention` is the same over a fixed number of pages, those whose keys can score highest.

Tables, lengths and starts are int32 tensors on the GPU and are read there: a step needs nothing from the host, and the same
captured graph serves any lengths.  What they hold is not trusted: lengths are clamped to the table, pages outside the pool are
never accessed (``include/anchor_attn_hip.h`` says what is done instead).  Nothing here is differentiable.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _hip
from .anchor_attn_v4 import _called_plainly
from .anchor_step_1_2_v2 import _raw_stream, _stream

PAGE_SIZES = (16, 32, 64, 128, 256)
_TYPES = (torch.Tensor, torch.nn.Parameter)
_HALF = (torch.bfloat16, torch.float16)
_INT32, _FLOAT32 = torch.int32, torch.float32


def _refuse(what: str):
    raise _hip.AnchorAttnHipError(f"paged cache: {what}")


def _rows(t, name, cache, heads):
    """``(data_ptr, token stride, head stride)`` of a tensor ``[tokens, heads, head dimension]`` and its shape."""
    if type(t) not in _TYPES or t.dtype != cache.dtype or t.get_device() != cache.index or t.dim() != 3:
        _refuse(f"{name} must be a tensor [tokens, heads, head dimension] of the cache's type and device")
    _, h, d = shape = t.shape
    st, sh, sd = t.stride()
    ptr = t.data_ptr()
    if d != cache.head_dim or (h != heads if heads else not h or h % cache.n_kv_heads):
        _refuse(f"{name} has {h} heads of {d}, the cache {cache.n_kv_heads} of {cache.head_dim}")
    if sd != 1 or (st | sh) & 7 or ptr & 15:
        _refuse(f"the rows of {name} must be contiguous and begin on 16-byte boundaries")
    return (ptr, st, sh), shape


def _indices(t, name, cache, dim, rows=None):
    """``data_ptr`` of a tensor of whole numbers."""
    if type(t) not in _TYPES or t.dtype != _INT32 or t.get_device() != cache.index or t.dim() != dim or (t.stride(-1) != 1 and t.shape[-1] > 1):
        _refuse(f"{name} must be an int32 tensor of {dim} dimension{'s' if dim > 1 else ''} on the cache's device, its rows contiguous")
    if rows is not None and t.shape[0] != rows:
        _refuse(f"{name} has {t.shape[0]} entries where {rows} are expected")
    return t.data_ptr()


def _dims(t):
    """``(stride, size)`` of a tensor's dimensions of more than one entry, the largest stride first."""
    return sorted(((s, n) for s, n in zip(t.stride(), t.shape) if n > 1), reverse=True)


def _extent(dims):
    """Elements from a tensor's first to its last."""
    return 1 + sum(s * (n - 1) for s, n in dims)


def _own_places(dims):
    """Whether every stride reaches beyond what the smaller ones span, as in every part or transposition of a contiguous tensor: no two entries are one place."""
    return all(s >= _extent(dims[i + 1:]) for i, (s, _) in enumerate(dims))


def _apart(a, b, distance):
    """Whether two such tensors, the second beginning ``distance`` elements behind the first, share no place (False where that cannot be told)."""
    if distance >= _extent(a) or -distance >= _extent(b):
        return True
    if not a or not b or a[0][0] != b[0][0]:
        return False
    stride = a[0][0]  # (one of the other's entries begins less than a stride behind each entry, and one less than a stride before it)
    return _apart(a[1:], b[1:], distance % stride) and _apart(a[1:], b[1:], distance % stride - stride)


class PagedCache:
    """Keys and values in pages: ``keys``, ``values`` ``[n_pages, n_kv_heads, page_size, head_dim]`` (bf16 or fp16 on one GPU, rows contiguous on
    16-byte boundaries, the other strides free; to be appended to, those of any part or transposition of a tensor, no two places the same memory) and, for
    sparse steps, ``bounds`` ``[n_pages, n_kv_heads, 2, head_dim]`` (contiguous): the smallest and the largest value of each channel over a page's keys, which :func:`append_to_pages` sets with a page's first key and widens with the
    others (keys that are taken back by a smaller length stay in them until the first is stored again; whoever copies pages copies their bounds).  The contents of pages that no table names
    do not matter.  The tensors stay the cache's own for as long as it is used: their contents may change, their memory may not, and a cache gets no others.  After
    ``cache.keys.data = ...`` or a ``resize_`` that moves them calls are refused.  ``weights``, optional, float32 ``[n_pages, n_kv_heads, page_size]`` (contiguous): how
    much attention each key has had, 0 when it is appended, counted by :func:`paged_weighing_decode_attention`, read by :func:`evict_from_pages`."""

    __slots__ = ("keys", "values", "bounds", "weights", "dtype", "device", "index", "n_pages", "n_kv_heads", "page_size", "head_dim", "_struct", "_address",
                 "_addresses", "_pointers", "_apart", "_memory", "_weights")

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, bounds: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None):
        tensors = (keys, values) if bounds is None else (keys, values, bounds)
        if any(type(t) not in _TYPES or t.dim() != 4 or t.dtype != keys.dtype or t.device != keys.device or not t.is_cuda for t in tensors):
            _refuse("keys, values and bounds must be tensors of four dimensions, one type and one GPU")
        if keys.dtype not in _HALF or any(t.requires_grad for t in tensors):
            _refuse("keys, values and bounds must be bf16 or fp16 and need no gradients")
        n_pages, kv_heads, page_size, d = keys.shape
        if values.shape != keys.shape or d not in (64, 128) or page_size not in PAGE_SIZES or not n_pages or not kv_heads or n_pages >= 1 << 31:
            _refuse(f"keys and values must be [pages, KV heads, page size, head dimension] with pages of {PAGE_SIZES} and a head dimension of 64 or 128, "
                    f"not {tuple(keys.shape)} and {tuple(values.shape)}")
        for t in (keys, values):
            sp, sh, sn, sd = t.stride()
            if sd != 1 or (sp | sh | sn) & 7 or t.data_ptr() & 15 or not d <= sn <= 1 << 14 or (not sp and n_pages > 1) or (not sh and kv_heads > 1):
                _refuse("the rows of keys and values must be contiguous, begin on 16-byte boundaries and lie at most 16384 elements apart, and no two share memory")
        if bounds is not None and (bounds.shape != (n_pages, kv_heads, 2, d) or not bounds.is_contiguous() or bounds.data_ptr() & 15):
            _refuse(f"bounds must be a contiguous tensor {(n_pages, kv_heads, 2, d)}, not {tuple(bounds.shape)}")
        if weights is not None:
            if type(weights) not in _TYPES or weights.dtype != _FLOAT32 or weights.device != keys.device or weights.shape != (n_pages, kv_heads, page_size):
                _refuse(f"weights must be a float32 tensor {(n_pages, kv_heads, page_size)} on the cache's device")
            if not weights.is_contiguous() or weights.data_ptr() & 15 or weights.requires_grad:
                _refuse("weights must be contiguous on a 16-byte boundary and need no gradients")
            begin, end = weights.data_ptr(), weights.data_ptr() + 4 * weights.numel()
            if any(begin < t.data_ptr() + 2 * _extent(_dims(t)) and t.data_ptr() < end for t in tensors):
                _refuse("weights must lie apart from keys, values and bounds")
        # (reading does not mind; what is written twice at once would be anything)
        dims = [_dims(t) for t in tensors]
        apart = all(map(_own_places, dims)) and all(_apart(dims[i], dims[j], (tensors[j].data_ptr() - tensors[i].data_ptr()) // 2)
                                                    for i in range(len(dims)) for j in range(i + 1, len(dims)))
        # (what the C interface is told of the cache, once: 13 arguments fewer in each call)
        struct = _hip.PagedCacheStruct(*_hip.t3(keys), *_hip.t3(values), None if bounds is None else bounds.data_ptr(), n_pages, kv_heads, page_size, d,
                                       _hip.dtype_code(keys))
        addresses = (keys.data_ptr, values.data_ptr, int if bounds is None else bounds.data_ptr)
        for name, value in zip(self.__slots__, (keys, values, bounds, weights, keys.dtype, keys.device, keys.get_device(), n_pages, kv_heads, page_size, d, struct,
                                                ctypes.addressof(struct), addresses, tuple(f() for f in addresses), apart,
                                                # (what the struct points to lives as long as the cache, also if a tensor is given other memory)
                                                tuple(t.detach() for t in (*tensors, *(() if weights is None else (weights,)))),
                                                0 if weights is None else weights.data_ptr())):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"a PagedCache does not change: {name}")

    def __reduce__(self):
        return PagedCache, (self.keys, self.values, self.bounds, self.weights)

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, dtype=torch.bfloat16, device="cuda", bounds: bool = True, weights: bool = False):
        """A cache with new memory, whose contents are undefined until they are appended."""
        keys, values = (torch.empty(n_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        return cls(keys, values, torch.empty(n_pages, n_kv_heads, 2, head_dim, dtype=dtype, device=device) if bounds else None,
                   torch.empty(n_pages, n_kv_heads, page_size, dtype=torch.float32, device=device) if weights else None)

    def _tables(self, page_table, lengths):
        """Arguments of a page table and lengths, and the sequences and most pages they are for."""
        lengths_ptr = _indices(lengths, "lengths", self, 1)
        batch = lengths.shape[0]
        table = _indices(page_table, "page_table", self, 2, batch)
        most = page_table.shape[1]
        if batch > 65535 or not most or most * self.page_size > 1 << 20:
            _refuse(f"{batch} sequences of up to {most} pages of {self.page_size} are not supported (at most 65535 sequences, 1048576 keys, at least one page)")
        return (table, page_table.stride(0), lengths_ptr), batch, most

    def _weighed(self):
        """``data_ptr`` of the weights; 0 without."""
        if self.weights is not None and self.weights.data_ptr() != self._weights:
            _refuse("a tensor of the cache has been given other memory, which a PagedCache does not follow: make a new one")
        return self._weights

    def _launch(self, fn, *packed):
        keys, values, bounds = self._addresses
        if (keys(), values(), bounds()) != self._pointers:
            _refuse("a tensor of the cache has been given other memory, which a PagedCache does not follow: make a new one")
        if self.index == torch.cuda.current_device():
            rc = fn(self._address, *packed, _raw_stream(self.index) if _raw_stream is not None else _stream())
        else:
            with torch.cuda.device(self.device):
                rc = fn(self._address, *packed, _stream())
        if rc:
            _hip.check(rc)


def _plain(cache, *tensors):
    if type(cache) is not PagedCache:
        _refuse("the first argument must be a PagedCache")
    if not _called_plainly():
        _refuse("these operators cannot be traced, compiled, vmapped or watched by a mode")
    if torch.is_grad_enabled():
        _without_gradients(*tensors)


def _without_gradients(*tensors):
    try:
        for t in tensors:
            if t is not None and t.requires_grad:
                _refuse("these operators have no gradients: detach their inputs or call them under torch.no_grad()")
    except AttributeError:
        pass  # (what is no tensor is refused where its type is looked at)


def append_to_pages(cache: PagedCache, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cos: Optional[torch.Tensor],
                    sin: Optional[torch.Tensor], page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, *, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                    positions: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Appends new tokens to the cache and returns their rotated queries (in ``out``, if it is given; that may be ``q`` and otherwise shares no memory with
    the inputs).

    ``q`` ``[tokens, query heads, D]``, ``k``, ``v`` ``[tokens, KV heads, D]``: the tokens of all sequences one after the other; sequence ``b`` has
    tokens ``starts[b]`` to ``starts[b + 1]`` (``[batch + 1]``, ascending; the first may lie below 0 and the last behind the
    tokens that are given; None: one token each).  ``lengths`` ``[batch]`` counts a sequence's keys
    **with** its new ones, which are its last; a token's place in the sequence is its position.  ``cos``, ``sin`` float32 ``[positions, D / 2]`` are the angles of all
    positions: channels ``d`` and ``d + D / 2`` are turned by the angle of ``d``, in float32 with one rounding.  Without them (and without
    queries) keys are stored as they are: those of a prompt that the model has rotated itself.

    Tokens without a place are left out - rows behind the last sequence, a length of 0, a position that ``cos`` or the table does not reach, a page
    outside the pool: their rows of ``out`` stay as they are (undefined in a new one).  Two sequences must not append to one page: the result is then one's or a mixture.
    ``k`` and ``v`` must not lie in the pages that are appended to.  A call has fewer than 2^23 rows of keys (tokens times KV heads).

    ``q_norm``, ``k_norm`` ``[D]`` of the cache's type (both, or ``k_norm`` where there are no queries): before it is rotated, each head ``x`` becomes
    ``x / sqrt(mean(x^2) + norm_eps) * weight``, in float32 with one rounding after both.  ``positions`` int32 ``[batch]``: how many positions a sequence has had, where
    that is more than its keys (:func:`evict_from_pages`): its last token is rotated by ``positions[b] - 1``; a sequence of fewer positions than keys is left out.
    ``k_out`` ``[tokens, KV heads, D]``, which may be ``k``: the keys as they are stored, for the prompt's own attention.  The weights of new keys, in a cache that keeps them, become 0."""
    _plain(cache, q, k, v, cos, sin, out)
    if not cache._apart:
        _refuse("keys, values and bounds that share memory cannot be appended to (parts of one tensor that lie between each other need the same strides)")
    k_args, (n, _, _) = _rows(k, "k", cache, cache.n_kv_heads)
    v_args, (n_values, _, _) = _rows(v, "v", cache, cache.n_kv_heads)
    tables, batch, most = cache._tables(page_table, lengths)
    starts_ptr = 0 if starts is None else _indices(starts, "starts", cache, 1, batch + 1)
    if n_values != n or (starts is None and n != batch) or n * cache.n_kv_heads >= 1 << 23:
        _refuse(f"{n} keys, {n_values} values and {batch} sequences{' without starts' if starts is None else ''} do not go together (and fewer than 2^23 rows of keys)")
    if cos is None:
        if sin is not None or q is not None or out is not None:
            _refuse("cos and sin come together, and queries need them")
        angles, n_positions, q_args, heads = (0, 0, 0), 0, (0,) * 6, 0
    else:
        try:
            strides = cos.stride()
        except AttributeError:
            strides = None
        for t in (cos, sin):
            if type(t) not in _TYPES or t.dtype != _FLOAT32 or t.get_device() != cache.index or t.dim() != 2 or t.shape != cos.shape or t.stride() != strides:
                _refuse("cos and sin must be float32 tensors [positions, D / 2] on the cache's device, laid out alike")
        n_positions, half = cos.shape
        angles = (cos.data_ptr(), sin.data_ptr(), strides[0])
        if half * 2 != cache.head_dim or not n_positions or strides[1] != 1 or strides[0] & 3 or strides[0] < half or (angles[0] | angles[1]) & 15:
            _refuse("the rows of cos and sin must hold D / 2 elements, contiguous on 16-byte boundaries")
        if q is None:
            if out is not None:
                _refuse("an output needs queries")
            q_args, heads = (0,) * 6, 0
        else:
            q_rows, shape = _rows(q, "q", cache, 0)
            heads = shape[1]
            if shape[0] != n:
                _refuse(f"q has {shape[0]} tokens, k {n}")
            q_args = (*q_rows, *_out_rows(out, shape, cache)) if out is not None else (*q_rows, *_new_rows(out := torch.empty_like(q)))
    more = None
    if cache._weights or q_norm is not None or k_norm is not None or positions is not None or k_out is not None:  # (a step without any does no more than look)
        if torch.is_grad_enabled():
            _without_gradients(q_norm, k_norm, k_out)
        if cos is None and not (k_norm is positions is k_out is None):
            _refuse("norms, positions and rotated keys need cos and sin")
        if (q_norm is None) != (k_norm is None or q is None):
            _refuse("norms of queries and keys come together, that of keys alone where there are no queries")
        norms = tuple(0 if t is None else _channels(t, name, cache) for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")))
        try:
            eps = float(norm_eps)
        except (TypeError, ValueError):
            eps = -1.0
        if not 0 <= eps <= 1:
            _refuse(f"norm_eps must be from 0 to 1, not {norm_eps}")
        more = _hip.PAGED_MORE.pack(*norms, *((0, 0, 0) if k_out is None else _out_rows(k_out, k.shape, cache, "k_out")),
                                    0 if positions is None else _indices(positions, "positions", cache, 1, batch), cache._weighed(), eps)
    if n and batch:
        tokens = _hip.PAGED_TOKENS.pack(*q_args, *k_args, *v_args, *angles, *tables, starts_ptr, n_positions, batch, n, heads, most)
        if more is None:
            cache._launch(_hip.lib().aa_paged_append, tokens)
        else:
            cache._launch(_hip.lib().aa_paged_append_more, tokens, more)
    return out


def _new_rows(t):
    st, sh, _ = t.stride()
    return t.data_ptr(), st, sh


def _channels(t, name, cache):
    """``data_ptr`` of a tensor ``[D]``."""
    if type(t) not in _TYPES or t.dtype != cache.dtype or t.get_device() != cache.index or t.shape != (cache.head_dim,) or t.stride() != (1,) or t.data_ptr() & 15:
        _refuse(f"{name} must be a contiguous tensor [head dimension] of the cache's type and device, on a 16-byte boundary")
    return t.data_ptr()


def _out_rows(out, shape, cache, name="out"):
    rows, out_shape = _rows(out, name, cache, shape[1])
    n, h, d = shape
    _, st, sh = rows
    if out_shape != shape or not (((h == 1 or sh >= d) and (n < 2 or st >= (h - 1) * sh + d)) or ((n < 2 or st >= d) and (h == 1 or sh >= (n - 1) * st + d))):
        _refuse(f"{name} must have the shape of {'q' if name == 'out' else 'k'}, and no two of its rows the same memory")
    return rows


def _decode_args(cache, q, page_table, lengths, sm_scale, out):
    _plain(cache, q, out)
    q_rows, shape = _rows(q, "q", cache, 0)
    tables, batch, most = cache._tables(page_table, lengths)
    if shape[0] != batch:
        _refuse(f"q has {shape[0]} tokens, the table {batch} sequences: a decode step has one of each")
    scale = cache.head_dim ** -0.5 if sm_scale is None else float(sm_scale)
    if not 1e-30 < scale < 1e30:
        _refuse(f"sm_scale must be positive, from 1e-30 to 1e30, not {sm_scale}")
    if out is not None:
        out_rows = _out_rows(out, shape, cache)
    else:
        out_rows = _new_rows(out := torch.empty_like(q))
    return out, (*q_rows, *out_rows, *tables), (batch, shape[1]), most, scale


def paged_decode_attention(cache: PagedCache, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, sm_scale: Optional[float] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, ``q`` ``[batch, query heads, D]``, over the first ``lengths[b]`` keys of each: ``softmax(q K^T
    sm_scale) V``, zeros for a sequence of none (NaN for one whose scores are all minus infinity).  ``sm_scale`` defaults to ``D ** -0.5``; ``out`` may be ``q`` and
    otherwise shares no memory with the inputs."""
    out, tensors, sizes, most, scale = _decode_args(cache, q, page_table, lengths, sm_scale, out)
    if sizes[0]:
        lib = _hip.lib()
        nbytes = lib.aa_paged_decode_workspace_bytes(*sizes, cache.n_kv_heads, cache.head_dim, cache.page_size, most)
        ws = lengths.new_empty((nbytes >> 2,)) if nbytes else None
        cache._launch(lib.aa_paged_decode_fwd, _hip.PAGED_STEP.pack(*tensors, ws.data_ptr() if nbytes else 0, nbytes, 0, *sizes, most, 0, 0, 0, scale))
    return out


def _whole(name, value):
    """A whole number that is given as any kind of number."""
    try:
        n = int(value)
    except (TypeError, ValueError, OverflowError):
        n = None
    if n is None or n != value:
        _refuse(f"{name} must be a whole number, not {value}")
    return n


def paged_weighing_decode_attention(cache: PagedCache, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, n_first: int = 0,
                                    sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`paged_decode_attention` that also counts how much attention each key has had: to ``cache.weights`` of key ``j`` of a sequence and KV head, from the
    ``n_first``-th key on, is added the sum over the heads of its group of ``softmax(q K^T sm_scale)[j]`` (NaN where the output is), in a fixed order.
    Two sequences must not share pages behind their first ``n_first`` keys.  Scratch: 4 bytes for each query head and key that the table has room for."""
    out, tensors, sizes, most, scale = _decode_args(cache, q, page_table, lengths, sm_scale, out)
    weights = cache._weighed()
    if not weights:
        _refuse("the weights of keys are counted in a cache that has them")
    n_first = _whole("n_first", n_first)
    if not 0 <= n_first < 1 << 31:
        _refuse(f"n_first must be from 0 to 2^31 - 1, not {n_first}")
    if sizes[0]:
        lib = _hip.lib()
        nbytes = lib.aa_paged_weighing_workspace_bytes(*sizes, cache.n_kv_heads, cache.head_dim, cache.page_size, most)
        ws = lengths.new_empty((nbytes >> 2,))
        cache._launch(lib.aa_paged_weighing_decode_fwd, _hip.PAGED_STEP.pack(*tensors, ws.data_ptr(), nbytes, 0, *sizes, most, 0, 0, 0, scale), weights, n_first)
    return out


def evict_from_pages(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, n_keys: int, n_first: int = 0, n_last: int = 1,
                     above: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cuts sequences of more than ``above`` keys (``n_keys`` if it is not given) down to ``n_keys``, for each KV head its own: the first ``n_first``, the last ``n_last``
    and, of those between, the ones with the largest ``cache.weights``, the lower place first among equals (as all keys are that no step has counted, a prompt's at first), NaN as infinity.  They become the
    sequence's first ``n_keys``, in order; their weights move along, and the bounds of pages that have other keys than before are formed anew.  What keeps its place is not
    written (pages that sequences share stay as they are if ``n_first`` counts their keys), nor are rows behind the last key.  Returns the sequences' new lengths, int32
    ``[batch]``, and the places that the keys had, int32 ``[batch, KV heads, n_keys]``, ascending (-1 for sequences of which nothing is given up).  The pages behind the new lengths are the program's again;
    tokens that are appended afterwards need ``positions``."""
    _plain(cache)
    weights = cache._weighed()
    if not weights:
        _refuse("keys are given up by their weights, which the cache must have")
    if not cache._apart:
        _refuse("keys, values and bounds that share memory cannot be moved")
    tables, batch, most = cache._tables(page_table, lengths)
    n_keys, n_first, n_last = _whole("n_keys", n_keys), _whole("n_first", n_first), _whole("n_last", n_last)
    above = n_keys if above is None else _whole("above", above)
    if n_first < 0 or n_last < 0 or not 0 < n_keys <= 1 << 20 or n_first + n_last > n_keys or not n_keys <= above < 1 << 31:
        _refuse(f"{n_keys} keys, the first {n_first} and the last {n_last} among them, of sequences of more than {above} are not supported (1 to 1048576)")
    if batch * cache.n_kv_heads >= 1 << 22:
        _refuse(f"{batch} sequences of {cache.n_kv_heads} KV heads are not supported (fewer than 2^22 together)")
    new_lengths, kept = lengths.new_empty((batch,)), lengths.new_empty((batch, cache.n_kv_heads, n_keys))
    if batch:
        lib = _hip.lib()
        nbytes = lib.aa_paged_evict_workspace_bytes(batch, cache.n_kv_heads, cache.head_dim, n_keys)
        ws = lengths.new_empty((nbytes >> 2,)) if nbytes else None
        cache._launch(lib.aa_paged_evict, _hip.PAGED_EVICTION.pack(*tables, new_lengths.data_ptr(), kept.data_ptr(), weights, ws.data_ptr() if nbytes else 0, nbytes, batch, most, n_keys,
                                                                   n_first, n_last, above))
    return new_lengths, kept


def paged_shared_decode_attention(cache: PagedCache, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, shared_pages: torch.Tensor,
                                  groups: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`paged_decode_attention` of sequences that begin with the same pages, which are read once for all of them.  Sequences ``groups[g]`` to
    ``groups[g + 1] - 1`` (``groups`` int32 ``[n_groups + 1]``, ascending; None: all sequences are one group) have the same first ``shared_pages[g]`` pages (int32 ``[n_groups]``) in their rows of
    the table; any of these rows may be what is read.  The first and last groups need not begin and end the batch: sequences in none, and those of fewer keys than their group's
    shared pages hold, are attended to by themselves.  Sequences append to pages of their own: only whole pages are shared.  A batch whose table has room for 256 MB of keys and values at most (340 with heads of 128) reads the shared pages once for each sequence, which is
    less time, since they stay in the caches."""
    out, tensors, sizes, most, scale = _decode_args(cache, q, page_table, lengths, sm_scale, out)
    shared_ptr = _indices(shared_pages, "shared_pages", cache, 1)
    n_groups = shared_pages.shape[0]
    if not 0 < n_groups <= 65535:
        _refuse(f"{n_groups} groups are not supported (1 to 65535)")
    if groups is None and n_groups != 1:
        _refuse(f"{n_groups} groups of sequences need to be told where they begin")
    groups_ptr = 0 if groups is None else _indices(groups, "groups", cache, 1, n_groups + 1)
    if sizes[0]:
        lib = _hip.lib()
        nbytes = lib.aa_paged_shared_workspace_bytes(*sizes, cache.n_kv_heads, cache.head_dim, cache.page_size, most, n_groups)
        ws = lengths.new_empty((nbytes >> 2,))
        cache._launch(lib.aa_paged_shared_decode_fwd, _hip.PAGED_STEP.pack(*tensors, ws.data_ptr(), nbytes, 0, *sizes, most, 0, 0, 0, scale), shared_ptr, groups_ptr, n_groups)
    return out


def paged_sparse_decode_attention(cache: PagedCache, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, n_pages: int, n_first: int = 1,
                                  n_last: int = 1, sm_scale: Optional[float] = None,
                                  out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`paged_decode_attention` over ``n_pages`` pages of each sequence and KV head (all where there are no more): the first ``n_first``, the last
    ``n_last`` and, of those between, the ones whose score is largest, the lower page first among equals.  The score of a page is the largest
    over the heads of the group of ``sum_d max over the page's bounds of q_d * x_d``: no key of the page has a larger product with the query.
    The products are exact, summed in float64 (in any order) and rounded to float32; NaN counts as infinity.  Returns the output and the chosen pages, int32 ``[batch, KV heads,
    n_pages]``: places in the sequence's row of the table, ascending, then -1.  The cache needs ``bounds``."""
    out, tensors, sizes, most, scale = _decode_args(cache, q, page_table, lengths, sm_scale, out)
    if cache.bounds is None:
        _refuse("sparse steps need a cache with bounds")
    given = n_pages, n_first, n_last
    try:
        n_pages, n_first, n_last = whole = tuple(map(int, given))
    except (TypeError, ValueError, OverflowError):
        whole = None
    if whole != given:
        _refuse("n_pages, n_first and n_last must be whole numbers, not %s, %s and %s" % given)
    if n_first < 0 or n_last < 1 or n_first + n_last > n_pages or n_pages > 1 << 16:
        _refuse(f"{n_pages} pages, the first {n_first} and the last {n_last} among them, are not supported (at most 65536, at least the last one)")
    pages = lengths.new_empty((sizes[0], cache.n_kv_heads, n_pages))
    if sizes[0]:
        lib = _hip.lib()
        nbytes = lib.aa_paged_sparse_workspace_bytes(*sizes, cache.n_kv_heads, cache.head_dim, cache.page_size, most, n_pages)
        ws = lengths.new_empty((nbytes >> 2,))
        cache._launch(lib.aa_paged_sparse_decode_fwd,
                      _hip.PAGED_STEP.pack(*tensors, ws.data_ptr(), nbytes, pages.data_ptr(), *sizes, most, n_pages, n_first, n_last, scale))
    return out, pages
