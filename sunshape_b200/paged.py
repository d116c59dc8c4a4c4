"""Paged compressed cache: what a serving engine calls around the quantized-key decode path.

* ``norm_rotate``: per-head RMS norms of queries and keys with the rotary position embedding, one launch;
* ``SunShapePagedCache``: one layer's pool of pages -- codeword indices ``[num_pages, kv_heads, page_size,
  n_blocks]`` uint8, values ``[num_pages, kv_heads, page_size, value_dim]`` and, for SunShape-Mixed codecs,
  dense key blocks ``[num_pages, kv_heads, page_size, n_heavy, block_dim]``.  The engine owns the page
  allocator: it hands out page numbers and names them in page tables and slots;
* ``append_paged``: rotates, permutes and encodes new keys and copies new values into token slots, one launch
  for a decode step's single tokens as for whole prompts;
* ``paged_attention``: decode attention over the pages of a ragged batch, optionally behind a prefix of pages
  that all sequences share and whose attention is computed once for all of them.

Counterpart for contiguous caches: ``codec.quantize_packed`` and ``vllm_attn_backend``.  16-bit keys and values
only (bf16, f16); ``norm_rotate`` also takes fp32.  Every call runs on the current stream of its tensors' device,
takes no workspace that outlives it and can be captured into a CUDA graph; tensors used on another stream than
the one they were made on need the usual ``record_stream``.  What only the device can see is checked there: a
position, slot, page, length or dense key out of range is skipped (or makes the row NaN) and recorded, see
``paged_error``.
Nothing here is differentiable: inputs that require gradients are refused where gradients are recorded.
"""
from __future__ import annotations

import ctypes
import math
import threading

import torch

from . import _lib
from .codec import SunShapeBlockCodec

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ERRORS = {131: "a position is outside the cosine/sine table", 132: "a slot is outside the page pool",
           133: "a page number is outside the page pool", 134: "a sequence is longer than its page table",
           135: "a pipeline wait gave up", 136: "a dense key block does not fit into fp16"}


def paged_error(device: torch.device | str | None = None, clear: bool = True) -> str | None:
    """What the paged kernels recorded on ``device`` since the last clear (None: nothing).  Waits for all of the
    device's streams; not to be called while one is captured."""
    code = ctypes.c_int32(0)
    dev = torch.device("cuda" if device is None else device)
    with torch.cuda.device(dev):
        _lib._check(_lib.load_library().sunshape_paged_error(ctypes.byref(code), 1 if clear else 0))
    return _ERRORS.get(code.value, f"error {code.value}") if code.value else None


def rotary_table(n_positions: int, rot_dim: int, *, base: float = 10000.0,
                 device: torch.device | str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin ``[n_positions, rot_dim / 2]`` fp32 of the angles ``p * base^(-2i / rot_dim)``, computed in 64 bits
    (at position 10^5 an fp32 angle is already off by 4e-3)."""
    inv = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / max(rot_dim, 1))
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


# ------------------------------------------------------------------------------------------- argument checks
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _device(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """Index of the CUDA device that all of the tensors are on."""
    dev = first.get_device()
    same = dev >= 0
    for t in others:
        same = same and (t is None or t.get_device() == dev)
    if not same:
        _lib.require_cuda(first, *others)     # says what is wrong
    return dev


def _forward_only() -> None:
    """For a call with an input that requires gradients."""
    if torch.is_grad_enabled():
        raise RuntimeError("the paged calls have no backward pass: call them under torch.no_grad() or "
                           "torch.inference_mode(), or detach their inputs.")


def _unit(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise RuntimeError(f"{what}: the last axis must have unit stride.")
    return t


def _rotation(cos, sin, positions, interleaved, B: int, L: int, dim: int, dev: int) -> bytes | None:
    if cos is None and sin is None and positions is None:
        return None
    if cos is None or sin is None or positions is None:
        raise RuntimeError("a rotation needs cos, sin and positions.")
    shape = cos.shape
    if len(shape) != 2 or shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise RuntimeError("cos and sin must be fp32 tables of one shape [n_positions, rot_dim / 2].")
    if 2 * shape[1] > dim:
        raise RuntimeError(f"cos and sin rotate {2 * shape[1]} elements of a head of {dim}.")
    if positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("positions must be int32 or int64.")
    if not cos.get_device() == sin.get_device() == positions.get_device() == dev:
        raise RuntimeError("all sunshape_b200 inputs must live on the same CUDA device.")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise RuntimeError("cos and sin must be contiguous.")
    sb, sl = _token_strides(positions, B, L, "positions")
    return _lib.rotation(cos, sin, positions, sb, sl, interleaved)


def _token_strides(t: torch.Tensor, B: int, L: int, what: str) -> tuple[int, int]:
    """Strides of a [B, L] tensor, or of one that broadcasts to it: [L], [1, L], [B, 1]."""
    if t.ndim == 1 and t.shape[0] == L:
        return 0, t.stride(0)
    if t.ndim == 2 and t.shape[0] in (1, B) and t.shape[1] in (1, L):
        return (t.stride(0) if t.shape[0] == B else 0), (t.stride(1) if t.shape[1] == L else 0)
    raise RuntimeError(f"{what} must have shape [batch, length] (or broadcast to it), got {list(t.shape)}.")


# ----------------------------------------------------------------------------------------- norms and rotation
def norm_rotate(query: torch.Tensor, key: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                k_weight: torch.Tensor | None = None, eps: float = 1e-6, cos: torch.Tensor | None = None,
                sin: torch.Tensor | None = None, positions: torch.Tensor | None = None, interleaved: bool = False,
                out: tuple[torch.Tensor, torch.Tensor | None] | None = None):
    """RMS norm of each query and key head, then the rotary embedding, in one launch: ``(query', key')``.

    ``query`` [B, q_heads, L, D] and ``key`` [B, kv_heads, L, D] (or None) of one dtype, any strides with a unit
    last one (views of a fused projection's output are read in place).  A weight [D] turns that tensor's norm on:
    ``x * w / sqrt(mean(x^2) + eps)``.  ``cos``/``sin`` [n_positions, R / 2] fp32 and ``positions`` [B, L] (int32 or
    int64; [L] broadcasts) rotate the first R <= D elements: pairs (i, i + R/2), or (2i, 2i + 1) if
    ``interleaved``.  fp32 arithmetic, one rounding to the inputs' dtype.  ``out`` may be the inputs themselves, each
    over its own; any other overlap of the tensors gives wrong results."""
    if (query.requires_grad or (key is not None and key.requires_grad) or (q_weight is not None and q_weight.requires_grad)
            or (k_weight is not None and k_weight.requires_grad)):
        _forward_only()
    dev = _device(query, key, q_weight, k_weight)
    code = _CODES.get(query.dtype)
    if query.ndim != 4 or (key is not None and key.ndim != 4):
        raise RuntimeError("norm_rotate expects query and key with shape [batch, heads, seq, dim].")
    if code is None:
        raise RuntimeError(f"norm_rotate takes fp32, bf16 or f16 rows, got {query.dtype}.")
    B, Hq, L, D = query.shape
    if key is not None:
        Bk, _, Lk, Dk = key.shape
        if key.dtype != query.dtype or (Bk, Lk, Dk) != (B, L, D):
            raise RuntimeError("query and key must agree in dtype, batch, length and head dimension.")
        _unit(key, "key")
    elif k_weight is not None:
        raise RuntimeError("k_weight without a key.")
    _unit(query, "query")
    for w in (q_weight, k_weight):
        if w is not None and (w.ndim != 1 or w.shape[0] != D or w.dtype not in _CODES or not w.is_contiguous()):
            raise RuntimeError(f"norm weights must be contiguous fp32, bf16 or f16 tensors of shape [{D}].")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise RuntimeError("both norm weights must have one dtype.")
    rot = _rotation(cos, sin, positions, interleaved, B, L, D, dev)
    if out is None:
        q_out, k_out = torch.empty_like(query), (None if key is None else torch.empty_like(key))
    else:
        q_out, k_out = out
        for t, o in ((query, q_out), (key, k_out)):
            if (t is None) != (o is None) or (t is not None and (
                    o.shape != t.shape or o.dtype != t.dtype or o.get_device() != dev)):
                raise RuntimeError("out must hold tensors of the inputs' shapes, dtype and device.")
            if t is not None and o.data_ptr() == t.data_ptr() and o.stride() != t.stride():
                raise RuntimeError("out over its own input needs the input's strides.")
            if t is not None:
                _unit(o, "out")
                if 0 in o.stride() and any(n > 1 and st == 0 for n, st in zip(o.shape, o.stride())):
                    raise RuntimeError("out must not hold an element twice.")
        if key is not None:
            at, k_at = q_out.data_ptr(), k_out.data_ptr()
            if at and (at == key.data_ptr() or at == k_at) or k_at and k_at == query.data_ptr():
                raise RuntimeError("out must not be another tensor's input or output.")
    w = q_weight if q_weight is not None else k_weight
    _lib.norm_rotate(dev, _lib.rows(query), _lib.rows(q_out), q_weight, None if key is None else _lib.rows(key),
                     None if key is None else _lib.rows(k_out), k_weight, code, _lib.F32 if w is None else _CODES[w.dtype],
                     B, L, D, eps, rot)
    return q_out, k_out


# ----------------------------------------------------------------------------------------- what a codec amounts to
class _CodecTables:
    """What the paged kernels read of a codec: tables derived from its codebooks, its permutation and its dense blocks'
    mask, in one buffer per tensor that the codec keeps.  They are renewed in place, so that captured graphs, which hold
    their addresses, see what the codec holds."""

    def __init__(self, key: tuple, desc: _lib.CodecDesc):
        self.key, self.desc, self.made, self.streams = key, None, None, set()
        device, _, n_heavy = key
        self.device, self.index, self.n_heavy = device, device.index, n_heavy
        self.buffer = torch.empty(_lib.paged_tables_bytes(desc), dtype=torch.uint8, device=device)
        self.perm = torch.empty(desc.head_dim, dtype=torch.int64, device=device)
        self.mask = torch.empty(desc.head_dim // desc.block_dim, dtype=torch.uint8, device=device) if n_heavy else None

    def fill(self, made: tuple) -> None:
        desc, (cents, perm, mask, _), _ = made
        self.perm.copy_(perm)
        if mask is not None:
            self.mask.copy_(mask)
        _lib.paged_tables(desc, self.buffer)
        # the kernels read no centroids of the descriptor, only the tables
        self.desc = _lib.codec_desc(cents, self.perm, self.mask, self.n_heavy, desc.head_dim, desc.block_dim)

    def used_on(self, stream: int) -> None:
        """Keeps the buffers from the allocator until what runs on this stream is done, once they are given up."""
        for t in (self.buffer, self.perm, self.mask):
            if t is not None:
                t.record_stream(torch.cuda.current_stream(self.device))
        self.streams.add(stream)


_renewing = threading.Lock()


def renew_tables(codec: SunShapeBlockCodec) -> _CodecTables:
    """Derives a codec's tables again.  Waits for the device on both sides: edits of the codec's buffers and readers of the
    tables, on whatever stream, come before; every later reader finds them written."""
    device = _lib.require_cuda(codec.centroids)
    # the buffers outlive an inference mode that they happen to be made in, and are written again outside it
    with _renewing, torch.cuda.device(device), torch.inference_mode(False), torch.no_grad():
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a codec's tables can not be derived while a CUDA graph is captured: make the cache, and call "
                               "codec.invalidate() after edits of the codec, before the capture.")
        tables = codec._paged_tables
        if tables is not None and tables.made is codec._desc_cache:      # another thread was faster
            return tables
        torch.cuda.synchronize()
        made = codec.kernel_desc()
        desc, (cents, *_), n_heavy = made
        key = (device, tuple(cents.shape), n_heavy)
        if tables is None or tables.key != key:
            if tables is not None:              # graphs captured with them may still be replayed
                codec._paged_retired = (*codec._paged_retired, tables)
            tables = _CodecTables(key, desc)
        tables.fill(made)
        torch.cuda.synchronize()
        tables.made = made
        codec._paged_tables = tables
    return tables


def renew_after_edit(codec: SunShapeBlockCodec) -> None:
    """Renews the tables of a codec that still has the shape they were made for; else the next call does, or says why not."""
    device, shape, _ = codec._paged_tables.key
    cents = codec.centroids
    if cents.device == device and tuple(cents.shape)[-3:] == shape[-3:] and codec.n_codebooks == shape[0]:
        with torch.cuda.device(device):
            capturing = torch.cuda.is_current_stream_capturing()
        if not capturing and codec.mode not in ("rotated", "legacy_strict"):
            renew_tables(codec)


# ---------------------------------------------------------------------------------------------------- the cache
class SunShapePagedCache:
    """One layer's page pool and the codec of its keys.  ``allocate`` makes the pool, ``from_pools`` takes one."""

    def __init__(self, codec: SunShapeBlockCodec, indices: torch.Tensor, values: torch.Tensor,
                 heavy: torch.Tensor | None = None):
        dev = _lib.require_cuda(indices, values, heavy)
        desc, keep, n_heavy = codec.kernel_desc()
        if keep[0].device != dev:
            raise RuntimeError("the codec and its page pools must live on the same CUDA device.")
        if codec.block_dim not in (2, 4, 8) or codec.n_centroids > 256:
            raise RuntimeError("the paged cache takes block_dim 2, 4 or 8 and at most 256 codewords a block.")
        if indices.ndim != 4 or indices.dtype != torch.uint8 or indices.shape[3] != codec.n_blocks:
            raise RuntimeError("indices must be uint8 [num_pages, kv_heads, page_size, n_blocks].")
        if values.ndim != 4 or values.shape[:3] != indices.shape[:3] or values.dtype not in _FLOATS[1:]:
            raise RuntimeError("values must be bf16 or f16 [num_pages, kv_heads, page_size, value_dim].")
        if n_heavy:
            if heavy is None or heavy.dtype != values.dtype or heavy.shape != (
                    *indices.shape[:3], n_heavy, codec.block_dim):
                raise RuntimeError("a codec with dense blocks needs heavy [num_pages, kv_heads, page_size, n_heavy, "
                                   "block_dim] of the values' dtype.")
        elif heavy is not None:
            raise RuntimeError("heavy pool given, but the codec has no dense blocks.")
        if indices.shape[2] < 16 or indices.shape[2] % 16:
            raise RuntimeError("page_size must be a multiple of 16.")
        if values.shape[3] % 8:
            raise RuntimeError("value_dim must be a multiple of 8.")
        if codec.n_codebooks not in (1, indices.shape[1]):
            raise RuntimeError(f"codec holds {codec.n_codebooks} codebooks for {indices.shape[1]} KV heads.")
        for t in (indices, values, heavy):
            if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
                raise RuntimeError("page pools must be contiguous and 16-byte aligned.")
        self.codec, self.indices, self.values, self.heavy = codec, indices, values, heavy
        self.device, self._index = dev, indices.get_device()
        self._n_heavy, self._held = n_heavy, None
        self._pages = _lib.PagesDesc(_lib.ptr(indices), _lib.ptr(heavy), _lib.ptr(values), indices.shape[0],
                                     indices.shape[1], indices.shape[2], values.shape[3], _lib.dtype_code(values))
        self._tables()

    @classmethod
    def from_pools(cls, codec, indices, values, heavy=None) -> "SunShapePagedCache":
        return cls(codec, indices, values, heavy)

    @classmethod
    def allocate(cls, codec: SunShapeBlockCodec, num_pages: int, kv_heads: int, *, page_size: int = 64,
                 value_dim: int | None = None, dtype: torch.dtype = torch.bfloat16) -> "SunShapePagedCache":
        """Zeroed pools of ``num_pages`` pages on the codec's device."""
        dev, shape = codec.centroids.device, (num_pages, kv_heads, page_size)
        n_heavy = codec.kernel_desc()[2]
        return cls(codec, torch.zeros(*shape, codec.n_blocks, dtype=torch.uint8, device=dev),
                   torch.zeros(*shape, value_dim or codec.head_dim, dtype=dtype, device=dev),
                   torch.zeros(*shape, n_heavy, codec.block_dim, dtype=dtype, device=dev) if n_heavy else None)

    num_pages = property(lambda self: int(self.indices.shape[0]))
    kv_heads = property(lambda self: int(self.indices.shape[1]))
    page_size = property(lambda self: int(self.indices.shape[2]))
    value_dim = property(lambda self: int(self.values.shape[3]))
    dtype = property(lambda self: self.values.dtype)

    def _tables(self) -> _CodecTables:
        """The codec's tables, derived once and renewed after ``invalidate``, for calls on the current stream."""
        codec = self.codec
        tables = codec._paged_tables
        if tables is None or tables.made is not codec._desc_cache:   # a descriptor of its own after each ``invalidate``
            tables = renew_tables(codec)
        if tables is not self._held:
            if (tables.n_heavy != self._n_heavy or tables.index != self._index
                    or tables.desc.n_cb not in (1, self.indices.shape[1])):
                raise RuntimeError("the codec's codebooks, dense blocks or device are not those that the page pools were made "
                                   "for.")
            self._held = tables
        stream = torch._C._cuda_getCurrentRawStream(self._index)
        if stream not in tables.streams:
            tables.used_on(stream)
        return tables

    def slots(self, page_table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """Slots [B, L] of the token positions [B, L] (within their sequences) under ``page_table`` [B, cols]; -1
        where a position is negative, a slot outside the pool (which ``append_paged`` records) beyond the table and where
        the table names no page."""
        cols, outside = page_table.shape[1], self.num_pages * self.page_size
        p = positions.long()
        s = p.new_full(p.shape, outside)
        if cols:
            page = page_table.long().gather(1, (p // self.page_size).clamp(0, cols - 1))
            s = torch.where((p < cols * self.page_size) & (page >= 0), page * self.page_size + p % self.page_size, s)
        return torch.where(p >= 0, s, -1)

    def append(self, key, value, slots, **rotation) -> None:
        append_paged(self, key, value, slots, **rotation)

    def attention(self, query, page_table, seq_lens, **kw) -> torch.Tensor:
        return paged_attention(self, query, page_table, seq_lens, **kw)


def append_paged(cache: SunShapePagedCache, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, *,
                 cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, interleaved: bool = False) -> None:
    """Write new tokens into their slots: keys rotated (with ``cos``, ``sin`` and ``positions`` as in
    ``norm_rotate``), permuted and encoded, values copied.

    ``key`` [B, kv_heads, L, D] and ``value`` [B, kv_heads, L, value_dim] of the cache's dtype, any strides with a unit
    last one; ``slots`` [B, L] int64, ``page * page_size + row``, -1 for rows to leave out (padding).  A flat
    ragged batch [N, kv_heads, D] is ``key.transpose(0, 1).unsqueeze(0)`` with slots [1, N].  Slots of one call
    must be distinct.  The codeword is the nearest to the rotated key in real arithmetic (decided in 64 bits
    where fp32 cannot tell; lowest index on ties), without rounding the rotated key in between."""
    if key.requires_grad or value.requires_grad:
        _forward_only()
    codec = cache.codec
    dev = _device(key, value, slots)
    if dev != cache._index:
        raise RuntimeError("all sunshape_b200 inputs must live on the same CUDA device.")
    if codec.is_metric:
        raise RuntimeError("append_paged does not encode under a SunShape-Pro metric; encode with "
                           "codec.quantize_packed and copy the indices into the pages.")
    if key.ndim != 4 or value.ndim != 4:
        raise RuntimeError("append_paged expects key and value with shape [batch, kv_heads, seq, dim].")
    B, H, L, D = key.shape
    pages = cache._pages
    if D != codec.head_dim:
        raise RuntimeError("Key head_dim does not match codec head_dim.")
    if H != pages.kv_heads or tuple(value.shape) != (B, H, L, pages.value_dim):
        raise RuntimeError("key and value must agree with each other and with the cache's kv_heads and value_dim.")
    dtype = cache.values.dtype
    if key.dtype != dtype or value.dtype != dtype:
        raise RuntimeError(f"key and value must have the cache's dtype {dtype}.")
    if slots.dtype != torch.int64 or tuple(slots.shape) != (B, L):
        raise RuntimeError("slots must be int64 [batch, length].")
    rot = _rotation(cos, sin, positions, interleaved, B, L, D, dev)
    tables = cache._tables()
    _lib.paged_append(dev, tables.desc, tables.buffer, pages, _lib.rows(_unit(key, "key")), _lib.rows(_unit(value, "value")),
                      B, L, slots, rot)


def paged_attention(cache: SunShapePagedCache, query: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                    prefix_table: torch.Tensor | None = None, prefix_len: int = 0, scale: float | None = None,
                    causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``query`` [B, q_heads, L, D] over a paged cache: [B, q_heads, L, value_dim].

    Sequence b's own tokens are the first ``seq_lens[b]`` rows of the pages ``page_table[b]`` ([B, cols] and [B], int32,
    on the device: lengths never visit the host).  With ``prefix_table`` [n] int32 and ``prefix_len``, the first
    ``prefix_len`` tokens of those pages come before every sequence's own, and are read and attended to once for
    the whole batch.  The last L tokens of a sequence are the queries' own: query l sees all but the last L - 1 -
    l of them, unless ``causal`` is false.  A row that sees nothing is zero.  ``scale`` defaults to 1 / sqrt(D).  ``out``
    must be contiguous and begin at a multiple of 8 bytes.

    Softmax statistics and sums are fp32.  Codewords are read as fp16 and softmax weights rounded to the cache's
    dtype before they multiply values; a codebook and a query row are each scaled by a power of two into fp16's range, and
    what is below 2^-25 of their largest is read as zero.  Dense key elements of bf16 must stay below 65504, or
    that many times the largest codeword's norm where that is above 1: a larger one is recorded and makes the rows NaN that
    see it."""
    if query.requires_grad:
        _forward_only()
    codec, pages = cache.codec, cache._pages
    dev = _device(query, page_table, seq_lens, prefix_table)
    if dev != cache._index:
        raise RuntimeError("all sunshape_b200 inputs must live on the same CUDA device.")
    if query.ndim != 4:
        raise RuntimeError("paged_attention expects query with shape [batch, heads, seq, dim].")
    B, Hq, L, D = query.shape
    if D != codec.head_dim:
        raise RuntimeError("Query head_dim does not match codec head_dim.")
    if Hq % pages.kv_heads:
        raise RuntimeError("Query head count must be divisible by kv-head count.")
    dtype = query.dtype
    if dtype != cache.values.dtype:
        raise RuntimeError(f"query must have the cache's dtype {cache.dtype}.")
    _unit(query, "query")
    if page_table.ndim != 2 or page_table.shape[0] != B or page_table.dtype != torch.int32:
        raise RuntimeError("page_table must be int32 [batch, pages].")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise RuntimeError("page_table: the last axis must have unit stride.")
    if seq_lens.ndim != 1 or seq_lens.shape[0] != B or seq_lens.dtype != torch.int32 or not seq_lens.is_contiguous():
        raise RuntimeError("seq_lens must be contiguous int32 [batch].")
    prefix_len = int(prefix_len)
    if prefix_len < 0 or (prefix_len and prefix_table is None):
        raise RuntimeError("prefix_len needs a prefix_table and must not be negative.")
    if prefix_len and (prefix_table.ndim != 1 or prefix_table.dtype != torch.int32 or not prefix_table.is_contiguous()
                       or prefix_table.shape[0] * pages.page_size < prefix_len):
        raise RuntimeError("prefix_table must be contiguous int32 [pages] and hold prefix_len tokens.")
    shape = (B, Hq, L, pages.value_dim)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=query.device)
    elif tuple(out.shape) != shape or out.dtype != dtype or out.get_device() != dev or not out.is_contiguous():
        raise RuntimeError("out must be contiguous [batch, q_heads, query_len, value_dim] of the query's dtype.")
    tables = cache._tables()
    _lib.paged_attention(dev, tables.desc, tables.buffer, pages, query, B, Hq, L, page_table, seq_lens,
                         prefix_table if prefix_len else None, prefix_len, 1.0 / math.sqrt(D) if scale is None else float(scale),
                         causal, out)
    return out


__all__ = ["SunShapePagedCache", "norm_rotate", "append_paged", "paged_attention", "paged_error", "rotary_table"]
