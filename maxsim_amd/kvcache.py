"""A reader model's key/value cache in the corpus' 4-bit row format, and attention over it.

What answers over the passages that a search found keeps a key and a value per
token and head.  ``Int4KVCache`` keeps them as the corpus keeps token
embeddings (``pack_int4_symmetric(..., scale_granularity="token")``): one
single precision scale per row, ``max|x| / 7``, and codes in [-7, 7], two to a
byte -- ``head_dim / 2 + 4`` bytes instead of ``2 * head_dim``.

The cache is a pool of pages.  Which pages a sequence holds, and how many
tokens, is the caller's to say, on the device: ``page_table`` int32
[batch, max_pages] and ``lengths`` int32 [batch].  The rows of a call are
packed, and are the last ones of their sequences: sequence b has rows
``offsets[b]`` to ``offsets[b + 1]`` (int32 [batch + 1]; without offsets one
row each), and ``lengths[b]`` counts them already.  So one decoding step of an
attention layer is::

    cache.append(k, v, page_table, lengths)
    out = cache.attend(q, page_table, lengths)

Every call enqueues its work on the current stream and returns; none copies
anything to the host, and none records gradients.  Indices on the device are
not visible to the checks here: lengths are cut to the table, and a page
number outside the pool is a hole (not written, read back as zeros, taking no
attention).  ``append`` and ``attend`` can be captured in a HIP graph.
"""
from __future__ import annotations

import ctypes
import math

from maxsim_amd import _native

HEAD_DIMS = (64, 96, 128, 192, 256)


_TYPES: dict = {}  # torch dtype -> type number of the C ABI, once torch is there


def _type_of(dtype) -> int:
    if not _TYPES:
        import torch

        _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    return kind


def _cuda_device(device):
    import torch

    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("device must be 'cuda'")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return device


def _launch(device, call, *args) -> None:
    """Calls the C ABI with the current stream of `device` as the last argument,
    that device being current."""
    import torch

    index = device.index
    if torch._C._cuda_getDevice() == index:
        status = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _native.check(status)


class Int4KVCache:
    """Keys and values of one attention layer in pages of 4-bit rows.

    num_pages, kv_heads, head_dim (64, 96, 128, 192 or 256) and page_size (a
    power of two from 16 up) shape the pool.  ``k_codes`` / ``v_codes`` u8
    [num_pages, kv_heads, page_size, head_dim / 2] and ``k_scales`` /
    ``v_scales`` f32 [num_pages, kv_heads, page_size] are the pool itself: a
    program saves, moves or restores pages through them.
    """

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        import torch

        num_pages, kv_heads, head_dim, page_size = int(num_pages), int(kv_heads), int(head_dim), int(page_size)
        if num_pages < 1:
            raise ValueError("num_pages must be positive")
        if not 1 <= kv_heads <= 1024:
            raise ValueError("kv_heads must be between 1 and 1024")
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError("head_dim must be 64, 96, 128, 192 or 256")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 65536")
        self.device = _cuda_device(device)
        self._lib = _native.load()
        self._tensor, self._int32 = torch.Tensor, torch.int32
        self._workspaces = {}  # bytes of attend's workspace by its sizes
        shape = (num_pages, kv_heads, page_size)
        self._k_codes, self._v_codes = (torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=self.device)
                                        for _ in range(2))
        self._k_scales, self._v_scales = (torch.zeros(shape, dtype=torch.float32, device=self.device)
                                          for _ in range(2))
        self.num_pages, self.kv_heads, self.head_dim, self.page_size = num_pages, kv_heads, head_dim, page_size
        self._pool = _native.Kv4Pool(self._k_codes.data_ptr(), self._k_scales.data_ptr(), self._v_codes.data_ptr(),
                                     self._v_scales.data_ptr(), num_pages, kv_heads, page_size, head_dim)
        self._pool_ptr = ctypes.addressof(self._pool)

    @property
    def k_codes(self):
        return self._k_codes

    @property
    def v_codes(self):
        return self._v_codes

    @property
    def k_scales(self):
        return self._k_scales

    @property
    def v_scales(self):
        return self._v_scales

    @property
    def resident_bytes(self) -> int:
        """Bytes of the pool."""
        return sum(t.numel() * t.element_size() for t in (self._k_codes, self._v_codes, self._k_scales,
                                                          self._v_scales))

    # ------------------------------------------------------------- arguments

    def _batch(self, page_table, lengths, offsets, rows):
        """(table, lengths, offsets, batch, max_pages, rows) for the C ABI; the
        int32 tensors must be dense."""
        self._index("page_table", page_table, 2)
        self._index("lengths", lengths, 1)
        batch, max_pages = page_table.shape
        if lengths.shape[0] != batch:
            raise ValueError("lengths must have shape [batch]")
        if offsets is None:
            if rows != batch:
                raise ValueError("without offsets there must be one row per sequence")
            return page_table.data_ptr(), lengths.data_ptr(), None, batch, max_pages, rows
        self._index("offsets", offsets, 1)
        if offsets.shape[0] != batch + 1:
            raise ValueError("offsets must have shape [batch + 1]")
        return page_table.data_ptr(), lengths.data_ptr(), offsets.data_ptr(), batch, max_pages, rows

    def _index(self, name, t, ndim) -> None:
        if not isinstance(t, self._tensor) or t.dtype != self._int32 or t.ndim != ndim or t.device != self.device:
            raise ValueError(f"{name} must be an int32 tensor of {ndim} dimension{'s' * (ndim > 1)} on {self.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")

    def _rows(self, name, t, heads=None):
        """Checks rows [rows, heads, head_dim]: any strides, dims dense."""
        if not isinstance(t, self._tensor) or t.ndim != 3 or t.shape[2] != self.head_dim or \
                (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{name} must be a tensor of shape [rows, {heads or 'heads'}, {self.head_dim}]")
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        if t.stride(2) != 1 and t.numel() > 0:
            raise ValueError(f"{name} must be dense in its last dimension")
        return _type_of(t.dtype)

    # ----------------------------------------------------------------- calls

    def append(self, k, v, page_table, lengths, offsets=None) -> None:
        """Quantise keys and values [rows, kv_heads, head_dim] (float32, float16
        or bfloat16, any strides with dense rows) into the cache.  A row that
        holds an infinity or a NaN reads back as NaN."""
        kind = self._rows("k", k, self.kv_heads)
        if self._rows("v", v, self.kv_heads) != kind or v.shape[0] != k.shape[0]:
            raise ValueError("k and v must have the same shape and dtype")
        batch = self._batch(page_table, lengths, offsets, k.shape[0])
        _launch(self.device, self._lib.msim_kv4_append_async, self._pool_ptr, *batch, k.data_ptr(), *k.stride()[:2],
                v.data_ptr(), *v.stride()[:2], kind)

    def read(self, page_table, lengths, offsets=None, *, rows=None, dtype=None, out=None):
        """The rows (keys, values) [rows, kv_heads, head_dim] read back, each
        value code * scale rounded once to ``dtype`` (default bfloat16).  ``rows``
        is their number; without it, and with offsets, the last offset is fetched
        from the device.  ``out`` is a pair of tensors to write."""
        import torch

        if out is not None:
            k, v = out
            kind = self._rows("out[0]", k, self.kv_heads)
            if self._rows("out[1]", v, self.kv_heads) != kind or v.shape[0] != k.shape[0]:
                raise ValueError("both outputs must have the same shape and dtype")
            if (rows is not None and int(rows) != k.shape[0]) or (dtype is not None and dtype != k.dtype):
                raise ValueError("rows and dtype must be those of out")
        else:
            dtype = torch.bfloat16 if dtype is None else dtype
            kind = _type_of(dtype)
            if rows is None:
                if offsets is not None:
                    if not torch.is_tensor(offsets) or offsets.ndim != 1 or offsets.shape[0] < 1:
                        raise ValueError("offsets must have shape [batch + 1]")
                    rows = int(offsets[-1])
                else:
                    rows = lengths.shape[0]
            rows = int(rows)
            if rows < 0:
                raise ValueError("rows must not be negative")
            k, v = (torch.empty((rows, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
                    for _ in range(2))
        batch = self._batch(page_table, lengths, offsets, k.shape[0])
        _launch(self.device, self._lib.msim_kv4_read_async, self._pool_ptr, *batch, k.data_ptr(), *k.stride()[:2],
                v.data_ptr(), *v.stride()[:2], kind)
        return k, v

    def attend(self, q, page_table, lengths, offsets=None, *, scale=None, causal=True, window=None, mask=None,
               out=None, return_lse=False):
        """Attention of queries [rows, heads, head_dim] over their sequences.

        ``heads`` is a multiple of kv_heads; query head h reads key/value head
        ``h // (heads // kv_heads)``.  Row i of a sequence's n stands at position
        p = length - n + i and sees the keys j < length with j <= p (``causal``),
        j > p - window (``window``) and mask[row, j] (``mask`` bool
        [rows, width]; keys past its width are hidden).  ``scale`` defaults to
        head_dim ** -0.5.  Returns [rows, heads, head_dim] in q's dtype, rounded
        once from single precision sums, and with ``return_lse`` the logarithm
        of each softmax's sum, float32 [rows, heads].  A row that sees nothing
        is zeros, with minus infinity.
        """
        import torch

        kind = self._rows("q", q)
        rows, heads = q.shape[0], q.shape[1]
        if heads < 1 or heads % self.kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        batch = self._batch(page_table, lengths, offsets, rows)
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        if window is not None and int(window) < 1:
            raise ValueError("window must be positive")
        mask_args = (None, 0, 0)
        if mask is not None:
            if not torch.is_tensor(mask) or mask.dtype != torch.bool or mask.ndim != 2 or mask.shape[0] != rows or \
                    mask.device != self.device:
                raise ValueError(f"mask must be a bool tensor of shape [rows, width] on {self.device}")
            if mask.shape[1] > 1 and mask.stride(1) != 1:
                raise ValueError("mask must be dense in its last dimension")
            # An empty mask has no memory: it hides every key all the same.
            mask_args = (mask.data_ptr() or self._k_scales.data_ptr(), mask.stride(0), mask.shape[1])
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif self._rows("out", out, heads) != kind or out.shape[0] != rows:
            raise ValueError("out must have q's shape and dtype")
        lse = torch.empty((rows, heads), dtype=torch.float32, device=self.device) if return_lse else None
        sizes = (batch[3], batch[4], rows, heads)
        need = self._workspaces.get(sizes)
        if need is None:
            size = ctypes.c_uint64(0)
            with torch.cuda.device(self.device):
                _native.check(self._lib.msim_kv4_attend_workspace(self._pool_ptr, *sizes, ctypes.byref(size)))
            if len(self._workspaces) >= 256:
                self._workspaces.clear()
            need = self._workspaces[sizes] = size.value
        work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        _launch(self.device, self._lib.msim_kv4_attend_async, self._pool_ptr, *batch, q.data_ptr(), *q.stride()[:2],
                heads, kind, scale, 1 if causal else 0, 0 if window is None else int(window), *mask_args,
                out.data_ptr(), *out.stride()[:2], None if lse is None else lse.data_ptr(),
                None if work is None else work.data_ptr(), need)
        return (out, lse) if return_lse else out
