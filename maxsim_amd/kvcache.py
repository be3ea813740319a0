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
attention).  ``append``, ``attend`` and ``keep`` can be captured in a HIP graph.
"""
from __future__ import annotations

from maxsim_amd import _native

HEAD_DIMS = (64, 96, 128, 192, 256)


def _cuda_device(device):
    import torch

    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("device must be 'cuda'")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return device


def _type_number(dtype) -> int:
    """The C ABI's number of an element type (None: bfloat16)."""
    import torch

    if dtype is None or dtype is torch.bfloat16:
        return 2
    if dtype is torch.float16:
        return 1
    if dtype is torch.float32:
        return 0
    raise ValueError("dtype must be float32, float16 or bfloat16")


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
        self._calls = _native.tensor_calls()
        shape = (num_pages, kv_heads, page_size)
        self._k_codes, self._v_codes = (torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=self.device)
                                        for _ in range(2))
        self._k_scales, self._v_scales = (torch.zeros(shape, dtype=torch.float32, device=self.device)
                                          for _ in range(2))
        self.num_pages, self.kv_heads, self.head_dim, self.page_size = num_pages, kv_heads, head_dim, page_size
        self._handle = self._calls.cache(self._k_codes, self._k_scales, self._v_codes, self._v_scales)

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

    # ----------------------------------------------------------------- calls

    def append(self, k, v, page_table, lengths, offsets=None) -> None:
        """Quantise keys and values [rows, kv_heads, head_dim] (float32, float16
        or bfloat16, any strides with dense rows) into the cache.  A row that
        holds an infinity or a NaN reads back as NaN.  Sequences may share pages
        that are only read: a slot given to two rows of one call is left with
        parts of both."""
        self._calls.append(self._handle, k, v, page_table, lengths, offsets)

    def read(self, page_table, lengths, offsets=None, *, rows=None, dtype=None, out=None):
        """The rows (keys, values) [rows, kv_heads, head_dim] read back, each
        value code * scale rounded once to ``dtype`` (default bfloat16).  ``rows``
        is their number; without it, and with offsets, the last offset is fetched
        from the device.  ``out`` is a pair of tensors to write."""
        if out is not None:
            k, v = out
            if (rows is not None and int(rows) != k.shape[0]) or (dtype is not None and dtype != k.dtype):
                raise ValueError("rows and dtype must be those of out")
            return self._calls.read(self._handle, page_table, lengths, offsets, 0, 0, k, v)
        if rows is None:
            if offsets is not None and (offsets.ndim != 1 or offsets.shape[0] < 1):
                raise ValueError("offsets must have shape [batch + 1]")
            rows = lengths.shape[0] if offsets is None else int(offsets[-1])
        return self._calls.read(self._handle, page_table, lengths, offsets, rows, _type_number(dtype), None, None)

    def keep(self, page_table, lengths, offsets, kept):
        """Of the rows that a call added, some stay: ``kept`` int32 [batch, width] lists
        the numbers of each sequence's rows that do, ascending; the list ends at the
        first entry that is no such number (-1).  They move up to the end of what
        the sequence held before, and the new lengths (int32 [batch]) are returned:
        length - rows + rows kept, 0 at least.  Table, lengths and offsets are those of the call
        that added the rows; pages that are spare now stay in the table.  A row that
        lies in a hole is zeros.  At most 2^20 sequences."""
        return self._calls.keep(self._handle, page_table, lengths, offsets, kept)

    def attend(self, q, page_table, lengths, offsets=None, *, scale=None, causal=True, window=None, sinks=None,
               mask=None, parents=None, out=None, return_lse=False):
        """Attention of queries [rows, heads, head_dim] over their sequences.

        ``heads`` is a multiple of kv_heads; query head h reads key/value head
        ``h // (heads // kv_heads)``.  Row i of a sequence's n stands at position
        p = length - n + i and sees the keys j < length with j <= p (``causal``),
        j > p - window (``window``) or j < sinks (``sinks``: first tokens that
        stay visible under a window), and mask[row, j] (``mask`` bool
        [rows, width]; keys past its width are hidden).

        ``parents`` int32 [rows] makes each sequence's rows a tree of drafted tokens:
        parents[row] is the number, among the sequence's rows, of the earlier one
        that the row comes after; any other number (-1): the last token before them.
        A row then sees the tokens before the sequence's rows, the rows that it comes
        after and itself, and stands at length - n + the number of rows that it comes
        after (``sinks`` and ``window`` go by these positions).  A sequence may have 1,024
        rows then; rows of a longer one see nothing.

        ``scale`` defaults to
        head_dim ** -0.5.  Returns [rows, heads, head_dim] in q's dtype, rounded
        once from single precision sums, and with ``return_lse`` the logarithm
        of each softmax's sum, float32 [rows, heads].  A row that sees nothing
        is zeros, with minus infinity.  ``out`` may be q itself, and must not
        overlap it otherwise.  Queries and values may have any size, keys up to
        2^102.
        """
        if window is not None and window < 1:
            raise ValueError("window must be positive")
        return self._calls.attend(self._handle, q, page_table, lengths, offsets,
                                  self.head_dim ** -0.5 if scale is None else scale, causal, window or 0, mask, out,
                                  bool(return_lse), sinks or 0, parents)
