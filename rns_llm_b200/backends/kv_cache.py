"""Paged 8-bit key/value cache and attention over it, as methods of ``CudaRNSBackend``.

The reference replaces the linears around attention and leaves its cache and its softmax to
the model, in floating point.  These operators keep the cache in 8 bits as well: keys and values
are quantised as they are written (one scale for each page of tokens and head), and attention
reads the 8-bit pages.  Sequences of different lengths share a call: their new tokens are packed
along one axis, ``query_starts`` says where each begins, ``page_table`` where its pages lie.

Lengths, starts and page indices stay on the device and may change between replays of a captured
graph; one that is out of range is reported by ``check_status`` (see ``rns_kv_cache`` in
include/rns_b200.h).  Everything here is forward only.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import torch

from .. import _native as N

_FORMATS = {torch.int8: N.KV_INT8, torch.float8_e4m3fn: N.KV_E4M3}
_FORMAT_NAMES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_FLOAT_TYPES = {torch.float16: N.F16, torch.bfloat16: N.BF16, torch.float32: N.F32}


@dataclass
class QuantizedKVCache:
    """Pages of a key/value cache in 8 bits.

    ``k`` and ``v`` are contiguous ``[pages, kv_heads, page_tokens, head_dim]`` tensors of
    torch.int8 or torch.float8_e4m3fn; ``k_scale`` and ``v_scale`` float32 ``[pages, kv_heads]``:
    a byte stands for its value times the scale of its page and head, which is not negative.
    ``page_tokens`` is 16, 32, 64 or 128, ``head_dim`` a multiple of 16 up to 256.  The object keeps
    the addresses of the four tensors it was made with.
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    # the struct that calls copy and the shape as plain attributes
    _args: N.KVCacheArgs = field(init=False, repr=False, compare=False)
    device: torch.device = field(init=False, repr=False, compare=False)
    pages: int = field(init=False, repr=False, compare=False)
    kv_heads: int = field(init=False, repr=False, compare=False)
    page_tokens: int = field(init=False, repr=False, compare=False)
    head_dim: int = field(init=False, repr=False, compare=False)

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if k.ndim != 4 or k.shape != v.shape or k.dtype not in _FORMATS or v.dtype != k.dtype:
            raise ValueError("k and v must be [pages, kv_heads, page_tokens, head_dim] of one 8-bit type")
        if not k.is_contiguous() or not v.is_contiguous() or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("k and v must be contiguous and 16-byte aligned")
        for scale in (self.k_scale, self.v_scale):
            if scale.shape != k.shape[:2] or scale.dtype != torch.float32 or not scale.is_contiguous():
                raise ValueError("k_scale and v_scale must be contiguous float32 [pages, kv_heads]")
        if _spans_meet(k, v) or _spans_meet(self.k_scale, self.v_scale):
            raise ValueError("k and v, and their scales, must not overlap")
        if not k.is_cuda or any(t.device != k.device for t in (v, self.k_scale, self.v_scale)):
            raise ValueError("the cache must be CUDA tensors on one device")
        pages, heads, page_tokens, dim = (int(x) for x in k.shape)
        if page_tokens not in (16, 32, 64, 128):
            raise ValueError("page_tokens must be 16, 32, 64 or 128")
        if dim % 16 or not 16 <= dim <= 256:
            raise ValueError("head_dim must be a multiple of 16 in [16, 256]")
        if pages < 1 or heads < 1:
            raise ValueError("a cache has at least one page and one head")
        self._args = N.KVCacheArgs(d_k=k.data_ptr(), d_v=v.data_ptr(), d_k_scale=self.k_scale.data_ptr(),
                                   d_v_scale=self.v_scale.data_ptr(), pages=pages, page_tokens=page_tokens,
                                   kv_heads=heads, head_dim=dim, format=_FORMATS[k.dtype])
        self.device, self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.device, pages, heads, page_tokens, dim

    # Copies and pickles hold the tensors (as bytes: pickles of 8-bit floats do not load); the addresses are the
    # new ones'.
    def __getstate__(self) -> dict:
        return {"k": self.k.view(torch.int8), "v": self.v.view(torch.int8), "k_scale": self.k_scale,
                "v_scale": self.v_scale, "type": self.k.dtype}

    def __setstate__(self, state: dict) -> None:
        self.__init__(state["k"].view(state["type"]), state["v"].view(state["type"]), state["k_scale"], state["v_scale"])


class KVCacheOperators:
    """Mixed into ``CudaRNSBackend``."""

    def create_kv_cache(self, *, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64,
                        format: str = "int8", device: torch.device | str = "cuda") -> QuantizedKVCache:
        """A cache of zeros; ``format`` is "int8" or "e4m3"."""
        if format not in _FORMAT_NAMES:
            raise ValueError("format must be 'int8' or 'e4m3'")
        shape = (int(pages), int(kv_heads), int(page_tokens), int(head_dim))
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(_FORMAT_NAMES[format]) for _ in range(2))
        k_scale, v_scale = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        cache = QuantizedKVCache(k=k, v=v, k_scale=k_scale, v_scale=v_scale)
        self._state(cache.device)                    # calls on it may be captured from the first on
        return cache

    def kv_cache_write(self, cache: QuantizedKVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                       seq_lens: torch.Tensor, query_starts: torch.Tensor, *, max_query_len: int | None = None) -> None:
        """Quantises new keys and values into the cache.

        ``k``, ``v`` [tokens, kv_heads, head_dim] float16, bfloat16 or float32 with unit inner
        stride; sequence b's rows are ``query_starts[b]:query_starts[b+1]`` (int32 [sequences+1])
        and become the last tokens of its ``seq_lens[b]`` (int32 [sequences], the lengths AFTER the
        write).  ``page_table`` int32 [sequences, pages per sequence].  A page that already holds
        tokens of the sequence is rescaled when a larger value arrives.  ``max_query_len`` bounds
        the new tokens of one sequence (default: all tokens); one that has more is reported and not
        written."""
        if k.ndim != 3 or k.shape != v.shape or k.shape[1] != cache.kv_heads or k.shape[2] != cache.head_dim:
            raise ValueError("k and v must be [tokens, kv_heads, head_dim] of the cache")
        if k.dtype not in _FLOAT_TYPES or v.dtype != k.dtype:
            raise ValueError("k and v must be float16, bfloat16 or float32")
        if k.stride(2) != 1 or v.stride(2) != 1:
            raise ValueError("k and v must have unit inner stride")
        device = cache.device
        if k.device != device or v.device != device:
            raise ValueError("k and v must be on the cache's device")
        tokens = k.shape[0]
        args = self._kv_args(cache, page_table, seq_lens, query_starts)
        self._stats["kv_write_calls"] += 1
        with _on(device):
            N.check(self._lib.rns_kv_write(
                C.byref(args), k.data_ptr(), v.data_ptr(), _FLOAT_TYPES[k.dtype], tokens, k.stride(0), k.stride(1),
                v.stride(0), v.stride(1), seq_lens.data_ptr(), query_starts.data_ptr(),
                _bound(max_query_len, tokens), _stream(device)))

    def kv_cache_read(self, cache: QuantizedKVCache, page_table: torch.Tensor, first: torch.Tensor,
                      row_starts: torch.Tensor, *, rows: int, max_rows: int | None = None,
                      dtype: torch.dtype = torch.float16,
                      out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a range of every sequence, as ``dtype`` [rows, kv_heads, head_dim].

        Rows ``row_starts[b]:row_starts[b+1]`` (int32 [sequences+1]) are sequence b's tokens from
        position ``first[b]`` (int32 [sequences]) on; rows behind the last sequence's are not
        written.  ``max_rows`` bounds the rows of one sequence (default: all rows); one that has more
        is reported and not read."""
        rows = int(rows)
        if rows < 0:
            raise ValueError("rows must not be negative")
        shape = (rows, cache.kv_heads, cache.head_dim)
        device = cache.device
        if out is None:
            if dtype not in _FLOAT_TYPES:
                raise ValueError("dtype must be float16, bfloat16 or float32")
            out = (torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))
        else:
            dtype = out[0].dtype
            if len(out) != 2 or dtype not in _FLOAT_TYPES or any(
                    o.shape != shape or o.dtype != dtype or not o.is_contiguous() or o.device != device for o in out):
                raise ValueError("out must be two contiguous [rows, kv_heads, head_dim] floating tensors")
            if _spans_meet(*out):
                raise ValueError("the two outputs must not overlap")
        args = self._kv_args(cache, page_table, first, row_starts)
        self._stats["kv_read_calls"] += 1
        with _on(device):
            N.check(self._lib.rns_kv_read(
                C.byref(args), first.data_ptr(), row_starts.data_ptr(), rows, _bound(max_rows, rows),
                out[0].data_ptr(), out[1].data_ptr(), _FLOAT_TYPES[dtype], _stream(device)))
        return out

    def kv_cache_attention(self, q: torch.Tensor, cache: QuantizedKVCache, page_table: torch.Tensor,
                           seq_lens: torch.Tensor, query_starts: torch.Tensor, *, max_query_len: int | None = None,
                           softmax_scale: float | None = None, causal: bool = True, window: int | None = None,
                           out: torch.Tensor | None = None, return_lse: bool = False):
        """Attention of packed query tokens over the cached sequences.

        ``q`` [tokens, heads, head_dim] float16 or bfloat16 with unit inner stride; ``heads`` is a
        multiple of the cache's, and consecutive query heads share one.  Sequence b's queries are
        rows ``query_starts[b]:query_starts[b+1]`` and sit at the last positions of its
        ``seq_lens[b]`` tokens; each sees the tokens up to its own (all of them with
        ``causal=False``), and with ``window`` only the last ``window`` of those.  One that sees
        nothing gets zeros.  Rows of no sequence are not written.  ``out``, where given, shares no
        element with ``q``.  Returns the output in q's type
        and, with ``return_lse``, also float32 [tokens, heads]: the log of the sum of the
        exponentials of the scaled scores (-inf where nothing is seen).

        ``max_query_len`` bounds the new tokens of one sequence and chooses the kernels by it; without
        it a decode step of many sequences counts as one of many new tokens, which costs time."""
        if q.ndim != 3 or q.shape[2] != cache.head_dim or q.shape[1] % cache.kv_heads or q.shape[1] == 0:
            raise ValueError("q must be [tokens, heads, head_dim] with heads a multiple of the cache's kv_heads")
        if q.dtype != torch.float16 and q.dtype != torch.bfloat16:
            raise ValueError("q must be float16 or bfloat16")
        if q.stride(2) != 1:
            raise ValueError("q must have unit inner stride")
        device = cache.device
        if q.device != device:
            raise ValueError("q must be on the cache's device")
        if window is not None and (window < 1 or not causal):
            raise ValueError("window must be at least 1 and needs causal")
        tokens, heads, dim = q.shape
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
        elif (out.shape != q.shape or out.dtype != q.dtype or out.device != device or
              not (out.is_contiguous() or _rows_apart(out))):
            raise ValueError("out must be [tokens, heads, head_dim] of q's type with separate rows and unit inner stride")
        elif _rows_meet(out, q):
            raise ValueError("out must not overlap q")
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
        cache_args = self._kv_args(cache, page_table, seq_lens, query_starts)
        args = N.KVAttentionArgs(
            q.data_ptr(), _FLOAT_TYPES[q.dtype], heads, tokens, q.stride(0), q.stride(1), seq_lens.data_ptr(),
            query_starts.data_ptr(), _bound(max_query_len, tokens), causal, min(window or 0, 2 ** 31 - 1),
            dim ** -0.5 if softmax_scale is None else softmax_scale, out.data_ptr(), out.stride(0), out.stride(1),
            None if lse is None else lse.data_ptr(), None, 0)
        self._stats["kv_attention_calls"] += 1
        with self.arena.lock, _on(device):
            need = self._lib.rns_kv_attention_workspace(C.byref(cache_args), C.byref(args))
            if need < 0:
                N.check(-need)
            stream = _stream(device)
            if need:
                if torch.cuda.is_current_stream_capturing():
                    # a captured graph keeps scratch of its own: graphs captured on one stream may be
                    # replayed on two
                    workspace = torch.empty(need, dtype=torch.uint8, device=device)
                else:
                    workspace = self.arena.buffer(device.index, stream, need)
                args.d_workspace = workspace.data_ptr()
                args.workspace_bytes = need
            N.check(self._lib.rns_kv_attention(C.byref(cache_args), C.byref(args), stream))
        return (out, lse) if return_lse else out

    def _kv_args(self, cache: QuantizedKVCache, page_table: torch.Tensor, per_sequence: torch.Tensor,
                 starts: torch.Tensor) -> N.KVCacheArgs:
        """The cache with one call's page table, after checking the index tensors."""
        device = cache.device
        shape = page_table.shape
        if len(shape) != 2 or page_table.dtype != torch.int32 or page_table.device != device or (
                shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be int32 [sequences, pages] on the cache's device, unit inner stride")
        sequences, width = shape
        for tensor, count in ((per_sequence, sequences), (starts, sequences + 1)):
            if (tensor.shape != (count,) or tensor.dtype != torch.int32 or tensor.device != device or
                    not tensor.is_contiguous()):
                raise ValueError("lengths must be contiguous int32 [sequences] and starts [sequences + 1] on the "
                                 "cache's device")
        args = N.KVCacheArgs.from_buffer_copy(cache._args)
        args.d_page_table = page_table.data_ptr()
        args.table_stride = page_table.stride(0) if sequences > 1 else width
        args.table_pages = width
        args.sequences = sequences
        args.d_status = self._state(device).status.data_ptr()
        return args


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NOTHING = _Nothing()


def _on(device: torch.device):
    """Makes ``device`` current, when it is not."""
    return _NOTHING if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _bound(value: int | None, most: int) -> int:
    if value is None:
        return most
    if value < 0:
        raise ValueError("a bound on the tokens of one sequence must not be negative")
    return min(int(value), most)


def _rows_apart(t: torch.Tensor) -> bool:
    """[a, b, d] with unit inner stride whose rows do not overlap."""
    if t.stride(2) != 1:
        return False
    need = t.shape[2]
    for stride, size in sorted(zip(t.stride()[:2], t.shape[:2])):
        if size > 1:
            if stride < need:
                return False
            need = stride * size
    return True


def _spans_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the stretches of memory from the first to the last element of two tensors meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    first, end = zip(*((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(
        stride * (size - 1) for stride, size in zip(t.stride(), t.shape)))) for t in (a, b)))
    return first[0] < end[1] and first[1] < end[0]


def _rows_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [a, b, d] tensors of one shape and type, with unit inner stride, share an element.  Exact where
    their strides are equal (column blocks of one buffer); others are told apart by their spans only."""
    if not _spans_meet(a, b):
        return False
    rows, heads, dim = a.shape
    apart, odd = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    row, head = (0 if size == 1 else stride for size, stride in zip(a.shape[:2], a.stride()[:2]))
    if odd or (row, head) != tuple(0 if size == 1 else stride for size, stride in zip(b.shape[:2], b.stride()[:2])):
        return True
    # apart = i * row + j * head + k with |i| < rows, |j| < heads, |k| < dim
    for j in range(1 - heads, heads):
        rest = apart - j * head
        for i in ((rest // row, rest // row + 1) if row else (0,)):
            if abs(i) < rows and abs(rest - i * row) < dim:
                return True
    return False
