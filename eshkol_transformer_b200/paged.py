"""Paged KV cache on torch CUDA tensors: appending (et_b200_paged_append_v1)
and attention of new tokens over it (et_b200_paged_attention_v1).

    cache = PagedCache(keys, values)             # one layer's pools
    batch = PagedBatch(offsets, lengths, table, tokens, max_new, max_length)
    cache.append(batch, k, v, rope=(cos, sin))
    attention = PagedAttention(cache, q_heads)
    attention.forward(batch, q, o, rope=(cos, sin))

The descriptors hold the tensors they were built from and may be kept while
their contents change (a decoding loop updates offsets, lengths and the page
table in place).  Calls are enqueued on `stream` of the current device and
return at once: None is torch's current stream, as for torch's own operations;
else a cudaStream_t address (0 = the legacy default stream), and on a stream
other than torch's current one the caller orders the two and keeps the tensors
(Tensor.record_stream) until the call has run.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _check, k1, load

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

BAD_PAGE = 1    # a page outside the pool: reads as zeros, writes are dropped
BAD_LENGTH = 2  # a length below 0 or beyond the table's columns: clamped
BAD_OFFSET = 4  # offsets that fall or leave the tensors: clamped
BAD_ROPE = 8    # a position beyond the RoPE tables: the last row is used
TIMEOUT = 16    # a kernel gave up waiting: o is not valid (only status tells)


class CacheDescriptor(C.Structure):
    """et_b200_paged_cache_v1"""
    _fields_ = [("struct_size", C.c_size_t), ("keys", C.c_void_p), ("values", C.c_void_p),
                ("pages", C.c_int64), ("page_size", C.c_int64), ("kv_heads", C.c_int64),
                ("head_dim", C.c_int64), ("page_stride", C.c_int64), ("head_stride", C.c_int64),
                ("token_stride", C.c_int64), ("dtype", C.c_uint32), ("reserved", C.c_uint32)]


class BatchDescriptor(C.Structure):
    """et_b200_paged_batch_v1"""
    _fields_ = [("struct_size", C.c_size_t), ("batch", C.c_int64), ("tokens", C.c_int64),
                ("table_columns", C.c_int64), ("max_new", C.c_int64), ("max_length", C.c_int64),
                ("offsets", C.c_void_p), ("lengths", C.c_void_p), ("page_table", C.c_void_p),
                ("status", C.c_void_p)]


class RopeDescriptor(C.Structure):
    """et_b200_paged_rope_v1"""
    _fields_ = [("cos", C.c_void_p), ("sin", C.c_void_p), ("rows", C.c_int64)]


def stream_of(stream: int | None, index: int) -> int:
    """A call's stream: torch's current one unless given.  (The raw handle:
    torch.cuda.current_stream builds an object, 1.3 us of a call's 8.)"""
    return torch._C._cuda_getCurrentRawStream(index) if stream is None else stream


def _need(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


class PagedCache:
    """One layer's pools of pages, torch tensors [pages, kv_heads, page_size,
    head_dim] (f32, f16 or bf16) with a dense last dimension; any other strides
    of whole 16-byte pieces, the same for both (a [pages, page_size, kv_heads,
    head_dim] pool is passed as its transpose(1, 2))."""

    def __init__(self, keys, values):
        _need(keys.is_cuda and values.is_cuda and keys.device == values.device,
              "the pools must be CUDA tensors of one device")
        _need(keys.dim() == 4 and keys.shape == values.shape and keys.dtype == values.dtype,
              "the pools must be [pages, kv_heads, page_size, head_dim] tensors of one type")
        _need(keys.dtype in DTYPES, "the pools must be f32, f16 or bf16")
        _need(keys.numel() > 0, "the pools are empty")
        # a dimension of one element has no stride of its own: its dense one
        strides = [self._strides(t) for t in (keys, values)]
        _need(strides[0] == strides[1], "both pools must have the same strides")
        self.lib = load()
        self.keys, self.values = keys, values
        self.device, self.index, self.dtype = keys.device, keys.get_device(), keys.dtype
        self.pages, self.kv_heads, self.page_size, self.head_dim = keys.shape
        page, head, token = strides[0]
        self.descriptor = CacheDescriptor(
            C.sizeof(CacheDescriptor), keys.data_ptr(), values.data_ptr(), self.pages,
            self.page_size, self.kv_heads, self.head_dim, page, head, token, DTYPES[keys.dtype], 0)
        self._ref = C.byref(self.descriptor)

    @staticmethod
    def _strides(t):
        pages, heads, slots, dim = t.shape
        page, head, token, last = t.stride()
        _need(last == 1 or dim == 1, "the pools' last dimension must be dense")
        if heads == 1 and slots == 1:
            head = token = dim
        elif slots == 1:
            token = heads * head if head >= dim else dim
        elif heads == 1:
            head = slots * token
        if pages == 1:
            page = max(slots * token, heads * head)
        return page, head, token

    def append(self, batch: "PagedBatch", k, v, rope=None, stream: int | None = None) -> None:
        """Stores k (rotated by rope = (cos, sin), [positions, head_dim / 2]
        each) and v, [tokens, kv_heads, head_dim] with dense heads."""
        err = k1.KernelError()
        k_stride = _rows(k, batch, self, self.kv_heads, "k")
        v_stride = _rows(v, batch, self, self.kv_heads, "v")
        rc = self.lib.et_b200_paged_append_v1(
            self._ref, batch.bind(self), batch.rope(rope, self), k.data_ptr(), k_stride,
            v.data_ptr(), v_stride, stream_of(stream, self.index), C.byref(err))
        if rc != 0:
            _check(rc, err)


class PagedBatch:
    """One step's requests: offsets [batch + 1] and lengths [batch] (i64),
    page_table [batch, columns] (i32) on the device, rows of the token-major
    tensors; max_new (new tokens of the largest request as far as the host
    knows; None counts all tokens as one request's, which for many single
    tokens is the slower kernel) only picks the kernel, max_length is not used
    so far.  status: an i32 tensor of one element that collects BAD_* and
    TIMEOUT bits, or None: then nothing tells of either."""

    def __init__(self, offsets, lengths, page_table, tokens: int, max_new: int | None = None,
                 max_length: int | None = None, status=None):
        batch = lengths.numel()
        _need(offsets.dtype == torch.int64 and lengths.dtype == torch.int64,
              "offsets and lengths must be i64")
        _need(page_table.dtype == torch.int32, "the page table must be i32")
        _need(offsets.shape == (batch + 1,) and lengths.dim() == 1, "offsets need batch + 1 entries")
        _need(page_table.dim() == 2 and page_table.shape[0] == batch and page_table.shape[1] > 0,
              "the page table must be [batch, columns]")
        tensors = [offsets, lengths, page_table]
        if status is not None:
            _need(status.dtype == torch.int32 and status.numel() == 1, "status must be one i32")
            tensors.append(status)
        for t in tensors:
            _need(t.is_cuda and t.device == offsets.device and t.is_contiguous(),
                  "the batch's tensors must be dense CUDA tensors of one device")
        self.tokens, self.index = int(tokens), offsets.get_device()
        self.keepalive = tensors
        columns = page_table.shape[1]
        self.descriptor = BatchDescriptor(
            C.sizeof(BatchDescriptor), batch, self.tokens, columns,
            self.tokens if max_new is None else max_new,
            (1 << 31) - 1 if max_length is None else max_length, offsets.data_ptr(),
            lengths.data_ptr(), page_table.data_ptr(),
            status.data_ptr() if status is not None else None)
        self._ref = C.byref(self.descriptor)

    def bind(self, cache: PagedCache):
        if self.index != cache.index:
            raise ValueError("the batch and the cache are on different devices")
        if torch.cuda.current_device() != cache.index:
            raise ValueError("the cache's device is not the current one")
        return self._ref

    def rope(self, tables, cache: PagedCache):
        if tables is None:
            return None
        cos, sin = tables
        shape = cos.shape
        if (len(shape) != 2 or shape[1] * 2 != cache.head_dim or sin.shape != shape or
                cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or
                not cos.is_contiguous() or not sin.is_contiguous() or
                cos.get_device() != cache.index or sin.get_device() != cache.index):
            raise ValueError("RoPE tables must be dense f32 [positions, head_dim / 2] on the "
                             "cache's device")
        return C.byref(RopeDescriptor(cos.data_ptr(), sin.data_ptr(), shape[0]))


def _rows(t, batch: PagedBatch, cache: PagedCache, heads: int, name: str) -> int:
    """Checks a [tokens, heads, head_dim] tensor; its row stride."""
    dim = cache.head_dim
    if t.shape != (batch.tokens, heads, dim):
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    if t.dtype is not cache.dtype or t.get_device() != cache.index:
        raise ValueError(f"{name} must have the cache's type and device")
    row, head, last = t.stride()
    if last != 1 or (head != dim and heads != 1):
        raise ValueError(f"the heads of {name} must be dense")
    return row if batch.tokens > 1 else max(row, heads * dim)


class PagedAttention:
    """Attention of query heads over a paged cache, with its workspace (one
    call at a time: objects whose calls may overlap need their own)."""

    def __init__(self, cache: PagedCache, q_heads: int):
        self.lib = load()
        self.cache, self.q_heads = cache, q_heads
        with torch.cuda.device(cache.device):
            self.ws_bytes = self.lib.et_b200_paged_attention_workspace_bytes_v1(cache._ref, q_heads)
        _need(self.ws_bytes > 0, "paged attention shape rejected")
        self.ws = torch.empty(self.ws_bytes + 256, dtype=torch.uint8, device=cache.device)
        self.ws_ptr = (self.ws.data_ptr() + 255) & ~255

    def forward(self, batch: PagedBatch, q, o, rope=None, lse=None,
                stream: int | None = None) -> None:
        """o = attention of q (rotated by rope) over the keys each token sees;
        q, o [tokens, q_heads, head_dim]; lse f32 [tokens, q_heads] or None."""
        err = k1.KernelError()
        cache = self.cache
        q_stride = _rows(q, batch, cache, self.q_heads, "q")
        o_stride = _rows(o, batch, cache, self.q_heads, "o")
        if lse is not None:
            _need(lse.shape == (batch.tokens, self.q_heads) and lse.dtype == torch.float32 and
                  lse.is_contiguous() and lse.device == cache.device,
                  "lse must be dense f32 [tokens, q_heads] on the cache's device")
        _check(self.lib.et_b200_paged_attention_v1(
            cache._ref, batch.bind(cache), batch.rope(rope, cache), self.q_heads, q.data_ptr(),
            q_stride, o.data_ptr(), o_stride, lse.data_ptr() if lse is not None else None,
            self.ws_ptr, self.ws_bytes, stream_of(stream, cache.index), C.byref(err)), err)
