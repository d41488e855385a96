"""Key / value cache in 4 or 8 bits: host interface of the mm4_kv_cache_* entry points.

The attention of `attention.AttentionPlan` reads whole fp16 K and V each time, as the reference's does
(attention.swift:398). This module is for programs that keep K and V between calls: `KVCachePlan.append`
quantises the tokens of a call into a paged cache, `KVCachePlan.attention` attends over the cache where it lies
(one token per sequence, a few, or prompts), and `KVCachePlan.read` gives the cached values back as fp16.
`KVCacheBatch` names the sequences of a call; one batch serves every layer's cache.

    dims = KVCacheDimensions(pages=4096, pageSize=64, Hq=32, Hk=8, K=128, bits=4)
    plan = KVCachePlan(dims)
    cache = plan.allocate("cuda")                                   # one per layer
    batch = KVCacheBatch(pageTable, lengths, offsets, tokens, maxNew)
    plan.append(K, V, cache, batch)                                 # K, V: fp16 [tokens][Hk][128]
    O = plan.attention(Q, cache, batch)                             # Q, O: fp16 [tokens][Hq][128]

The layout of the cache and the meaning of its codes are in include/mm4.h.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

from . import _lib


@dataclass
class KVCacheDimensions:
    """pages of pageSize tokens (16, 32, 64, 128 or 256); Hq query heads over Hk key / value heads of K elements
    (128 or 64), as in AttentionDimensions; 4 or 8 bits."""
    pages: int
    pageSize: int
    Hq: int
    Hk: int
    K: int
    bits: int = 4


def _fits(width: int, **sizes):
    """Refuses sizes that the descriptors' integers, of `width` bits beside the sign, would cut."""
    for name, n in sizes.items():
        if not -(1 << width) <= n < 1 << width:
            raise ValueError(f"{name} {n} is out of range")


class KVCacheBatch:
    """The sequences of one call (mm4_kv_cache_batch). `pageTable` [sequences][pages per sequence], `lengths`
    [sequences] and `offsets` [sequences + 1] are contiguous CUDA int32 tensors; rows offsets[b] .. offsets[b+1]-1
    of K, V, Q and O are the last tokens of sequence b, whose length counts them. `tokens` is the number of rows,
    `maxNew` the most rows of one sequence. The tensors' contents are read when the kernels run, so they may be
    updated in place between calls and between replays of a captured call. The attributes are fixed: calls use the
    addresses and sizes of the tensors that the batch was made of."""

    def __init__(self, pageTable, lengths, offsets, tokens: int, maxNew: int):
        import torch
        dev = pageTable.get_device()
        for n, t, dims in (("pageTable", pageTable, 2), ("lengths", lengths, 1), ("offsets", offsets, 1)):
            if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.dim() != dims:
                raise ValueError(f"{n} must be a contiguous CUDA int32 tensor with {dims} dimension(s)")
            if t.get_device() != dev:
                raise ValueError("pageTable, lengths and offsets must be on one device")
        sequences = lengths.shape[0]
        if pageTable.shape[0] != sequences or offsets.shape[0] != sequences + 1:
            raise ValueError(f"{sequences} lengths need {sequences} page-table rows and {sequences + 1} offsets")
        if tokens < 0 or maxNew < 0:
            raise ValueError("tokens and maxNew must not be negative")
        _fits(31, tokens=tokens, maxNew=maxNew, sequences=sequences, pagesPerSequence=pageTable.shape[1])
        self.pageTable, self.lengths, self.offsets = pageTable, lengths, offsets
        self.sequences, self.tokens, self.maxNew, self.device = sequences, int(tokens), int(maxNew), dev
        self.desc = _lib.KVCacheBatchDesc(sequences, self.tokens, self.maxNew, pageTable.shape[1],
                                          pageTable.data_ptr(), lengths.data_ptr(), offsets.data_ptr())
        self._ref = ctypes.addressof(self.desc)  # last: from here on attributes are fixed

    def __setattr__(self, name, value):
        if "_ref" in self.__dict__:
            raise AttributeError(f"{name} of a KVCacheBatch is fixed: update the tensors in place or make another batch")
        object.__setattr__(self, name, value)


class KVCachePlan:
    """Cache geometry and attention options. `causal`: a token attends to itself and what lies before it (else to
    all its sequence has cached); `scale` None, 0 or less: 1 / sqrt(K). Immutable; may be used from several streams.

    `stream` of a call is a torch stream of the tensors' device (None: the current one). Its kernels follow what that
    stream holds already; inputs that another stream writes need a wait of the caller's, as do outputs read elsewhere.
    Tensors that a call allocates come from the memory of that stream."""

    def __init__(self, dims: KVCacheDimensions, causal: bool = True, scale: float | None = None):
        self._L = _lib.lib()
        _fits(63, pages=dims.pages)
        _fits(31, pageSize=dims.pageSize, Hq=dims.Hq, Hk=dims.Hk, K=dims.K, bits=dims.bits)
        self.dims = dims
        self.causal = bool(causal)
        d = _lib.KVCacheDesc(dims.pages, dims.pageSize, dims.Hq, dims.Hk, dims.K, dims.bits, int(self.causal),
                             0.0 if scale is None else float(scale))
        h = ctypes.c_void_p()
        _lib.check(self._L.mm4_kv_cache_plan_create(ctypes.byref(h), ctypes.byref(d)))
        self._h = h
        self.scale = float(scale) if d.scale > 0 else 1.0 / math.sqrt(dims.K)  # what the kernels use, as in mm4.h
        import torch
        self._f16, self._u8, self._f32 = torch.float16, torch.uint8, torch.float32
        self._empty_like, self._device = torch.empty_like, torch._C._cuda_getDevice
        self.pageBytes = int(self._L.mm4_kv_cache_page_bytes(h))
        self.cacheBytes = int(self._L.mm4_kv_cache_bytes(h))

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            self._L.mm4_kv_cache_plan_destroy(h)
            self._h = None

    def allocate(self, device="cuda"):
        """A cache for this plan: uint8 [pages][pageBytes], zeros."""
        import torch
        return torch.zeros(self.dims.pages, self.pageBytes, dtype=torch.uint8, device=device)

    def _cache(self, cache, batch, stream):
        if cache.dtype is not self._u8 or cache.numel() != self.cacheBytes or not cache.is_contiguous():
            raise ValueError(f"cache must be a contiguous CUDA uint8 tensor of {self.cacheBytes} bytes")
        dev = batch.device
        if cache.get_device() != dev:
            raise ValueError("cache and batch must be on one device")
        if dev != self._device():
            raise ValueError(f"the tensors are on device {dev}, which is not the current CUDA device")
        if stream is not None and stream.device_index != dev:
            raise ValueError(f"the stream belongs to device {stream.device_index}, the tensors are on device {dev}")
        return cache.data_ptr()

    def _rows(self, name, t, heads, batch):
        """(address, elements from row to row) of rows fp16 [tokens][heads][K]."""
        K = self.dims.K
        if t.shape != (batch.tokens, heads, K) or t.dtype is not self._f16 or t.get_device() != batch.device:
            raise ValueError(f"{name} must be an fp16 tensor of shape {(batch.tokens, heads, K)} on the batch's device")
        row, head, element = t.stride()
        if element != 1 or (head != K and heads > 1):
            raise ValueError(f"the heads of each row of {name} must be contiguous")
        return t.data_ptr(), row if batch.tokens > 1 else heads * K

    def append(self, K, V, cache, batch, stream=None) -> None:
        """Quantises the rows of K and V (fp16 [tokens][Hk][K]; rows may be strided, as slices of a fused
        projection are) into the cache (mm4_kv_cache_append)."""
        kp, ks = self._rows("K", K, self.dims.Hk, batch)
        vp, vs = self._rows("V", V, self.dims.Hk, batch)
        _lib.check(self._L.mm4_kv_cache_append(self._h, batch._ref, kp, ks, vp, vs, self._cache(cache, batch, stream),
                                               _lib.stream_handle(stream)))

    def read(self, cache, batch, K=None, V=None, stream=None):
        """(K, V): the fp16 values [tokens][Hk][K] that an append of this batch left in the cache
        (mm4_kv_cache_read). Padding rows of given tensors are left as they were; of new ones they are
        uninitialised."""
        Hk, D = self.dims.Hk, self.dims.K
        cp = self._cache(cache, batch, stream)
        if K is None and V is None:
            if stream is None:
                K = cache.new_empty((batch.tokens, Hk, D), dtype=self._f16)
                V = self._empty_like(K)
            else:
                K, V = _lib.new_on_stream(stream, lambda: tuple(
                    cache.new_empty((batch.tokens, Hk, D), dtype=self._f16) for _ in range(2)))
            kp, vp, ks = K.data_ptr(), V.data_ptr(), Hk * D
            vs = ks
        elif K is None or V is None:
            raise ValueError("give both K and V, or neither")
        else:
            kp, ks = self._rows("K", K, Hk, batch)
            vp, vs = self._rows("V", V, Hk, batch)
        _lib.check(self._L.mm4_kv_cache_read(self._h, batch._ref, cp, kp, ks, vp, vs, _lib.stream_handle(stream)))
        return K, V

    def attention_workspace_bytes(self, batch) -> int:
        """Bytes of scratch `attention` needs for this batch (any contents, 16-byte aligned)."""
        return int(self._L.mm4_kv_cache_attention_workspace_size(self._h, batch._ref))

    def attention_kernel_name(self, batch) -> str:
        return self._L.mm4_kv_cache_attention_kernel_name(self._h, batch._ref).decode()

    def attention(self, Q, cache, batch, O=None, lse=None, workspace=None, stream=None):
        """O = softmax(scale Q K^T) V over each sequence's cached keys and values, fp16 [tokens][Hq][K]
        (mm4_kv_cache_attention); append the call's tokens first. With `lse` (fp32 [tokens][Hq]) also writes each
        row's natural-log sum of exp(scale * S). A row that attends to nothing gets O = 0 and lse = -inf.
        `workspace`: a CUDA uint8 tensor; by default each call takes one from torch's allocator."""
        Hq, D = self.dims.Hq, self.dims.K
        qp, qs = self._rows("Q", Q, Hq, batch)
        cp = self._cache(cache, batch, stream)
        if O is None:
            if stream is None and Q.is_contiguous():
                O = self._empty_like(Q)
            else:
                O = _lib.new_on_stream(stream, lambda: Q.new_empty((batch.tokens, Hq, D)))
            op, os_ = O.data_ptr(), Hq * D
        else:
            op, os_ = self._rows("O", O, Hq, batch)
        lp = None
        if lse is not None:
            if lse.shape != (batch.tokens, Hq) or lse.dtype is not self._f32 or not lse.is_contiguous() or \
                    lse.get_device() != batch.device:
                raise ValueError(f"lse must be a contiguous CUDA fp32 tensor of shape {(batch.tokens, Hq)}")
            lp = lse.data_ptr()
        nbytes = self._L.mm4_kv_cache_attention_workspace_size(self._h, batch._ref)
        wp = None
        if nbytes:
            if workspace is None:
                workspace = cache.new_empty(nbytes) if stream is None else \
                    _lib.new_on_stream(stream, lambda: cache.new_empty(nbytes), returned=False)
            elif workspace.get_device() != batch.device or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous tensor on the batch's device")
            else:
                nbytes = workspace.numel() * workspace.element_size()
            wp = workspace.data_ptr()
        _lib.check(self._L.mm4_kv_cache_attention(self._h, batch._ref, qp, qs, cp, op, os_, lp, wp, nbytes,
                                                  _lib.stream_handle(stream)))
        return O
