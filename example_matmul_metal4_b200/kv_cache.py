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


class KVCacheBatch:
    """The sequences of one call (mm4_kv_cache_batch). `pageTable` [sequences][pages per sequence], `lengths`
    [sequences] and `offsets` [sequences + 1] are contiguous CUDA int32 tensors; rows offsets[b] .. offsets[b+1]-1
    of K, V, Q and O are the last tokens of sequence b, whose length counts them. `tokens` is the number of rows,
    `maxNew` the most rows of one sequence. The tensors' contents are read when the kernels run, so they may be
    updated in place between calls and between replays of a captured call."""

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
        self.pageTable, self.lengths, self.offsets = pageTable, lengths, offsets
        self.sequences, self.tokens, self.maxNew, self.device = sequences, int(tokens), int(maxNew), dev
        self.desc = _lib.KVCacheBatchDesc(sequences, self.tokens, self.maxNew, pageTable.shape[1],
                                          pageTable.data_ptr(), lengths.data_ptr(), offsets.data_ptr())
        self._ref = ctypes.addressof(self.desc)


class KVCachePlan:
    """Cache geometry and attention options. `causal`: a token attends to itself and what lies before it (else to
    all its sequence has cached); `scale` as in AttentionPlan. Immutable; may be used from several streams."""

    def __init__(self, dims: KVCacheDimensions, causal: bool = True, scale: float | None = None):
        self._L = _lib.lib()
        self.dims = dims
        self.causal = bool(causal)
        self.scale = scale if scale is not None else 1.0 / math.sqrt(dims.K) if dims.K > 0 else 0.0
        d = _lib.KVCacheDesc(dims.pages, dims.pageSize, dims.Hq, dims.Hk, dims.K, dims.bits, int(self.causal),
                             float(self.scale))
        h = ctypes.c_void_p()
        _lib.check(self._L.mm4_kv_cache_plan_create(ctypes.byref(h), ctypes.byref(d)))
        self._h = h
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

    def _cache(self, cache, batch):
        import torch
        if cache.dtype is not torch.uint8 or cache.numel() != self.cacheBytes or not cache.is_contiguous():
            raise ValueError(f"cache must be a contiguous CUDA uint8 tensor of {self.cacheBytes} bytes")
        dev = batch.device
        if cache.get_device() != dev:
            raise ValueError("cache and batch must be on one device")
        if dev != torch._C._cuda_getDevice():
            raise ValueError(f"the tensors are on device {dev}, which is not the current CUDA device")
        return cache.data_ptr()

    def _rows(self, name, t, heads, batch):
        import torch
        shape = t.shape
        if len(shape) != 3 or shape[0] != batch.tokens or shape[1] != heads or shape[2] != self.dims.K or \
                t.dtype is not torch.float16 or t.get_device() != batch.device:
            raise ValueError(f"{name} must be an fp16 tensor of shape {(batch.tokens, heads, self.dims.K)} on the "
                             "batch's device")
        stride = t.stride()
        if stride[2] != 1 or (stride[1] != self.dims.K and heads > 1):
            raise ValueError(f"the heads of each row of {name} must be contiguous")
        width = heads * self.dims.K
        if shape[0] <= 1:
            return t.data_ptr(), width
        return t.data_ptr(), stride[0]

    def append(self, K, V, cache, batch, stream=None) -> None:
        """Quantises the rows of K and V (fp16 [tokens][Hk][K]; rows may be strided, as slices of a fused
        projection are) into the cache (mm4_kv_cache_append)."""
        kp, ks = self._rows("K", K, self.dims.Hk, batch)
        vp, vs = self._rows("V", V, self.dims.Hk, batch)
        _lib.check(self._L.mm4_kv_cache_append(self._h, batch._ref, kp, ks, vp, vs, self._cache(cache, batch),
                                               _lib.stream_handle(stream)))

    def read(self, cache, batch, K=None, V=None, stream=None):
        """(K, V): the fp16 values [tokens][Hk][K] that an append of this batch left in the cache
        (mm4_kv_cache_read). Padding rows of given tensors are left as they were; of new ones they are
        uninitialised."""
        import torch
        shape = (batch.tokens, self.dims.Hk, self.dims.K)
        if K is None:
            K = torch.empty(shape, dtype=torch.float16, device=cache.device)
            _keep(K, stream)
        if V is None:
            V = torch.empty(shape, dtype=torch.float16, device=cache.device)
            _keep(V, stream)
        kp, ks = self._rows("K", K, self.dims.Hk, batch)
        vp, vs = self._rows("V", V, self.dims.Hk, batch)
        _lib.check(self._L.mm4_kv_cache_read(self._h, batch._ref, self._cache(cache, batch), kp, ks, vp, vs,
                                             _lib.stream_handle(stream)))
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
        import torch
        Hq = self.dims.Hq
        qp, qs = self._rows("Q", Q, Hq, batch)
        cp = self._cache(cache, batch)
        if O is None:
            O = torch.empty((batch.tokens, Hq, self.dims.K), dtype=torch.float16, device=Q.device)
            _keep(O, stream)
        op, os_ = self._rows("O", O, Hq, batch)
        lp = None
        if lse is not None:
            if tuple(lse.shape) != (batch.tokens, Hq) or lse.dtype != torch.float32 or not lse.is_contiguous() or \
                    lse.get_device() != batch.device:
                raise ValueError(f"lse must be a contiguous CUDA fp32 tensor of shape {(batch.tokens, Hq)}")
            lp = lse.data_ptr()
        nbytes = self._L.mm4_kv_cache_attention_workspace_size(self._h, batch._ref)
        wp = None
        if nbytes:
            if workspace is None:
                workspace = torch.empty(nbytes, dtype=torch.uint8, device=Q.device)
                _keep(workspace, stream)
            elif workspace.get_device() != batch.device or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous tensor on the batch's device")
            else:
                nbytes = workspace.numel() * workspace.element_size()
            wp = workspace.data_ptr()
        _lib.check(self._L.mm4_kv_cache_attention(self._h, batch._ref, qp, qs, cp, op, os_, lp, wp, nbytes,
                                                  _lib.stream_handle(stream)))
        return O


def _keep(t, stream) -> None:
    """A tensor made here on torch's current stream and used on a stream of the caller's is not reused before
    that stream is done with it."""
    if stream is not None:
        t.record_stream(stream)
