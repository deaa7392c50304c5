"""A paged KV cache in 8 bits with one scale for each block of 16 tokens and head.

Storage, page tables, lengths and reference counts are torch CUDA tensors of the
caller; the calls only read and write them, on the context's stream, so that a
decode step (fork the beams, grow the streams, append, attend) is launched
without reading anything back. The definitions are in include/vkb200.h
(vkb_bkv_*, vkb_pages_*).

    cache = BlockKvCache.empty(ctx, n_layer, n_kv_head, d_head, n_pages)
    pages = cache.pages(status)
    a, b = PageState.empty(n_seq, max_pages, n_pages), PageState.empty(...)
    pages.advance(a, b, parent, n_new)                 # b is the new state
    step = Batch(tok_start, b.len, b.table, n_tok, max_q, status)
    for layer in range(n_layer):
        cache.append(layer, step, k, v)
        out = cache.attention(layer, step, q, scale)

The context's stream is the one that was torch's current stream when the context
was made (Context.set_stream changes it). Tensors that were written, or are read
or freed, on another stream are ordered by the caller, with an event, as for any
other kernel; a tensor that a call allocates belongs to torch's current stream.
Waits inside the kernels are bounded: ctx.synchronize() raises where one gave up and a result is not complete.
A whole decode loop is in examples/beam_decode.py.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check, VkbError  # noqa: F401
from .logits import _DTYPES, _at_home, _bad, _device, _tensor

_L = _lib.load()
BLOCK = _lib.BKV_BLOCK


def _i32(t, name, ndim):
    if t is None:
        _bad(f"{name}: missing")
    return _tensor(t, name, (torch.int32,), ndim)


class Batch:
    """The streams of a step: stream s owns rows tok_start[s] .. tok_start[s + 1] - 1 of the step's row
    tensors, which are its last rows; kv_len[s] counts its tokens, the step's included; table[s] lists its
    pages. n_tok = tok_start[-1], max_q the largest number of rows of a stream; status (optional): the
    status of PagePool, append stores nothing where it is not 0; max_kv (optional): tokens of the longest
    stream, for the choice of the attention's kernel (0: as many as the table holds)."""

    def __init__(self, tok_start, kv_len, table, n_tok: int, max_q: int, status=None, max_kv: int = 0):
        s = _lib.BkvBatch()
        s.tok_start, s.kv_len, s.table = _i32(tok_start, "tok_start", 1), _i32(kv_len, "kv_len", 1), _i32(table, "table", 2)
        if not tok_start.is_contiguous() or not kv_len.is_contiguous():
            _bad("tok_start and kv_len must be contiguous")
        n_seq = kv_len.shape[0]
        if tok_start.shape[0] != n_seq + 1 or table.shape[0] != n_seq:
            _bad(f"{n_seq} lengths want {n_seq + 1} starts and {n_seq} rows of the table")
        s.n_seq, s.n_tok, s.max_q, s.max_kv = n_seq, n_tok, max_q, max_kv
        s.table_ld = table.stride(0) if n_seq > 1 else table.shape[1]
        if s.table_ld != table.shape[1]:
            _bad("table: its rows must follow one another")
        s.status = None if status is None else _i32(status, "status", 1)
        self.n_tok = n_tok
        self.tensors = (tok_start, kv_len, table, status)
        self.device = _device(self.tensors)
        self.struct, self.ref = s, C.byref(s)


class PageState:
    """Page tables int32 [n_seq, max_pages] (-1 behind a stream's last page), lengths int32 [n_seq] and
    reference counts int32 [n_pages]."""

    def __init__(self, table, len, refs):  # noqa: A002
        self.table, self.len, self.refs = table, len, refs
        s = _lib.PageState(_i32(table, "table", 2), _i32(len, "len", 1), _i32(refs, "refs", 1))
        if not (table.is_contiguous() and len.is_contiguous() and refs.is_contiguous()):
            _bad("a page state's tensors must be contiguous")
        if len.shape[0] != table.shape[0]:
            _bad("as many lengths as rows of the table are wanted")
        self.device = _device((table, len, refs))
        self.struct, self.ref = s, C.byref(s)

    @staticmethod
    def empty(n_seq: int, max_pages: int, n_pages: int, device="cuda") -> "PageState":
        """Streams without tokens."""
        return PageState(torch.full((n_seq, max_pages), -1, dtype=torch.int32, device=device),
                         torch.zeros(n_seq, dtype=torch.int32, device=device),
                         torch.zeros(n_pages, dtype=torch.int32, device=device))


class PagePool:
    """The pages of one or more arenas [n_layer, n_pages, ...], contiguous tensors of any type."""

    def __init__(self, ctx, arenas, status, page_tokens: int = BLOCK):
        if not arenas or any(t.dim() < 2 or not t.numel() for t in arenas):
            _bad("arenas: one tensor of pages at least, none of them empty, is wanted")
        n_layer, n_pages = arenas[0].shape[:2]
        planes = (_lib.PagePlane * len(arenas))()
        for p, t in zip(planes, arenas):
            if not t.is_cuda or not t.is_contiguous() or tuple(t.shape[:2]) != (n_layer, n_pages):
                _bad(f"arenas: contiguous CUDA tensors of shape [{n_layer}, {n_pages}, ...] are wanted")
            page = t.element_size() * (t.numel() // (n_layer * n_pages))
            p.base, p.page_bytes, p.layer_bytes = t.data_ptr(), page, page * n_pages
        _at_home(ctx, _device((*arenas, status)), "arenas and status")
        self.ctx, self.status, self.n_pages = ctx, status, n_pages
        self._keep = (arenas, planes)
        self.struct = _lib.PagePool(n_layer, len(arenas), planes, n_pages, 0, page_tokens, 0, _i32(status, "status", 1))
        self.ref = C.byref(self.struct)

    def _states(self, a: PageState, b: PageState):
        if a.table.shape != b.table.shape or a.refs.shape != b.refs.shape or a.refs.shape[0] != self.n_pages:
            _bad("pages: the two states have other shapes than each other or than the arenas")
        _at_home(self.ctx, a.device, "state")
        _at_home(self.ctx, b.device, "state")
        self.struct.n_seq, self.struct.table_ld = a.table.shape

    def advance(self, a: PageState, b: PageState, parent=None, n_new=None):
        """b = a with stream i made stream parent[i] (negative: freed; None: as it was), then grown by n_new[i]
        tokens; a partly filled page that others share is copied first. Where it cannot be done, the status
        is raised (PAGES_EXHAUSTED, PAGES_TABLE_FULL, PAGES_BAD_INPUT) and b is a."""
        self._states(a, b)
        for t, name in ((parent, "parent"), (n_new, "n_new")):
            if t is not None and (_i32(t, name, 1) is None or t.shape[0] != a.len.shape[0] or not t.is_contiguous()):
                _bad(f"{name}: a contiguous int32 tensor with one entry a stream is wanted")
            if t is not None:
                _at_home(self.ctx, t.get_device(), name)
        check(_L.vkb_pages_advance(self.ctx.h, self.ref, None if parent is None else parent.data_ptr(),
                                   None if n_new is None else n_new.data_ptr(), a.ref, b.ref))

    def compact(self, a: PageState, b: PageState, n_used=None):
        """b = a with the pages in use moved to the front of the arenas; n_used (int32 [1]): how many there are."""
        self._states(a, b)
        if n_used is not None:
            _at_home(self.ctx, n_used.get_device(), "n_used")
        check(_L.vkb_pages_compact(self.ctx.h, self.ref, a.ref, b.ref, None if n_used is None else _i32(n_used, "n_used", 1)))

    def check(self):
        """Raises when an advance could not be done (waits for the stream)."""
        st = int(self.status.cpu()[0])
        if st == _lib.PAGES_EXHAUSTED:
            raise VkbError(_lib.ERROR_KV_CACHE_EXHAUSTED, f"paged KV cache exhausted: arena has {self.n_pages} pages")
        if st:
            _bad("pages: a stream outgrows its table" if st == _lib.PAGES_TABLE_FULL else "pages: bad parents, counts or tables")


class BlockKvCache:
    """The arenas k int8 [n_layer, n_pages, n_kv_head, 16, d_head], v int8 [n_layer, n_pages, n_kv_head,
    d_head, 16] and their scales f32 [n_layer, n_pages, n_kv_head]; d_head 32, 64, 96, 128 or 256."""

    def __init__(self, ctx, k, v, k_scale, v_scale):
        _tensor(k, "k", (torch.int8,), 5)
        _tensor(v, "v", (torch.int8,), 5)
        n_layer, n_pages, n_kv_head, block, d_head = k.shape
        if block != BLOCK or tuple(v.shape) != (n_layer, n_pages, n_kv_head, d_head, BLOCK):
            _bad("k must be [n_layer, n_pages, n_kv_head, 16, d_head] and v [..., d_head, 16]")
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _tensor(t, name, (torch.float32,), 3)
            if tuple(t.shape) != (n_layer, n_pages, n_kv_head):
                _bad(f"{name} must be [n_layer, n_pages, n_kv_head]")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            _bad("the arenas must be contiguous")
        _at_home(ctx, _device((k, v, k_scale, v_scale)), "arenas")
        self.ctx, self.k, self.v, self.k_scale, self.v_scale = ctx, k, v, k_scale, v_scale
        self.n_layer, self.n_pages, self.n_kv_head, self.d_head = n_layer, n_pages, n_kv_head, d_head
        self.struct = _lib.BkvCache(n_layer, n_kv_head, d_head, n_pages, k.data_ptr(), v.data_ptr(), k_scale.data_ptr(),
                                    v_scale.data_ptr())
        self.ref = C.byref(self.struct)

    @staticmethod
    def empty(ctx, n_layer: int, n_kv_head: int, d_head: int, n_pages: int) -> "BlockKvCache":
        dev = f"cuda:{ctx.device}"
        k = torch.zeros(n_layer, n_pages, n_kv_head, BLOCK, d_head, dtype=torch.int8, device=dev)
        v = torch.zeros(n_layer, n_pages, n_kv_head, d_head, BLOCK, dtype=torch.int8, device=dev)
        ks = torch.zeros(n_layer, n_pages, n_kv_head, dtype=torch.float32, device=dev)
        return BlockKvCache(ctx, k, v, ks, torch.zeros_like(ks))

    def pages(self, status) -> PagePool:
        """The pages of this cache; status: int32 [1], zero."""
        return PagePool(self.ctx, (self.k, self.v, self.k_scale, self.v_scale), status)

    def _rows(self, t, name, heads, batch):
        """(pointer, row stride, dtype code) of rows [n_tok, heads, d_head] or [n_tok, heads * d_head]."""
        dt = _DTYPES.get(t.dtype)
        if dt is None:
            _bad(f"{name}: f32 or f16 rows are wanted, got {t.dtype}")
        shape, stride, d = t.shape, t.stride(), self.d_head
        if len(shape) == 3:
            ok = shape[1] == heads and shape[2] == d and stride[2] == 1 and (stride[1] == d or heads == 1)
        else:
            ok = len(shape) == 2 and shape[1] == heads * d and stride[1] == 1
        if not ok or shape[0] < batch.n_tok or not t.is_cuda:
            _bad(f"{name}: CUDA rows [{batch.n_tok}, {heads}, {d}] with contiguous rows are wanted, got {tuple(shape)}")
        on = t.get_device()
        if on != self.ctx.device or batch.device != on:
            _at_home(self.ctx, on, name)
            _at_home(self.ctx, batch.device, "batch")
        return t.data_ptr(), stride[0] if shape[0] > 1 else heads * d, dt

    def append(self, layer: int, batch: Batch, k, v):
        """Stores the batch's rows of k and v ([n_tok, n_kv_head, d_head], f32 or f16, any row stride)."""
        kp, k_ld, dt = self._rows(k, "k", self.n_kv_head, batch)
        vp, v_ld, dt_v = self._rows(v, "v", self.n_kv_head, batch)
        if dt != dt_v:
            _bad("k and v must have the same type")
        status = _L.vkb_bkv_append(self.ctx.h, self.ref, layer, batch.ref, kp, k_ld, vp, v_ld, dt)
        if status:
            check(status)

    def attention(self, layer: int, batch: Batch, q, scale: float = 1.0, out=None):
        """Causal attention of the rows q [n_tok, n_head, d_head] over their streams' caches; out like q unless given."""
        heads = q.shape[1] if q.dim() == 3 else q.shape[-1] // self.d_head if q.dim() else 0
        qp, q_ld, q_dt = self._rows(q, "q", heads, batch)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            op, o_ld, o_dt = out.data_ptr(), heads * self.d_head, q_dt
        else:
            op, o_ld, o_dt = self._rows(out, "out", heads, batch)
        status = _L.vkb_bkv_attention(self.ctx.h, self.ref, layer, batch.ref, heads, qp, q_ld, q_dt, scale, op, o_ld, o_dt)
        if status:
            check(status)
        return out

    def read(self, layer: int, batch: Batch, dtype=None):
        """(k, v): the stored values of the streams' last rows, [n_tok, n_kv_head, d_head], f32 or f16."""
        dtype = dtype or torch.float32
        dt = _DTYPES.get(dtype)
        if dt is None:
            _bad(f"read: dtype must be f32 or f16, got {dtype}")
        _at_home(self.ctx, batch.device, "batch")
        k = torch.empty((batch.n_tok, self.n_kv_head, self.d_head), dtype=dtype, device=self.k.device)
        v = torch.empty_like(k)
        status = _L.vkb_bkv_read(self.ctx.h, self.ref, layer, batch.ref, k.data_ptr(), v.data_ptr(), dt)
        if status:
            check(status)
        return k, v
