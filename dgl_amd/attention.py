"""Attention over the nodes of an instance or the positions of a sequence, as an operator of its own.

The policy network evaluates its attention inside fused kernels over the neighbourhood of one node (at most 256 tokens,
TSP/TSPModel.py:420-441).  Here it is for whole instances and long sequences, with capped scores, a bias that falls with
distance, document / causal / prefix masks, and its gradients (include/dgl_amd.h, dgl_attention_t):

    s_ij = cap tanh(scale q_i.k_j / cap) - slope[h] dist(i, j),     out_i = sum_j softmax_j(s_ij) v_j

Tensors are [batch, heads, tokens, head size] views of any strides whose last axis is consecutive (16-byte aligned; others
are copied), float32, float16 or bfloat16.  The computation runs in libdgl_amd on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_WIDE = (torch.int64, torch.uint32)                                 # integers that int32 does not hold
_VEC = {torch.float32: 4, torch.float16: 8, torch.bfloat16: 8}      # elements of 16 bytes

# A call of a few microseconds on the device is lost in a host path that sets ctypes fields one by one: the ABI structs are
# packed in one go (the formats restate include/dgl_amd.h; a wrong size fails here, at import).
_PACK_ATTENTION = struct.Struct("@8i2f12q5P3P2q2P2q2P")
_PACK_GRAD = struct.Struct("@4P12qP")
_PACK_CACHE = struct.Struct("@7i7q4P")
_PACK_STEP = struct.Struct("@2i2f4q6Pq2iPq")
_STEP_AT = _lib.AttentionStep.rows_per_instance.offset
assert _PACK_ATTENTION.size == ctypes.sizeof(_lib.Attention) and _PACK_GRAD.size == ctypes.sizeof(_lib.AttentionGrad)
assert _PACK_CACHE.size == ctypes.sizeof(_lib.KVCache)
assert _STEP_AT == ctypes.sizeof(_lib.KVCache) and _STEP_AT + _PACK_STEP.size == ctypes.sizeof(_lib.AttentionStep)
# The short ways to the current stream and device are not torch's documented ones (they save 1.2 of a call's 14 us): without them the
# documented ones serve.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(device, function, *args, what: str) -> None:
    """An entry point on the device's current stream, with that device current."""
    index = device.index
    if index == _current_device():              # (a tensor on the device is there: nothing is left to initialise)
        code = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = function(*args, _raw_stream(index))
    if code:
        check(code, what)


def forward_mode() -> bool:
    """Inside a dual level, where inputs may have tangents."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def derivatives(*inputs) -> bool:
    """Whether some input (a tensor or None) may have a gradient or a tangent to pass on: the quick question of every call."""
    if torch.is_grad_enabled():
        for t in inputs:
            if t is not None and t.requires_grad:
                return True
    return forward_mode()


def no_derivatives(what: str, **inputs) -> None:
    """Refuse inputs whose gradient or tangent the call would drop without a word."""
    if torch.is_grad_enabled():
        for name, t in inputs.items():
            if t is not None and t.requires_grad:
                raise ValueError(f"{what}: {name} requires grad, but no gradient passes here: detach it, or call under no_grad")
    if forward_mode():
        for name, t in inputs.items():
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what}: {name} has a tangent, but forward-mode derivatives do not pass here")


def _usable(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where the kernels can address it, else a contiguous copy."""
    vec, st = _VEC[t.dtype], t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0:
        if len(st) == 4:
            if not (st[0] % vec or st[1] % vec or st[2] % vec) and st[2] < (1 << 24):
                return t
        elif not any(x % vec for x in st[:-1]):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_qkv(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} has shape {tuple(t.shape)}: expected [batch, heads, tokens, head size]")
        if not t.is_cuda or t.device != q.device:
            raise ValueError(f"{name} is on {t.device}: q, k and v belong on one GPU")
        if t.dtype != q.dtype:
            raise ValueError(f"{name} is {t.dtype}, q is {q.dtype}")
    if q.dtype not in _DTYPES:
        raise ValueError(f"{q.dtype}: float32, float16 or bfloat16 is expected")
    B, H, _, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    if k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"{H} query heads over {k.shape[1]} key heads")


def _side(t: Optional[torch.Tensor], name, shape, dtype, device) -> Optional[torch.Tensor]:
    """A float32 / int32 / int64 side input, broadcast over the batch where it may be, inner axes consecutive."""
    if t is None:
        return None
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        if t.is_floating_point() != (dtype == torch.float32) or t.is_complex() or t.dtype == torch.uint64:
            raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
        if t.dtype in _WIDE and dtype == torch.int32:      # (2^32 + 5 is no 5: what does not fit stays beyond every bound)
            t = t.to(torch.int64).clamp(-(1 << 31), (1 << 31) - 1)
        t = t.to(dtype)
    if t.is_contiguous():
        return t
    n = 1
    for size, stride in zip(reversed(shape[1:]), reversed(t.stride()[1:])):
        if size > 1 and stride != n:
            return t.contiguous()
        n *= size
    return t.contiguous() if len(shape) == 1 else t


def _documents(doc_q, doc_k, B: int, L: int, M: int, device):
    """Both sides' document ids as int32.  Ids of wider types are mapped to small ones that are equal where they are."""
    if doc_q is None or not (doc_q.dtype in _WIDE or doc_k.dtype in _WIDE):
        return _side(doc_q, "doc_q", (B, L), torch.int32, device), _side(doc_k, "doc_k", (B, M), torch.int32, device)
    doc_q, doc_k = _side(doc_q, "doc_q", (B, L), torch.int64, device), _side(doc_k, "doc_k", (B, M), torch.int64, device)
    ids_q, ids_k = (torch.empty((B, n), dtype=torch.int32, device=device) for n in (L, M))
    if B:
        lib = _lib.load()
        ws = torch.empty(max(lib.dgl_document_ids_workspace_floats(B, M), 2), dtype=torch.float32, device=device)
        _launch(device, lib.dgl_document_ids, B, L, M, doc_q.data_ptr(), doc_q.stride(0), doc_k.data_ptr(), doc_k.stride(0),
                ids_q.data_ptr(), ids_k.data_ptr(), ws.data_ptr(), what="dgl_document_ids")
    return ids_q, ids_k


def _cap(cap) -> float:
    cap = float(cap)
    if not 0.0 <= cap < float("inf") or 0.0 < cap < 2.0 ** -126:       # (what binary32 rounds to 0 would be no cap)
        raise ValueError(f"cap {cap}: a number >= 0 is expected (0: no cap; else at least 2^-126)")
    return cap


def _both(a, b):
    """Addresses of a pair of side inputs.  An empty tensor has none, and NULL says "not given": nothing of it is read, so the
    other's stands in."""
    a, b = ptr(a), ptr(b)
    return a or b, b or a


class _Call:
    """Arguments of one operator call: the tensors the kernels can address, and the ABI struct over them."""
    __slots__ = ("q", "k", "v", "slope", "pos_q", "pos_k", "doc_q", "doc_k", "prefix", "head", "tail", "a", "out", "lse",
                 "rest")

    def __init__(self, q, k, v, scale, cap, slope, pos_q, pos_k, doc_q, doc_k, causal, prefix):
        _check_qkv(q, k, v)
        B, H, L, D = q.shape
        _, K, M, _ = k.shape
        dev = q.device
        cap = _cap(cap)
        if (pos_q is None) != (pos_k is None) or (doc_q is None) != (doc_k is None):
            raise ValueError("coordinates and document ids are given for both sides or for neither")
        if pos_q is not None and slope is None:
            raise ValueError("coordinates without a slope")
        if prefix is not None and not causal:
            raise ValueError("a prefix belongs to a causal mask")
        if max(L, M) > _lib.ATTENTION_MAX_LENGTH or B * H * (max(L, M) + 63) // 64 >= 1 << 30:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}: too long")
        self.q, self.k, self.v = _usable(q), _usable(k), _usable(v)
        self.slope = _side(slope, "slope", (H,), torch.float32, dev)
        self.pos_q = _side(pos_q, "pos_q", (B, L, 2), torch.float32, dev)
        self.pos_k = _side(pos_k, "pos_k", (B, M, 2), torch.float32, dev)
        self.doc_q, self.doc_k = _documents(doc_q, doc_k, B, L, M, dev)
        self.prefix = _side(prefix, "prefix", (B,), torch.int32, dev)
        self.head = (_DTYPES[q.dtype], B, H, K, L, M, D, 1 if causal else 0, D ** -0.5 if scale is None else float(scale), cap,
                     *self.q.stride()[:3], *self.k.stride()[:3], *self.v.stride()[:3])
        pos, doc = self.pos_q is not None, self.doc_q is not None
        self.tail = (ptr(self.slope), *_both(self.pos_q, self.pos_k), self.pos_q.stride(0) if pos else 0,
                     self.pos_k.stride(0) if pos else 0, *_both(self.doc_q, self.doc_k), self.doc_q.stride(0) if doc else 0,
                     self.doc_k.stride(0) if doc else 0, ptr(self.prefix))

    def set_out(self, out, lse, rest=None):
        self.out, self.lse, self.rest = out, lse, rest
        self.a = _lib.Attention()
        _PACK_ATTENTION.pack_into(self.a, 0, *self.head, *out.stride()[:3], self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(),
                                  out.data_ptr(), ptr(lse), *self.tail, ptr(rest))


def _like_heads(t: torch.Tensor) -> torch.Tensor:
    """An empty [batch, heads, tokens, size] tensor stored token by token (as the linear layer after the operator reads
    it) where its model is, head by head otherwise."""
    B, H, L, D = t.shape
    if t.stride(1) < t.stride(2):
        return torch.empty_strided((B, H, L, D), (L * H * D, D, H * D, 1), dtype=t.dtype, device=t.device)
    return torch.empty_strided((B, H, L, D), (H * L * D, L * D, D, 1), dtype=t.dtype, device=t.device)


def _forward(call: _Call, want_lse: bool, want_rest: bool = False):
    q = call.q
    out = _like_heads(q)
    rest = torch.empty_like(out) if want_rest and q.dtype != torch.float32 else None
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    call.set_out(out, lse, rest)
    if out.numel():
        lib = _lib.load()
        a = ctypes.byref(call.a)
        need = lib.dgl_attention_forward_workspace_floats(a)
        ws = torch.empty(need, dtype=torch.float32, device=q.device) if need > 0 else None
        _launch(q.device, lib.dgl_attention_forward, a, ptr(ws), what="dgl_attention_forward")
    return out, lse


def _backward(call: _Call, dout: torch.Tensor, want_slope: bool):
    lib, q = _lib.load(), call.q
    if dout.shape != q.shape or dout.dtype != q.dtype or dout.device != q.device:
        raise ValueError(f"dout is {tuple(dout.shape)} {dout.dtype} on {dout.device}, expected out's "
                         f"{tuple(q.shape)} {q.dtype} on {q.device}")
    dout = _usable(dout)
    dq, dk, dv = _like_heads(q), _like_heads(call.k), _like_heads(call.v)
    dslope = torch.empty(q.shape[1], dtype=torch.float32, device=q.device) if want_slope else None
    if q.shape[0] == 0:
        return dq, dk, dv, None if dslope is None else dslope.zero_()
    g = _lib.AttentionGrad()
    _PACK_GRAD.pack_into(g, 0, dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dout.stride()[:3], *dq.stride()[:3],
                         *dk.stride()[:3], *dv.stride()[:3], ptr(dslope))
    a = ctypes.byref(call.a)
    ws = torch.empty(max(lib.dgl_attention_backward_workspace_floats(a), 1), dtype=torch.float32, device=q.device)
    _launch(q.device, lib.dgl_attention_backward, a, ctypes.byref(g), ws.data_ptr(), what="dgl_attention_backward")
    return dq, dk, dv, dslope


def attention_forward(q, k, v, *, scale=None, cap=0.0, slope=None, pos_q=None, pos_k=None, doc_q=None, doc_k=None,
                      causal=False, prefix=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, lse) without autograd: the pair of calls to use where the backward pass is driven by hand, for instance
    inside a captured graph.  (In 16 bits the differentiable call also keeps what the rounding of ``out`` left off; here the
    backward pass works with the rounded output.)"""
    with torch.no_grad():
        return _forward(_Call(q, k, v, scale, cap, slope, pos_q, pos_k, doc_q, doc_k, causal, prefix), True)


def attention_backward(dout, q, k, v, out, lse, *, scale=None, cap=0.0, slope=None, pos_q=None, pos_k=None, doc_q=None,
                       doc_k=None, causal=False, prefix=None):
    """(dq, dk, dv, dslope or None) of the forward call with the same arguments, given its out and lse."""
    with torch.no_grad():
        call = _Call(q, k, v, scale, cap, slope, pos_q, pos_k, doc_q, doc_k, causal, prefix)
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out is {tuple(out.shape)} {out.dtype}, expected {tuple(q.shape)} {q.dtype}")
        if tuple(lse.shape) != tuple(q.shape[:3]) or lse.dtype != torch.float32 or lse.device != q.device:
            raise ValueError(f"lse is {tuple(lse.shape)} {lse.dtype}, expected {tuple(q.shape[:3])} float32")
        call.set_out(_usable(out), lse.contiguous())
        return _backward(call, dout, slope is not None)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slope, scale, cap, pos_q, pos_k, doc_q, doc_k, causal, prefix):
        call = _Call(q, k, v, scale, cap, slope, pos_q, pos_k, doc_q, doc_k, causal, prefix)
        need = any(ctx.needs_input_grad[:4])
        out, lse = _forward(call, need, need)
        if need:
            # (the saved inputs are the caller's: autograd notices a change in place between the two passes)
            ctx.save_for_backward(q, k, v, slope, pos_q, pos_k, doc_q, doc_k, prefix, out, lse, call.rest)
            ctx.scalars = (scale, cap, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, slope, pos_q, pos_k, doc_q, doc_k, prefix, out, lse, rest = ctx.saved_tensors
        scale, cap, causal = ctx.scalars
        call = _Call(q, k, v, scale, cap, slope, pos_q, pos_k, doc_q, doc_k, causal, prefix)
        call.set_out(out, lse, rest)
        dq, dk, dv, dslope = _backward(call, dout, slope is not None and ctx.needs_input_grad[3])
        if dslope is not None and slope.dtype != torch.float32:
            dslope = dslope.to(slope.dtype)
        return dq, dk, dv, dslope, None, None, None, None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None, cap: float = 0.0,
              slope: Optional[torch.Tensor] = None, pos_q: Optional[torch.Tensor] = None,
              pos_k: Optional[torch.Tensor] = None, doc_q: Optional[torch.Tensor] = None,
              doc_k: Optional[torch.Tensor] = None, causal: bool = False,
              prefix: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [B, H, Lq, D] over k, v [B, Hkv, Lk, D] (H a multiple of Hkv), differentiable in q, k, v and slope.

    ``scale``: default D ** -0.5.  ``cap`` > 0: scores pass through cap tanh(. / cap).  ``slope`` [H]: bias -slope dist,
    between the coordinates ``pos_q`` [B, Lq, 2] and ``pos_k`` [B, Lk, 2], or, without them, between positions
    (|i + Lk - Lq - j|).  ``doc_q`` [B, Lq] / ``doc_k`` [B, Lk]: whole numbers; tokens see their own document, negative ids
    are padding (such rows give zeros); int32 ids are taken as they are, int64 ones mapped to those in 15 us.  ``causal``: j <= i +
    Lk - Lq, and in front of ``prefix`` [B] everything.

    Under graph capture, leaves that collect gradients are refused: a leaf's accumulation belongs to the stream on which
    it was first used, and a captured backward pass that meets an eager graph of the same leaf ends the process.  Capture
    attention_forward and attention_backward instead."""
    if torch.is_grad_enabled():
        leaves = [t for t in (q, k, v, slope) if t is not None and t.requires_grad and t.is_leaf]
        if leaves and q.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("attention: a leaf that requires grad inside a graph capture; capture attention_forward "
                               "and attention_backward instead")
    if derivatives(pos_q, pos_k):
        no_derivatives("attention", pos_q=pos_q, pos_k=pos_k)
        with torch.no_grad():                    # (q, k, v and slope: in reverse mode only)
            no_derivatives("attention", q=q, k=k, v=v, slope=slope)
    if not torch.is_grad_enabled() or not (q.requires_grad or k.requires_grad or v.requires_grad or
                                           (slope is not None and slope.requires_grad)):
        return _forward(_Call(q, k, v, scale, cap, slope, pos_q, pos_k, doc_q, doc_k, causal, prefix), False)[0]
    return _Attention.apply(q, k, v, slope, scale, cap, pos_q, pos_k, doc_q, doc_k, causal, prefix)


class PagedCache:
    """Keys and values of ``batch`` sequences in pages (include/dgl_amd.h, dgl_kv_cache_t): pages [num_pages, kv_heads,
    page_size, head_dim], a table [batch, pages per sequence] and the live lengths.

    Without ``num_pages`` every sequence owns the pages for ``max_tokens`` from the start; with it, sequences share a pool
    and ``reserve`` / ``release`` move pages between them (host-side bookkeeping; the table is updated on the current
    stream).  Appends and attention never look at the lengths on the host."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, max_tokens: int, *, page_size: int = 64,
                 num_pages: Optional[int] = None, dtype: torch.dtype = torch.float32, device="cuda"):
        if batch < 1 or max_tokens < 1:
            raise ValueError(f"a cache of {batch} sequences of {max_tokens} tokens")
        per = (max_tokens + page_size - 1) // page_size
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"device {dev}: a GPU is expected")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        total = batch * per if num_pages is None else num_pages
        shape = (total, kv_heads, page_size, head_dim)
        table = torch.full((batch, per), -1, dtype=torch.int32, device=dev)
        self._set(torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev), table,
                  torch.zeros(batch, dtype=torch.int32, device=dev))
        self._owned = [[] for _ in range(batch)]
        self._free = list(range(total - 1, -1, -1))
        if num_pages is None:
            for b in range(batch):
                self._owned[b] = [self._free.pop() for _ in range(per)]
            table.copy_(torch.tensor(self._owned, dtype=torch.int32))

    @classmethod
    def over(cls, k_pages, v_pages, table, lengths) -> "PagedCache":
        """A cache over tensors that exist already (their owner manages the pages)."""
        self = cls.__new__(cls)
        self._set(k_pages, v_pages, table, lengths)
        self._owned = self._free = None
        return self

    def _set(self, k_pages, v_pages, table, lengths):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError(f"pages {tuple(k_pages.shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}: "
                             "equal [pages, heads, page size, head size] are expected")
        if k_pages.dtype not in _DTYPES:
            raise ValueError(f"{k_pages.dtype}: float32, float16 or bfloat16 is expected")
        dev = k_pages.device
        if table.dim() != 2 or lengths.dim() != 1 or lengths.shape[0] != table.shape[0]:
            raise ValueError(f"table {tuple(table.shape)} and lengths {tuple(lengths.shape)} do not fit")
        if table.dtype != torch.int32 or lengths.dtype != torch.int32:
            raise ValueError("table and lengths are int32")
        if dev.type != "cuda" or v_pages.device != dev or table.device != dev or lengths.device != dev:
            raise ValueError("pages, table and lengths belong on one GPU")
        if k_pages.stride(3) != 1 or v_pages.stride(3) != 1 or table.stride(1) != 1 or lengths.stride(0) != 1:
            raise ValueError("the head size, a row of the table and the lengths have to be consecutive")
        self.k_pages, self.v_pages, self.table, self.lengths = k_pages, v_pages, table, lengths
        self.device, self.dtype = dev, k_pages.dtype
        self.page_size, self.batch = k_pages.shape[2], table.shape[0]
        c = self.struct = _lib.KVCache()
        pages, heads, page_size, size = k_pages.shape
        _PACK_CACHE.pack_into(c, 0, _DTYPES[self.dtype], self.batch, heads, size, page_size, table.shape[1], pages,
                              *k_pages.stride()[:3], *v_pages.stride()[:3], table.stride(0), k_pages.data_ptr(),
                              v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr())

    # ---- pages of a pool ------------------------------------------------------------------
    def _pool(self, sequence: int):
        if self._free is None:
            raise ValueError("the pages of this cache are managed by their owner")
        if not 0 <= sequence < self.batch:
            raise ValueError(f"sequence {sequence}: the cache holds {self.batch}")

    def reserve(self, sequence: int, tokens: int) -> None:
        """Give ``sequence`` the pages for ``tokens`` tokens (those it has stay)."""
        self._pool(sequence)
        need = (tokens + self.page_size - 1) // self.page_size
        if need > self.table.shape[1]:
            raise ValueError(f"{tokens} tokens: a sequence holds at most {self.table.shape[1] * self.page_size}")
        own = self._owned[sequence]
        if need - len(own) > len(self._free):
            raise RuntimeError(f"{need - len(own)} pages wanted, {len(self._free)} are free")
        if need > len(own):
            have = len(own)
            own.extend(self._free.pop() for _ in range(need - have))
            self.table[sequence, have:need] = torch.tensor(own[have:need], dtype=torch.int32).to(self.device)

    def release(self, sequence: int) -> None:
        """Return the pages of ``sequence`` to the pool; it is empty afterwards."""
        self._pool(sequence)
        self._free.extend(reversed(self._owned[sequence]))
        self._owned[sequence] = []
        self.table[sequence].fill_(-1)
        self.lengths[sequence:sequence + 1].zero_()

    # ---- tokens ---------------------------------------------------------------------------
    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, *, counts: Optional[torch.Tensor] = None,
               start: Optional[torch.Tensor] = None) -> None:
        """Write new tokens [batch, kv heads, tokens, head size] behind each sequence (or from position ``start`` [batch]
        on) and set the lengths to their end.  ``counts`` [batch]: only the first counts[b] of a ragged batch.  Tokens
        beyond a sequence's pages are dropped, and its length ends before the first of them.  No gradient passes through a
        cache: tokens that require one are refused."""
        if derivatives(k_new, v_new):
            no_derivatives("PagedCache.append", k_new=k_new, v_new=v_new)
        with torch.no_grad():
            c = self.struct
            want = (self.batch, c.Hkv, k_new.shape[2] if k_new.dim() == 4 else -1, c.D)
            for name, t in (("k_new", k_new), ("v_new", v_new)):
                if tuple(t.shape) != want or t.dtype != self.dtype or t.device != self.device:
                    raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}, expected {want} {self.dtype} on {self.device}")
            k_new, v_new = _usable(k_new), _usable(v_new)
            counts = _side(counts, "counts", (self.batch,), torch.int32, self.device)
            start = self.lengths if start is None else _side(start, "start", (self.batch,), torch.int32, self.device)
            strides = (ctypes.c_int64 * 6)(*k_new.stride()[:3], *v_new.stride()[:3])
            _launch(self.device, _lib.load().dgl_cache_append, ctypes.byref(c), k_new.data_ptr(), v_new.data_ptr(),
                    ctypes.addressof(strides), ctypes.addressof(strides) + 24, want[2], start.data_ptr(), ptr(counts),
                    self.lengths.data_ptr(), what="dgl_cache_append")


def attention_step(q: torch.Tensor, cache: PagedCache, *, rows_per_instance: int = 1, scale: Optional[float] = None,
                   cap: float = 0.0, slope: Optional[torch.Tensor] = None, pos_q: Optional[torch.Tensor] = None,
                   pos_k: Optional[torch.Tensor] = None, blocked: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of one new token per row, q [R, H, D], over the cache of its instance (row r: sequence r //
    rows_per_instance).  ``cap`` / ``slope`` as in ``attention``; coordinates ``pos_q`` [R, 2] and ``pos_k`` [batch, n, 2]
    (n at least the live lengths), or, without them, the distance lengths[b] - 1 - j.  ``blocked`` int64 [R, words]: bit j of
    word j // 64 set = key j is not seen, as the states' visited words.  A row that sees nothing is zeros (lse -inf).  For
    serving: inputs that require grad are refused."""
    if derivatives(q, slope, pos_q, pos_k):
        no_derivatives("attention_step", q=q, slope=slope, pos_q=pos_q, pos_k=pos_k)
    c, dev = cache.struct, cache.device
    if q.dim() != 3 or q.shape[0] != cache.batch * rows_per_instance or q.shape[2] != c.D or q.shape[1] % c.Hkv or q.shape[1] < 1:
        raise ValueError(f"q has shape {tuple(q.shape)}: expected [{cache.batch} x {rows_per_instance}, a multiple of {c.Hkv}, {c.D}]")
    if q.dtype != cache.dtype or q.device != dev:
        raise ValueError(f"q is {q.dtype} on {q.device}, the cache {cache.dtype} on {dev}")
    if (pos_q is None) != (pos_k is None) or (pos_q is not None and slope is None):
        raise ValueError("coordinates are given for both sides and with a slope")
    q = _usable(q)
    R, H, D = q.shape
    out = torch.empty(R, H, D, dtype=q.dtype, device=dev)
    lse = torch.empty(R, H, dtype=torch.float32, device=dev) if return_lse else None
    slope = _side(slope, "slope", (H,), torch.float32, dev)
    n = pos_stride = words = bits_stride = 0
    if pos_q is not None:
        pos_q = _side(pos_q, "pos_q", (R, 2), torch.float32, dev)
        if pos_q.stride(0) != 2:             # rows of one wide tensor, or one row for all
            pos_q = pos_q.clone(memory_format=torch.contiguous_format)
        n = pos_k.shape[1] if pos_k.dim() == 3 else -1
        pos_k = _side(pos_k, "pos_k", (cache.batch, n, 2), torch.float32, dev)
        if pos_k.data_ptr() % 8 or pos_k.stride(0) % 2:
            pos_k = pos_k.clone(memory_format=torch.contiguous_format)
        pos_stride = pos_k.stride(0)
    if blocked is not None:
        if blocked.dim() != 2 or blocked.shape[0] != R or blocked.dtype != torch.int64 or blocked.device != dev:
            raise ValueError(f"blocked is {tuple(blocked.shape)} {blocked.dtype}: int64 words [{R}, n] on {dev} are expected")
        words = blocked.shape[1]
        if words > 1 and blocked.stride(1) != 1:
            blocked = blocked.contiguous()
        bits_stride = blocked.stride(0)
    a = _lib.AttentionStep()
    a.cache = c
    _PACK_STEP.pack_into(a, _STEP_AT, rows_per_instance, H, D ** -0.5 if scale is None else float(scale), _cap(cap),
                         *q.stride()[:2], H * D, D, q.data_ptr(), out.data_ptr(), ptr(lse), ptr(slope), ptr(pos_q),
                         ptr(pos_k), pos_stride, n, words, ptr(blocked), bits_stride)
    lib, ref = _lib.load(), ctypes.byref(a)
    need = lib.dgl_attention_step_workspace_floats(ref)
    ws = torch.empty(need, dtype=torch.float32, device=dev) if need > 0 else None
    _launch(dev, lib.dgl_attention_step, ref, ptr(ws), what="dgl_attention_step")
    return (out, lse) if return_lse else out
