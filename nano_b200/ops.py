"""Operators on device tensors: the binding of the nb200_dev_* entry points (include/nano_b200.h) for torch CUDA tensors.

    token_logprobs   log probabilities of given tokens with entropy and top alternatives, from rows of logits
    kv4_cache        a pool of pages for a key/value cache held in 4 bits (5 with the groups' pairs)
    kv4_write        rows of keys and values into such a pool
    kv4_read         what rows of a pool stand for
    kv4_attention    attention of queries over the pages of their sequences
    pages_copy       pages of a paged cache copied (forked, moved) in many pools at once

Calls run on the current stream of the tensors' device, wait for nothing and may be captured into a CUDA graph.  Outputs are new tensors.  Arguments that an operator
does not take are refused with NB200Error before anything is queued; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import engine as E
from .engine import NB200Error, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _need(ok, text, *args):
    if not ok:
        raise NB200Error(text % args if args else text)


class _on:
    """The device of `t` made current for a call (it is already, nearly always)."""

    def __init__(self, t):
        self.guard = None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _cuda(name, t, like=None):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, "%s is to be a CUDA tensor", name)
    _need(like is None or t.device == like.device, "%s is on another device", name)


def _check(rc):
    if rc != 0:
        E._check(rc)


def token_logprobs(logits, tokens, top=0):
    """logits [rows, vocab] (float32, bfloat16 or float16; rows may lie any stride apart), tokens [rows] (int32 or int64) ->
    (logprob [rows], entropy [rows], top_logprob [rows, top], top_id [rows, top]), float32 and int32; top <= 32.

    Alternatives are ordered by logit, equal ones by id.  -inf masks a token; a row of nothing but -inf has log probabilities -inf and entropy 0, one with NaN or
    +inf has NaN; a token outside the vocabulary has log probability NaN."""
    _cuda("logits", logits)
    _cuda("tokens", tokens, logits)
    _need(logits.dim() == 2 and logits.dtype in _TYPES, "logits are [rows, vocab] of float32, bfloat16 or float16")
    rows, vocab = logits.shape
    _need(vocab > 0 or rows == 0, "the vocabulary is empty")
    _need(tokens.shape == (rows,) and tokens.dtype in (torch.int32, torch.int64), "tokens are [rows] of int32 or int64")
    _need(0 <= top <= 32 and (top <= vocab or rows == 0), "%d alternatives asked for: at most 32, and no more than the vocabulary has", top)
    if rows and vocab > 1 and logits.stride(1) != 1 or logits.stride(0) < 0:
        logits = logits.contiguous()
    tokens = tokens.contiguous()
    both = torch.empty((2, rows), dtype=torch.float32, device=logits.device)
    top_logprob = torch.empty((rows, top), dtype=torch.float32, device=logits.device)
    top_id = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
    if rows:
        with _on(logits):
            at = both.data_ptr()
            _check(lib(True).nb200_dev_token_logprobs(at, at + 4 * rows, top_logprob.data_ptr() or None, top_id.data_ptr() or None, logits.data_ptr(), _TYPES[logits.dtype],
                                                      logits.stride(0), rows, vocab, tokens.data_ptr(), tokens.element_size(), top, _stream(logits)))
    return both[0], both[1], top_logprob, top_id


def pages_copy(pools, src, dst):
    """Page src[i] is copied over page dst[i] in every pool, in place.  pools: tensors [pages, ...] of any type, each page contiguous; src, dst: numbers on the host.
    A source may appear many times; a destination that is a source too or appears twice is refused."""
    pools = list(pools)
    src, dst = np.ascontiguousarray(src, np.int64), np.ascontiguousarray(dst, np.int64)
    _need(src.ndim == 1 and src.shape == dst.shape, "src and dst are lists of the same length")
    n = len(pools)
    if n == 0:
        return
    base, size, stride, pages = (C.c_void_p * n)(), (C.c_uint64 * n)(), (C.c_uint64 * n)(), (C.c_uint32 * n)()
    first = pools[0]
    for i, p in enumerate(pools):
        _cuda("pool %d" % i, p, first)
        _need(p.dim() >= 1 and (p.shape[0] == 0 or p[0].is_contiguous()), "pool %d: a page is to be contiguous", i)
        e = p.element_size()
        pages[i] = p.shape[0]
        size[i] = p[0].numel() * e if p.shape[0] else 0
        stride[i] = p.stride(0) * e if p.shape[0] > 1 else size[i]
        base[i] = p.data_ptr()
    most = min(pages)
    _need(src.size == 0 or (min(src.min(), dst.min()) >= 0 and max(src.max(), dst.max()) < most), "a page outside the smallest pool's %d", most)
    src, dst = src.astype(np.uint32), dst.astype(np.uint32)
    with _on(first):
        _check(lib(True).nb200_dev_pages_copy(base, size, stride, pages, n, E._p(src, E.u32p), E._p(dst, E.u32p), src.size, _stream(first)))


def kv4_cache(pages, kv_heads, head_dim, device="cuda"):
    """A pool of zeros: uint8 [pages, kv_heads, 40 * head_dim], pages of 32 tokens.  head_dim: a multiple of 32 up to 256."""
    _need(head_dim > 0 and head_dim % 32 == 0 and head_dim <= 256, "head_dim %d: a cache in 4 bits holds multiples of 32 up to 256", head_dim)
    return torch.zeros((pages, kv_heads, 40 * head_dim), dtype=torch.uint8, device=device)


def _pool(pool):
    _cuda("the pool", pool)
    _need(pool.dim() == 3 and pool.dtype == torch.uint8 and pool.shape[2] % 1280 == 0 and pool.shape[2] > 0, "a pool is uint8 [pages, kv_heads, 40 * head_dim]")
    _need(pool.stride(2) == 1 and (pool.stride(1) == pool.shape[2] or pool.shape[1] == 1), "a pool's pages are to be contiguous")
    return pool.shape[0], pool.shape[1], pool.shape[2] // 40


def _rows(call, pool, k, v, slots):
    pages, heads, dim = _pool(pool)
    r = E.Kv4Rows(pool.data_ptr(), pool.stride(0), pages, heads, dim, _TYPES[k.dtype], k.shape[0], slots.data_ptr(), k.data_ptr(), v.data_ptr(),
                  k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    with _on(pool):
        _check(call(C.byref(r), _stream(pool)))


def _slots(slots, pool):
    _cuda("slots", slots, pool)
    _need(slots.dim() == 1 and slots.dtype == torch.int32, "slots are [tokens] of int32")
    return slots.contiguous()


def kv4_write(pool, k, v, slots):
    """Row t of k and v ([tokens, kv_heads, head_dim], float32, bfloat16 or float16, any strides of rows and heads) goes to place slots[t] = page * 32 + place in the
    page of the pool, in place.  Rows whose slot lies outside the pool (-1: padding) are skipped; no slot may be given twice."""
    pages, heads, dim = _pool(pool)
    for name, x in (("k", k), ("v", v)):
        _cuda(name, x, pool)
        _need(x.dim() == 3 and tuple(x.shape[1:]) == (heads, dim) and x.dtype in _TYPES, "%s is [tokens, %d, %d] of float32, bfloat16 or float16", name, heads, dim)
    _need(k.shape == v.shape and k.dtype == v.dtype, "k and v are of one shape and type")
    slots = _slots(slots, pool)
    _need(slots.shape[0] == k.shape[0], "a slot for each row")
    if not k.shape[0]:
        return
    k, v = (x if x.stride(2) == 1 and x.stride(0) >= 0 and x.stride(1) >= 0 else x.contiguous() for x in (k, v))
    _rows(lib(True).nb200_dev_kv4_write, pool, k, v, slots)


def kv4_read(pool, slots, dtype=torch.float32):
    """What the places `slots` stand for: (k, v), [tokens, kv_heads, head_dim] each; zeros where a slot lies outside the pool."""
    pages, heads, dim = _pool(pool)
    slots = _slots(slots, pool)
    _need(dtype in _TYPES, "rows are float32, bfloat16 or float16")
    both = torch.empty((2, slots.shape[0], heads, dim), dtype=dtype, device=pool.device)
    k, v = both[0], both[1]
    if slots.shape[0]:
        _rows(lib(True).nb200_dev_kv4_read, pool, k, v, slots)
    return k, v


def kv4_attention(q, pool, table, lens, scale=None, window=0, block=0, softcap=0.0, sinks=None):
    """Attention over a cache held in 4 bits.  q [batch, tokens, heads, head_dim] (bfloat16 or float32) -> the same shape and type.

    Query t of sequence b sits at position lens[b] - tokens + t; lens [batch] (int32) counts all tokens of a sequence, the new ones (written before) among them;
    table [batch, width] (int32) names its pages.  Head h reads key/value head h // (heads / kv_heads).  A query sees the keys up to its own position, of these only the last
    `window` (0: all) and those in its own block of `block` positions (0: all).  scale: 1 / sqrt(head_dim) unless given; softcap > 0: softcap * tanh(score / softcap);
    sinks [heads] (float32): one more term exp(sink) in a head's denominator.  A query at a negative position or without a key in sight has zeros.  head_dim 32, 64, 96, 128
    or 256.  Products take 11-bit operands and sum in 32 bits, whichever type q has."""
    pages, heads, dim = _pool(pool)
    _cuda("q", q, pool)
    _cuda("table", table, pool)
    _cuda("lens", lens, pool)
    _need(q.dim() == 4 and q.dtype in (torch.float32, torch.bfloat16) and q.shape[3] == dim, "q is [batch, tokens, heads, %d] of bfloat16 or float32", dim)
    B, T, H, _ = q.shape
    _need(table.dim() == 2 and table.shape[0] == B and table.dtype == torch.int32, "table is [batch, width] of int32")
    _need(lens.shape == (B,) and lens.dtype == torch.int32, "lens is [batch] of int32")
    _need(window >= 0 and block >= 0, "window and block are not negative")
    if sinks is not None:
        _cuda("sinks", sinks, pool)
        _need(sinks.shape == (H,) and sinks.dtype == torch.float32, "sinks are [heads] of float32")
        sinks = sinks.contiguous()
    lens = lens.contiguous()
    if table.stride(1) != 1 and table.shape[1] > 1 or table.stride(0) < 0:
        table = table.contiguous()
    if q.stride(3) != 1 or min(q.stride()) < 0:
        q = q.contiguous()
    out = torch.empty((B, T, H, dim), dtype=q.dtype, device=q.device)
    p = E.Kv4Attention(q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), q.stride(2), T * H * dim, H * dim, dim, pool.data_ptr(), pool.stride(0), pages, heads, dim,
                       _TYPES[q.dtype], B, T, H, table.shape[1], table.stride(0), table.data_ptr() or None, lens.data_ptr(), None if sinks is None else sinks.data_ptr(),
                       dim ** -0.5 if scale is None else scale, softcap, window, block)
    L, need = lib(True), C.c_uint64(0)
    with _on(pool):
        _check(L.nb200_dev_kv4_attention_workspace(C.byref(p), C.byref(need)))
        room = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        _check(L.nb200_dev_kv4_attention(C.byref(p), None if room is None else room.data_ptr(), need.value, _stream(pool)))
    return out
