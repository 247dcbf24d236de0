"""Operators on device tensors: the binding of the nb200_dev_* entry points (include/nano_b200.h) for torch CUDA tensors.

    token_logprobs   log probabilities of given tokens with entropy and top alternatives, from rows of logits
    kv4_cache        a pool of pages for a key/value cache held in 4 bits (5 with the groups' pairs)
    kv4_write        rows of keys and values into such a pool
    kv4_read         what rows of a pool stand for
    kv4_attention    attention of queries over the pages of their sequences
    pages_copy       pages of a paged cache copied (forked, moved) in many pools at once

Calls run on the current stream of the tensors' device, wait for nothing and may be captured into a CUDA graph.  Outputs are new tensors, which carry no gradients.
Arguments that an operator does not take are refused with NB200Error before anything is queued; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import struct
from array import array

import torch

from . import engine as E
from .engine import NB200Error, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# the argument blocks nb200_kv4_rows and nb200_kv4_attention as bytes: a ctypes.Structure of as many fields takes four times as long to fill
_ROWS, _ATTENTION = struct.Struct("@QQIIIIIQQQQQQQ").pack, struct.Struct("@QQQQQQQQQQIIIIIIIIQQQQffII").pack
assert len(_ROWS(*[0] * 14)) == C.sizeof(E.Kv4Rows) and len(_ATTENTION(*[0] * 26)) == C.sizeof(E.Kv4Attention)
_stream_of, _device_now = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice          # (torch.cuda's functions of that purpose cost two microseconds a call)


def _no(text, *args):
    raise NB200Error(text % args if args else text)


def _cuda(name, t, device=None):
    """The device of a CUDA tensor, which is to be `device`."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        _no("%s is to be a CUDA tensor", name)
    d = t.get_device()
    if device is not None and d != device:
        _no("%s is on another device", name)
    return d


def _call(device, f, *args):
    """f(*args, stream) on the device and its current stream."""
    if device == _device_now():
        rc = f(*args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _stream_of(device))
    if rc:
        E._check(rc)


def token_logprobs(logits, tokens, top=0):
    """logits [rows, vocab] (float32, bfloat16 or float16; rows may lie any stride apart), tokens [rows] (int32 or int64) ->
    (logprob [rows], entropy [rows], top_logprob [rows, top], top_id [rows, top]), float32 and int32; top <= 32.

    Alternatives are ordered by logit, equal ones by id.  -inf masks a token; a row of nothing but -inf has log probabilities -inf and entropy 0, one with NaN or
    +inf has NaN; a token outside the vocabulary has log probability NaN."""
    device = _cuda("logits", logits)
    _cuda("tokens", tokens, device)
    kind = _TYPES.get(logits.dtype)
    if logits.dim() != 2 or kind is None:
        _no("logits are [rows, vocab] of float32, bfloat16 or float16")
    rows, vocab = logits.shape
    if rows and not vocab:
        _no("the vocabulary is empty")
    if tokens.dim() != 1 or tokens.shape[0] != rows or tokens.dtype not in (torch.int64, torch.int32):
        _no("tokens are [rows] of int32 or int64")
    if not 0 <= top <= 32 or (top > vocab and rows):
        _no("%d alternatives asked for: at most 32, and no more than the vocabulary has", top)
    if rows >> 32 or vocab >> 31:          # (counts are 32-bit numbers in the C calls: ctypes would cut larger ones off; struct refuses them)
        _no("%d rows of %d logits are too many for one call", rows, vocab)
    stride, step = logits.stride()
    if (step != 1 and vocab > 1) or stride < 0:
        logits = logits.contiguous()
        stride = vocab
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device)          # (sizes as a tuple cost a microsecond more each)
    entropy, top_logprob = torch.empty_like(logprob), logprob.new_empty(rows, top)
    top_id = torch.empty_like(top_logprob, dtype=torch.int32)
    if rows:
        _call(device, lib(True).nb200_dev_token_logprobs, logprob.data_ptr(), entropy.data_ptr(), top_logprob.data_ptr() or None, top_id.data_ptr() or None, logits.data_ptr(), kind,
              stride, rows, vocab, tokens.data_ptr(), tokens.element_size(), top)
    return logprob, entropy, top_logprob, top_id


def _numbers(pages):
    """Page numbers on the host as 32-bit numbers."""
    if getattr(pages, "is_cuda", False):
        _no("src and dst are lists of page numbers on the host")
    try:
        return array("I", pages.tolist() if hasattr(pages, "tolist") else pages)
    except OverflowError:
        _no("a page outside the pools")
    except (TypeError, ValueError):
        _no("src and dst are lists of page numbers")


def pages_copy(pools, src, dst):
    """Page src[i] is copied over page dst[i] in every pool, in place.  pools: tensors [pages, ...] of any type, each page contiguous; src, dst: numbers on the host.
    A source may appear many times; a destination that is a source too or appears twice is refused, and so are pools that share memory where a page that is written in one is read or written
    in another (x[:, 0] and x[:, 1] do not meet; x[:-1] and x[1:] may)."""
    pools = list(pools)
    src, dst = _numbers(src), _numbers(dst)
    if len(src) != len(dst):
        _no("src and dst are lists of the same length")
    if len(src) >> 32:
        _no("%d pairs are too many for one call", len(src))
    if not pools:
        return
    device = _cuda("pool 0", pools[0])
    base, size, stride, pages = [], [], [], []
    for i, p in enumerate(pools):
        if not isinstance(p, torch.Tensor) or p.get_device() != device or not p.dim():
            _cuda("pool %d" % i, p, device)
            _no("pool %d has no pages", i)
        count = p.shape[0]
        if p.is_contiguous():
            one = step = p.nbytes // count if count else 0
        else:
            if not p[0].is_contiguous() or p.stride(0) < 0:
                _no("pool %d: a page is to be contiguous", i)
            one = p[0].nbytes
            step = p.stride(0) * p.element_size() if count > 1 else one
        base.append(p.data_ptr())
        size.append(one)
        stride.append(step)
        pages.append(count)
    n = len(pools)
    numbers = array("Q", base + size + stride)
    try:
        counts = array("I", pages)
    except OverflowError:
        _no("pools of %d pages are too large", max(pages))
    at = numbers.buffer_info()[0]
    _call(device, lib(True).nb200_dev_pages_copy, at, at + 8 * n, at + 16 * n, counts.buffer_info()[0], n, src.buffer_info()[0], dst.buffer_info()[0], len(src))


def kv4_cache(pages, kv_heads, head_dim, device="cuda"):
    """A pool of zeros: uint8 [pages, kv_heads, 40 * head_dim], pages of 32 tokens.  head_dim: a multiple of 32 up to 256."""
    if not 0 < head_dim <= 256 or head_dim % 32:
        _no("head_dim %d: a cache in 4 bits holds multiples of 32 up to 256", head_dim)
    return torch.zeros((pages, kv_heads, 40 * head_dim), dtype=torch.uint8, device=device)


def _pool(pool):
    """(device, pages, kv_heads, head_dim, bytes from page to page)"""
    device = _cuda("the pool", pool)
    if pool.dim() != 3 or pool.dtype != torch.uint8 or pool.shape[2] % 1280 or not pool.shape[2]:
        _no("a pool is uint8 [pages, kv_heads, 40 * head_dim]")
    pages, heads, block = pool.shape
    if not pool.is_contiguous() and (pool.stride(2) != 1 or (pool.stride(1) != block and heads != 1)):
        _no("a pool's pages are to be contiguous")
    if (pages | heads) >> 32:
        _no("a pool of %d pages of %d heads is too large", pages, heads)
    return device, pages, heads, block // 40, pool.stride(0)


def _slots(slots, device):
    _cuda("slots", slots, device)
    if slots.dim() != 1 or slots.dtype != torch.int32:
        _no("slots are [tokens] of int32")
    if slots.is_contiguous():
        return slots
    if slots.shape[0] >> 32:
        _no("%d tokens are too many for one call", slots.shape[0])
    return slots.contiguous()


def _row_strides(x):
    """x with neighbouring coordinates, and its strides of rows and heads"""
    t, h, c = x.stride()
    if c != 1 or t < 0 or h < 0:
        x = x.contiguous()
        t, h, c = x.stride()
    return x, t, h


def kv4_write(pool, k, v, slots):
    """Row t of k and v ([tokens, kv_heads, head_dim], float32, bfloat16 or float16, any strides of rows and heads) goes to place slots[t] = page * 32 + place in the
    page of the pool, in place.  Rows whose slot lies outside the pool (-1: padding) are skipped; no slot may be given twice."""
    device, pages, heads, dim, stride = _pool(pool)
    for name, x in (("k", k), ("v", v)):
        _cuda(name, x, device)
        if x.dim() != 3 or x.shape[1] != heads or x.shape[2] != dim or x.dtype not in _TYPES:
            _no("%s is [tokens, %d, %d] of float32, bfloat16 or float16", name, heads, dim)
    tokens = k.shape[0]
    if v.shape[0] != tokens or k.dtype != v.dtype:
        _no("k and v are of one shape and type")
    slots = _slots(slots, device)
    if slots.shape[0] != tokens:
        _no("a slot for each row")
    if not tokens:
        return
    k, kt, kh = _row_strides(k)
    v, vt, vh = _row_strides(v)
    if tokens >> 32:
        _no("%d tokens are too many for one call", tokens)
    rows = _ROWS(pool.data_ptr(), stride, pages, heads, dim, _TYPES[k.dtype], tokens, slots.data_ptr(), k.data_ptr(), v.data_ptr(), kt, kh, vt, vh)
    _call(device, lib(True).nb200_dev_kv4_write, rows)


def kv4_read(pool, slots, dtype=torch.float32):
    """What the places `slots` stand for: (k, v), [tokens, kv_heads, head_dim] each; zeros where a slot lies outside the pool."""
    device, pages, heads, dim, stride = _pool(pool)
    slots = _slots(slots, device)
    kind = _TYPES.get(dtype)
    if kind is None:
        _no("rows are float32, bfloat16 or float16")
    tokens = slots.shape[0]
    k = pool.new_empty(tokens, heads, dim, dtype=dtype)
    v = torch.empty_like(k)
    if tokens:
        rows = _ROWS(pool.data_ptr(), stride, pages, heads, dim, kind, tokens, slots.data_ptr(), k.data_ptr(), v.data_ptr(), heads * dim, dim, heads * dim, dim)
        _call(device, lib(True).nb200_dev_kv4_read, rows)
    return k, v


def kv4_attention(q, pool, table, lens, scale=None, window=0, block=0, softcap=0.0, sinks=None):
    """Attention over a cache held in 4 bits.  q [batch, tokens, heads, head_dim] (bfloat16 or float32) -> the same shape and type.

    Query t of sequence b sits at position lens[b] - tokens + t; lens [batch] (int32) counts all tokens of a sequence, the new ones (written before) among them;
    table [batch, width] (int32) names its pages.  Head h reads key/value head h // (heads / kv_heads).  A query sees the keys up to its own position, of these only the last
    `window` (0: all) and those in its own block of `block` positions (0: all).  scale: 1 / sqrt(head_dim) unless given; softcap > 0: softcap * tanh(score / softcap);
    sinks [heads] (float32): one more term exp(sink) in a head's denominator.  A query at a negative position or without a key in sight has zeros; places that no query sees may hold any bytes.  head_dim 32, 64, 96, 128
    or 256.  Products take 11-bit operands and sum in 32 bits, whichever type q has."""
    device, pages, heads, dim, stride = _pool(pool)
    _cuda("q", q, device)
    _cuda("table", table, device)
    _cuda("lens", lens, device)
    kind = _TYPES.get(q.dtype, 2)
    if q.dim() != 4 or kind == 2 or q.shape[3] != dim:
        _no("q is [batch, tokens, heads, %d] of bfloat16 or float32", dim)
    B, T, H, _ = q.shape
    if table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32:
        _no("table is [batch, width] of int32")
    if lens.dim() != 1 or lens.shape[0] != B or lens.dtype != torch.int32:
        _no("lens is [batch] of int32")
    if (B | T | H) >> 32:
        _no("%d sequences of %d tokens of %d heads are too many for one call", B, T, H)
    if window < 0 or block < 0:
        _no("window and block are not negative")
    if sinks is not None:
        _cuda("sinks", sinks, device)
        if sinks.dim() != 1 or sinks.shape[0] != H or sinks.dtype != torch.float32:
            _no("sinks are [heads] of float32")
        sinks = sinks.contiguous()
    if not lens.is_contiguous():
        lens = lens.contiguous()
    if (table.stride(1) != 1 and table.shape[1] > 1) or table.stride(0) < 0:
        table = table.contiguous()
    qb, qt, qh, qd = q.stride()
    if qd != 1 or qb < 0 or qt < 0 or qh < 0:
        q = q.contiguous()
        qb, qt, qh, qd = q.stride()
    out = q.new_empty(B, T, H, dim)
    try:
        p = _ATTENTION(q.data_ptr(), out.data_ptr(), qb, qt, qh, T * H * dim, H * dim, dim, pool.data_ptr(), stride, pages, heads, dim, kind, B, T, H, table.shape[1], table.stride(0),
                       table.data_ptr(), lens.data_ptr(), 0 if sinks is None else sinks.data_ptr(), dim ** -0.5 if scale is None else scale, softcap, window, block)
    except (struct.error, OverflowError):
        _no("scale and softcap are numbers of 32 bits, window and block whole ones")
    L, need = lib(True), C.c_uint64()
    _call(device, _workspace, L, p, need)
    room = pool.new_empty(need.value) if need.value else None
    _call(device, L.nb200_dev_kv4_attention, p, None if room is None else room.data_ptr(), need.value)
    return out


def _workspace(L, p, need, stream):
    return L.nb200_dev_kv4_attention_workspace(p, C.byref(need))
