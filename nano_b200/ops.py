"""Operators on device tensors: the binding of the nb200_dev_* entry points (include/nano_b200.h) for torch CUDA tensors.

    token_logprobs   log probabilities of given tokens with entropy and top alternatives, from rows of logits
    kv4_cache        a pool of pages for a key/value cache held in 4 bits (5 with the groups' pairs)
    kv4_write        rows of keys and values into such a pool
    kv4_read         what rows of a pool stand for
    kv4_attention    attention of queries over the pages of their sequences
    pages_copy       pages of a paged cache copied (forked, moved) in many pools at once
    mx4_quantize     rows in microscaled 4-bit floating point (Mx4)
    mx4_read         what such rows stand for
    mx4_product      rows times a matrix in that format
    experts_sort     which rows go to which expert (Routing)
    experts_gather   tokens' rows in the order of their experts
    experts_product  those rows times their experts' matrices in 4 bits
    experts_combine  experts' rows back to their tokens, weighted and summed

Calls run on the current stream of the tensors' device, wait for nothing and may be captured into a CUDA graph.  Outputs are new tensors; only those of experts_gather and experts_combine
carry gradients, backwards and once.
Arguments that an operator does not take are refused with NB200Error before anything is queued; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import struct
from array import array
from typing import NamedTuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import engine as E
from .engine import NB200Error, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# the argument blocks nb200_kv4_rows and nb200_kv4_attention as bytes: a ctypes.Structure of as many fields takes four times as long to fill
_ROWS, _ATTENTION = struct.Struct("@QQIIIIIQQQQQQQ").pack, struct.Struct("@QQQQQQQQQQIIIIIIIIQQQQffII").pack
_MX4_ROWS, _MX4_PRODUCT, _EXPERTS_ROWS = struct.Struct("@QQQQQQIII4x").pack, struct.Struct("@QQQQQQQQQQQQQIIIIII").pack, struct.Struct("@QQQQQQQIIIIIQQQQQ").pack
assert len(_MX4_ROWS(*[0] * 9)) == C.sizeof(E.Mx4Rows) and len(_MX4_PRODUCT(*[0] * 19)) == C.sizeof(E.Mx4Product) and len(_EXPERTS_ROWS(*[0] * 17)) == C.sizeof(E.ExpertsRows)
assert len(_ROWS(*[0] * 14)) == C.sizeof(E.Kv4Rows) and len(_ATTENTION(*[0] * 26)) == C.sizeof(E.Kv4Attention)
_U8 = torch.uint8
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


class Mx4(NamedTuple):
    """Rows of numbers in microscaled 4-bit floating point: groups of 32 neighbours share a scale, the last group is filled up with zeros.

    codes [..., 16 * groups] (uint8): two to a byte, the lower four bits first; a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  scales [..., groups] (uint8): E stands for 2^(E - 127), 255
    for NaN.  columns: how many numbers a row has; groups = ceil(columns / 32)."""
    codes: torch.Tensor
    scales: torch.Tensor
    columns: int


class Routing(NamedTuple):
    """Places of a list of experts' numbers [tokens, top], sorted by expert.  order [tokens * top] (int32): the places t * top + j by expert and, within one, ascending, then -1 for those without an
    expert; offsets [experts + 1] (int32): where each expert's rows begin in it; place [tokens, top] (int32): where in order a place stands, or -1."""
    order: torch.Tensor
    offsets: torch.Tensor
    place: torch.Tensor


def _rows_of(name, x):
    """A tensor [..., columns] of numbers as (device, tensor of neighbouring numbers, rows, columns, stride from row to row)."""
    device = _cuda(name, x)
    if x.is_neg() or x.is_conj():          # (a view that leaves that to whoever reads it)
        x = x.resolve_neg().resolve_conj()
    if x.dim() == 2:
        rows, columns = x.shape
        stride, one = x.stride()
        if (one != 1 and columns > 1) or stride < 0:
            x, stride = x.contiguous(), columns
    else:
        if not x.dim():
            _no("%s is [..., columns]", name)
        columns = x.shape[-1]
        x, stride = x.contiguous(), columns
        rows = x.numel() // columns if columns else 0
    if (rows | columns) >> 31:
        _no("%s: %d rows of %d are too many for one call", name, rows, columns)
    return device, x, rows, columns, stride


def _mx4(name, m, device=None):
    """(device, groups) of an Mx4"""
    if not isinstance(m, Mx4):
        _no("%s is an Mx4", name)
    codes, scales, columns = m
    at = _cuda(name, codes, device)
    groups, n = -(-columns // 32), codes.dim()
    shape, scale_shape = codes.shape, scales.shape
    if codes.dtype is not _U8 or scales.dtype is not _U8 or not n or scales.dim() != n or shape[-1] != 16 * groups or scale_shape[-1] != groups or \
            (shape[0] != scale_shape[0] if n == 2 else shape[:-1] != scale_shape[:-1]):
        _no("%s has uint8 codes [..., %d] and scales [..., %d] for %d columns", name, 16 * groups, groups, columns)
    if not (scales.is_cuda and scales.get_device() == at):
        _cuda(name, scales, at)
    if not (codes.is_contiguous() and scales.is_contiguous()) and ((codes.stride(-1) != 1 and groups) or (scales.stride(-1) != 1 and groups > 1)):
        _no("%s: a row's bytes are to be neighbours", name)
    return at, groups


def _mx4_rows(name, m):
    """The rows of an Mx4 as (device, codes [rows, ...], scales [rows, ...])."""
    device, groups = _mx4(name, m)
    codes, scales, columns = m
    if codes.dim() != 2:
        codes, scales = codes.reshape(-1, 16 * groups) if groups else codes.new_empty(0, 0), scales.reshape(-1, groups) if groups else scales.new_empty(0, 0)
    if codes.stride(0) < 0 or scales.stride(0) < 0:
        codes, scales = codes.contiguous(), scales.contiguous()
    if (codes.shape[0] | columns) >> 31:
        _no("%s: %d rows of %d are too many for one call", name, codes.shape[0], columns)
    return device, codes, scales


def mx4_quantize(x):
    """x [..., columns] (float32, bfloat16 or float16; rows of a matrix may lie any stride apart) as an Mx4.  Of a group's largest magnitude a the scale is 2^(floor(log2 a) - 2); a number becomes the
    nearest code, of two as near the one with an even number, and what lies beyond 6 becomes 6.  A group with a NaN or an infinity is NaN.  No gradient passes."""
    device, x2, rows, columns, stride = _rows_of("x", x)
    kind = _TYPES.get(x.dtype)
    if kind is None:
        _no("x is float32, bfloat16 or float16")
    groups = -(-columns // 32)
    if x.dim() == 2:          # (sizes as arguments: see token_logprobs)
        codes = x2.new_empty(rows, 16 * groups, dtype=torch.uint8)
        scales = codes.new_empty(rows, groups)
    else:
        codes = x2.new_empty((*x.shape[:-1], 16 * groups), dtype=torch.uint8)
        scales = codes.new_empty((*x.shape[:-1], groups))
    if rows and columns:
        _call(device, lib(True).nb200_dev_mx4_quantize, _MX4_ROWS(codes.data_ptr(), scales.data_ptr(), 16 * groups, groups, x2.data_ptr(), stride, kind, rows, columns))
    return Mx4(codes, scales, columns)


def mx4_read(m, dtype=torch.float32):
    """What an Mx4 stands for: [..., columns], without a gradient."""
    device, codes, scales = _mx4_rows("m", m)
    kind = _TYPES.get(dtype)
    if kind is None:
        _no("rows are float32, bfloat16 or float16")
    rows, columns = codes.shape[0], m.columns
    out = codes.new_empty(rows, columns, dtype=dtype) if m.codes.dim() == 2 else codes.new_empty((*m.codes.shape[:-1], columns), dtype=dtype)
    if rows and columns:
        _call(device, lib(True).nb200_dev_mx4_read, _MX4_ROWS(codes.data_ptr(), scales.data_ptr(), codes.stride(0), scales.stride(0), out.data_ptr(), columns, kind, rows, columns))
    return out


def _product(x, w, offsets, dtype):
    device, groups = _mx4("w", w)
    wc, ws, columns = w
    experts = 0
    if offsets is None:
        if wc.dim() != 2:
            _no("w is an Mx4 of [outputs, columns]")
        outputs, w_expert, ws_expert, w_stride, ws_stride = wc.shape[0], 0, 0, wc.stride(0), ws.stride(0)
    else:
        if wc.dim() != 3 or not wc.shape[0]:
            _no("w is an Mx4 of [experts, outputs, columns]")
        experts, outputs, _ = wc.shape
        w_expert, w_stride, _ = wc.stride()
        ws_expert, ws_stride, _ = ws.stride()
        _cuda("offsets", offsets, device)
        if offsets.dim() != 1 or offsets.shape[0] != experts + 1 or offsets.dtype != torch.int32:
            _no("offsets are [experts + 1] of int32")
        offsets = offsets.contiguous()
    if isinstance(x, Mx4):
        at, x2, xs = _mx4_rows("x", x)
        given_x, kind, rows, given = x.codes, 3, x2.shape[0], x.columns
        x_stride, xs_at, xs_stride = x2.stride(0), xs.data_ptr(), xs.stride(0)
        dtype = dtype or torch.bfloat16
    else:
        at, x2, rows, given, x_stride = _rows_of("x", x)
        given_x, kind, xs_at, xs_stride = x, _TYPES.get(x.dtype), 0, 0
        if kind is None:
            _no("x is float32, bfloat16, float16 or an Mx4")
        dtype = dtype or x.dtype
    if at != device:
        _no("x is on another device")
    if given != columns:
        _no("x has %d columns, w %d", given, columns)
    if offsets is not None and given_x.dim() != 2:
        _no("x is [rows, columns]")
    out_kind = _TYPES.get(dtype)
    if out_kind is None:
        _no("results are float32, bfloat16 or float16")
    out = x2.new_empty(rows, outputs, dtype=dtype) if given_x.dim() == 2 else x2.new_empty((*given_x.shape[:-1], outputs), dtype=dtype)
    if not rows or not outputs:
        return out.zero_() if out.numel() else out
    if not columns:
        return out.zero_()
    try:
        p = _MX4_PRODUCT(x2.data_ptr(), xs_at, x_stride, xs_stride, wc.data_ptr(), ws.data_ptr(), w_stride, ws_stride, w_expert, ws_expert, out.data_ptr(), outputs,
                         0 if offsets is None else offsets.data_ptr(), kind, out_kind, rows, outputs, columns, experts)
    except struct.error:
        _no("strides are not negative, counts numbers of 32 bits")
    L, need = lib(True), C.c_uint64()
    if L.nb200_dev_mx4_product_workspace(p, C.byref(need)):          # (sizes alone: no device is asked)
        E._check(-1)
    need = need.value
    room = wc.new_empty(need) if need else None
    _call(device, L.nb200_dev_mx4_product, p, room.data_ptr() if need else None, need)
    return out


def mx4_product(x, w, dtype=None):
    """x w^T: x [..., columns], an Mx4 or numbers (float32, bfloat16 or float16) that the call quantises as mx4_quantize does; w an Mx4 of [outputs, columns] -> [..., outputs] of dtype (x's; bfloat16
    where x is an Mx4).  Products are exact, sums have 32 bits.  No gradient goes to x, whether it asks for one or not."""
    return _product(x, w, None, dtype)


def experts_product(x, w, offsets, dtype=None):
    """Rows sorted by expert times their experts' matrices: x [rows, columns] as in mx4_product, w an Mx4 of [experts, outputs, columns], offsets [experts + 1] (int32, Routing.offsets): rows
    offsets[e] .. offsets[e + 1] - 1 are multiplied with w[e], what lies outside of all becomes zeros -> [rows, outputs].  At most 1024 experts.  No gradient goes to x,
    whether it asks for one or not: between experts_gather and experts_combine it ends here."""
    if offsets is None:
        _no("offsets are [experts + 1] of int32")
    return _product(x, w, offsets, dtype)


def experts_sort(ids, experts):
    """ids [tokens, top] or [tokens] (int32 or int64): the experts of each token, in [0, experts); other numbers name none -> Routing.  At most 1024 experts."""
    device = _cuda("ids", ids)
    if ids.dim() not in (1, 2) or ids.dtype not in (torch.int64, torch.int32):
        _no("ids are [tokens, top] of int32 or int64")
    if not 0 < experts <= 1024:
        _no("%d experts: 1 to 1024", experts)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    n = ids.numel()
    if n >> 31:
        _no("%d places are too many for one call", n)
    place = torch.empty_like(ids, dtype=torch.int32)
    order, offsets = place.new_empty(n), place.new_empty(experts + 1)
    _call(device, lib(True).nb200_dev_experts_sort, order.data_ptr(), offsets.data_ptr(), place.data_ptr(), ids.data_ptr(), ids.element_size(), n, experts)
    return Routing(order, offsets, place)


def _routing(routing, device):
    """(order, place, tokens, top), contiguous"""
    if not isinstance(routing, Routing):
        _no("a routing is what experts_sort gives")
    order, _, place = routing
    _cuda("order", order, device)
    _cuda("place", place, device)
    shape, n = place.shape, order.shape[0] if order.dim() == 1 else -1
    if order.dtype is not torch.int32 or place.dtype is not torch.int32 or len(shape) not in (1, 2) or place.numel() != n:
        _no("a routing has order [tokens * top] and place [tokens, top] of int32")
    if n >> 31:
        _no("%d places are too many for one call", n)
    return order if order.is_contiguous() else order.contiguous(), place if place.is_contiguous() else place.contiguous(), shape[0], shape[1] if len(shape) == 2 else 1


def _gather(x, order, tokens, top):
    """Rows order[r] / top of x [tokens, columns], any type."""
    device, x, rows, columns, stride = _rows_of("x", x)
    if rows != tokens:
        _no("x has %d rows for %d tokens", rows, tokens)
    n, size = order.shape[0], x.element_size()
    out = x.new_empty(n, columns)
    if out.numel():
        _call(device, lib(True).nb200_dev_experts_gather, out.data_ptr(), columns * size, x.data_ptr(), stride * size, columns * size, order.data_ptr(), n, top, tokens)
    return out


def _combine(y, place, weights, tokens, top):
    device, y, rows, columns, stride = _rows_of("y", y)
    out = y.new_empty(tokens, columns)
    if out.numel():
        _call(device, lib(True).nb200_dev_experts_combine, _EXPERTS_ROWS(out.data_ptr(), columns, y.data_ptr(), stride, 0 if weights is None else weights.data_ptr(), place.data_ptr(), 0,
                                                                         _TYPES[y.dtype], tokens, top, rows, columns, 0, 0, 0, 0, 0))
    return out


def _no_tangents(*inputs):
    """No derivatives in forward mode (which autograd.Function is not asked for where no input requires a gradient)."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in inputs):
        _no("the operators of experts have no derivatives in forward mode")


def _once(grad, *factors):
    """No gradient of a gradient, by the one that comes in or by what it is multiplied with."""
    _no_tangents(grad)
    if torch.is_grad_enabled() and (grad.requires_grad or any(f is not None and f.requires_grad for f in factors)):
        _no("the operators of experts have no gradients of gradients")


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, place, tokens, top):
        ctx.save_for_backward(place)          # (so that a routing changed in between is noticed)
        ctx.sizes = tokens, top
        return _gather(x, order, tokens, top)

    @staticmethod
    def backward(ctx, grad):
        _once(grad)
        return _combine(grad, ctx.saved_tensors[0], None, *ctx.sizes), None, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, place, tokens, top):
        by_y, by_weights = ctx.needs_input_grad[:2]
        ctx.save_for_backward(y if by_weights else None, weights if by_y else None, order, place)          # (what a gradient is multiplied with)
        ctx.sizes = tokens, top
        return _combine(y, place, weights, tokens, top)

    @staticmethod
    def backward(ctx, grad):
        y, weights, order, place = ctx.saved_tensors
        _once(grad, y, weights)
        tokens, top = ctx.sizes
        by_y, by_weights = ctx.needs_input_grad[:2]
        device, grad, _, columns, grad_stride = _rows_of("the gradient", grad)
        rows, y_stride = order.shape[0], 0
        if y is not None:
            _, y, _, _, y_stride = _rows_of("y", y)
        dy = grad.new_empty(rows, columns) if by_y else None
        dw = torch.empty_like(place, dtype=torch.float32) if by_weights else None
        _call(device, lib(True).nb200_dev_experts_combine_grad, _EXPERTS_ROWS(0, 0, 0 if y is None else y.data_ptr(), y_stride, 0 if weights is None else weights.data_ptr(), place.data_ptr(),
                                                                              order.data_ptr(), _TYPES[grad.dtype], tokens, top, rows, columns, grad.data_ptr(), grad_stride,
                                                                              0 if dy is None else dy.data_ptr(), columns, 0 if dw is None else dw.data_ptr()))
        return dy, dw, None, None, None, None


def experts_gather(x, routing):
    """Tokens' rows in the order of their experts: x [tokens, columns] (any type, or an Mx4) -> [tokens * top, columns], row r that of token order[r] / top, zeros behind the last place that has an
    expert.  A token's gradient is the sum, in 32 bits, of those of its rows (float32, bfloat16 and float16); forward mode is refused."""
    if isinstance(x, Mx4):
        device, _ = _mx4("x", x)
        order, _, tokens, top = _routing(routing, device)
        if x.codes.dim() != 2:
            _no("x is an Mx4 of [tokens, columns]")
        return Mx4(_gather(x.codes, order, tokens, top), _gather(x.scales, order, tokens, top), x.columns)
    order, place, tokens, top = _routing(routing, _cuda("x", x))
    if x.dim() != 2:
        _no("x is [tokens, columns]")
    _no_tangents(x)
    if x.requires_grad and torch.is_grad_enabled():
        if x.dtype not in _TYPES:
            _no("rows with gradients are float32, bfloat16 or float16")
        return _Gather.apply(x, order, place, tokens, top)
    return _gather(x, order, tokens, top)


def experts_combine(y, routing, weights=None):
    """Experts' rows back to their tokens: y [rows, columns] (float32, bfloat16 or float16), rows as experts_gather gives them, weights [tokens, top] (ones unless given) ->
    [tokens, columns], sum over j of weights[t, j] y[place[t, j]] in 32 bits, rounded once to y's type; a place without an expert adds nothing.  Gradients go to y and weights; forward mode is refused."""
    device = _cuda("y", y)
    order, place, tokens, top = _routing(routing, device)
    if y.dim() != 2 or y.shape[0] != order.shape[0] or y.dtype not in _TYPES:
        _no("y is [%d, columns] of float32, bfloat16 or float16", order.shape[0])
    if weights is not None:
        _cuda("weights", weights, device)
        if weights.shape != routing.place.shape or not weights.is_floating_point():
            _no("weights are [tokens, top] of numbers")
        if weights.dtype is not torch.float32 or not weights.is_contiguous() or weights.is_neg():
            weights = weights.float().contiguous().resolve_neg()
    _no_tangents(y, weights)
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(y, weights, order, place, tokens, top)
    return _combine(y, place, weights, tokens, top)
