"""Operators on device tensors: the binding of the nb200_dev_* entry points (include/nano_b200.h) for torch CUDA tensors.

    token_logprobs   log probabilities of given tokens with entropy and top alternatives, from rows of logits
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
