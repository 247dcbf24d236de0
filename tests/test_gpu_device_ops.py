"""Operators on device memory (nano_b200.ops) against their definitions in 64 bits, at the sizes, masks, strides and values where they can go wrong.

Tolerances.  log p = (x - M) - log Z: the fp32 result rounds x - M and the difference once each, log Z carries the relative error of Z.  A thread adds k = vocab / 512
terms one after the other (256 threads, pairs of numbers; with 128 threads, only below 32768 numbers, vocab / 256, which is at most 64 more) (at most 2^-24 each), two dozen joins and the exponential (2^-22, and 2 |d| 2^-24 for its argument d = x - M, weighted by exp d) add the rest.
A cache in 4 bits is exact: its codes, pairs and values are fixed numbers.  Attention rounds keys, values, queries and weights to 11 significant bits (half a step
2^-11 each) and the output to its type."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from nano_b200 import ops
from nano_b200.engine import NB200Error

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------- log probabilities ----------------
def logprobs_reference(x, tokens, top):
    """In 64 bits; rows with NaN or +inf are NaN, rows of -inf alone -inf / 0; order of alternatives: value descending (NaN as -inf), index ascending."""
    x = x.double()
    bad = (x.isnan() | (x == math.inf)).any(1)
    order = torch.sort(torch.where(x.isnan(), -math.inf, x), dim=1, descending=True, stable=True)
    peak = order.values[:, :1]
    empty = (peak == -math.inf)[:, 0]
    d = x - torch.where(empty[:, None], 0.0, peak)
    z = d.exp().sum(1)
    lz = torch.where(empty, 0.0, z.log())
    inside = (tokens >= 0) & (tokens < x.shape[1])
    lp = d.gather(1, tokens.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0] - lz
    lp = torch.where(empty, -math.inf, lp)
    p = d.exp() / torch.where(empty, 1.0, z)[:, None]
    h = torch.where(empty, 0.0, lz + (p * torch.where(p > 0, -d, 0.0)).sum(1))
    tl = torch.where(empty[:, None], -math.inf, order.values[:, :top] - torch.where(empty[:, None], 0.0, peak) - lz[:, None])
    nan = torch.full_like(lp, math.nan)
    return torch.where(bad | ~inside, nan, lp), torch.where(bad, nan, h), torch.where(bad[:, None], math.nan, tl), order.indices[:, :top].int()


def near(got, want, tol, what):
    got, want = got.double(), want.double()
    tol = tol if isinstance(tol, torch.Tensor) else torch.full_like(want, tol)
    same = (got == want) | (got.isnan() & want.isnan())
    ok = same | ((got - want).abs() <= tol)
    assert ok.all(), f"{what}: {(~ok).sum()} of {ok.numel()} off, worst {((got - want).abs() - tol)[~ok].max()} over the tolerance, at {torch.nonzero(~ok)[0].tolist()}"


def check_logprobs(x, tokens, top):
    lp, h, tl, ids = ops.token_logprobs(x, tokens, top=top)
    wlp, wh, wtl, wids = logprobs_reference(x, tokens, top)
    e, k = 2.0 ** -24, x.shape[1] / 512 + 64
    ent = torch.where(wh.isfinite(), wh, 0.0)
    rel = e * (k + 4 * ent)          # of Z: sum of p |d| is the entropy less log Z
    near(lp, wlp, (rel + 4 * e * (1 + wlp.abs() + ent)).nan_to_num(0, 0, 0), "log probability")
    near(h, wh, rel + 4 * e + 2 * ent * e * (k + 8), "entropy")
    near(tl, wtl, (rel[:, None] + 4 * e * (1 + wtl.abs() + ent[:, None])).nan_to_num(0, 0, 0), "alternatives")
    assert torch.equal(ids, wids)
    assert lp.dtype == h.dtype == tl.dtype == torch.float32 and ids.dtype == torch.int32
    again = ops.token_logprobs(x, tokens, top=top)
    assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip((lp, h, tl, ids), again))          # no order of arrival in it


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,rows,top", [(1, 3, 1), (2, 1, 0), (31, 5, 31), (33, 7, 32), (100, 700, 5), (4097, 3, 20), (8191, 2, 32), (32000, 64, 0), (50257, 9, 8), (151936, 1, 5), (151936, 150, 20), (4097, 593, 32), (16383, 592, 20), (20000, 600, 8)])
def test_logprobs(kind, vocab, rows, top):
    g = gen(vocab + rows)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(DT[kind])          # 16-bit rows are full of equal numbers
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    check_logprobs(x, tokens, top)
    check_logprobs(x, tokens.int(), min(top, 3))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("offset,pad", [(1, 0), (3, 5), (0, 1), (7, 8)])
@pytest.mark.parametrize("rows", [6, 700])
def test_logprobs_of_rows_anywhere(kind, offset, pad, rows):
    vocab = 5003
    x = (torch.randn(rows, vocab + pad + offset, device="cuda", generator=gen(5)) * 2).to(DT[kind])
    x[:, :offset] = math.nan          # what lies beside the rows is not looked at
    x[:, offset + vocab:] = math.nan
    check_logprobs(x[:, offset:offset + vocab], torch.arange(rows, device="cuda"), 20)
    check_logprobs(x.t().contiguous().t()[:, offset:offset + vocab], torch.arange(rows, device="cuda"), 4)


@pytest.mark.parametrize("times", [1, 40])
def test_logprobs_of_special_rows(times):
    V, low = 3000, torch.finfo(torch.float32).min
    x = torch.randn(16, V, device="cuda", generator=gen(1))
    x[0] = 0.5                                            # all equal: the first ids, log p = -log V
    x[1] = -math.inf                                      # nothing is left
    x[2, 1:] = -math.inf                                  # one token is left
    x[3, ::2] = -math.inf
    x[4, 17] = math.nan
    x[5, 17] = math.inf
    x[6] = low                                            # masked by the type's lowest number, all of it: a row of equal numbers
    x[7, 100:] = low
    x[8] = -0.0
    x[8, ::2] = 0.0                                       # zeros of both signs are equal
    x[9] = torch.arange(V, device="cuda").float()         # every vector beats the ones before
    x[10] = -torch.arange(V, device="cuda").float()
    x[11] = 3e38
    x[12, :] = -math.inf
    x[12, 2990:] = 1.0                                    # fewer left than asked for
    x[13] *= 1e30
    x[14, 5] = 1000.0                                     # all but certain
    x[15] = math.nan
    tokens = torch.tensor([0, 5, 0, 2, 3, 4, 9, 200, 1, 2999, 0, 7, 3, 11, 5, 1], device="cuda")
    x, tokens = x.repeat(times, 1), tokens.repeat(times)
    check_logprobs(x, tokens, 20)
    lp, h, tl, ids = ops.token_logprobs(x, tokens, top=3)
    assert lp[0].item() == pytest.approx(-math.log(V), abs=1e-6) and ids[0].tolist() == [0, 1, 2]
    assert lp[1] == -math.inf and h[1] == 0 and ids[1].tolist() == [0, 1, 2]
    assert lp[2] == 0 and h[2] == 0 and lp[3] == -math.inf
    assert lp[6].item() == pytest.approx(-math.log(V), abs=1e-6) and lp[7] == low


def test_logprobs_of_tokens_outside_the_vocabulary():
    x = torch.randn(4, 50, device="cuda")
    check_logprobs(x, torch.tensor([-1, 50, 1 << 40, 49], device="cuda"), 0)
    lp, h, _, _ = ops.token_logprobs(x, torch.tensor([-1, 50, -100, 49], device="cuda", dtype=torch.int32))
    assert lp[:3].isnan().all() and lp[3].isfinite() and h.isfinite().all()


def test_logprobs_of_many_rows_and_none():
    x = torch.randn(70001, 9, device="cuda", generator=gen(3))          # more rows than a grid's second dimension
    check_logprobs(x, torch.randint(0, 9, (70001,), device="cuda", generator=gen(4)), 2)
    out = ops.token_logprobs(x[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), top=4)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 4), (0, 4)]


def test_logprobs_refusals():
    x, t = torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for args, text in [((x, t[:1]), "tokens"), ((x, t.float()), "tokens"), ((x[0], t), "logits"), ((x.double(), t), "logits"), ((x, t, 9), "alternatives"), ((x, t, -1), "alternatives"),
                       ((x, t.cpu()), "CUDA tensor")]:
        with pytest.raises(NB200Error, match=text):
            ops.token_logprobs(*args)


# ---------------- copies of pages ----------------
@pytest.mark.parametrize("pairs", [1, 64, 65, 1024, 2500])
@pytest.mark.parametrize("shape,kind", [((40,), torch.uint8), ((3, 7), torch.uint8), ((2, 33), torch.float32), ((9000,), torch.bfloat16)])
def test_pages_copy(pairs, shape, kind):
    g = gen(pairs)
    pools = [torch.randint(0, 200, (2 * pairs + 1 + i, *shape), device="cuda", generator=g).to(kind) for i in range(3)]
    order = torch.randperm(2 * pairs + 1, generator=torch.Generator().manual_seed(1))
    src, dst = order[:pairs], order[pairs:2 * pairs]
    want = [p.clone() for p in pools]
    for p in want:
        p[dst.cuda()] = p[src.cuda()]
    ops.pages_copy(pools, src.tolist(), dst.numpy())
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_pages_copy_of_many_pools_of_all_sizes():
    """More pools than one launch takes, pages of sizes of their own, one source for several destinations, pages a stride apart."""
    pools = [torch.randint(0, 255, (9, 16 + 24 * i), device="cuda", dtype=torch.uint8) for i in range(70)]
    wide = torch.randint(0, 255, (9, 500), device="cuda", dtype=torch.uint8)
    pools += [wide[:, 4:260], torch.zeros(9, 0, device="cuda")]
    want = [p.clone() for p in pools]
    around = wide.clone()
    for p in want:
        p[[3, 7, 0]] = p[[5, 5, 8]]
    ops.pages_copy(pools, [5, 5, 8], [3, 7, 0])
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    assert torch.equal(wide[:, :4], around[:, :4]) and torch.equal(wide[:, 260:], around[:, 260:])


def test_pages_copy_beyond_32_bits():
    pool = torch.zeros(5000, 1 << 20, dtype=torch.uint8, device="cuda")          # 5 GB
    pool[4999] = torch.randint(0, 255, (1 << 20,), device="cuda", dtype=torch.uint8)
    ops.pages_copy([pool], [4999], [4500])
    assert torch.equal(pool[4500], pool[4999]) and int(pool[:4500].max()) == 0 and int(pool[4501:4999].max()) == 0


def test_pages_copy_refusals():
    pool = torch.zeros(6, 32, device="cuda")
    for src, dst, text in [([0], [0], "read"), ([0, 1], [2, 2], "twice"), ([0, 2], [2, 3], "read"), ([6], [0], "outside"), ([-1], [0], "outside"), ([0, 1], [2], "same length"),
                           ([1 << 32], [0], "outside"), (np.array([(1 << 32) + 1]), [0], "outside"), ([0.5], [1], "page numbers"), ([[0, 1]], [[2, 3]], "page numbers"), (3, 4, "page numbers"), (torch.tensor([0], device="cuda"), [1], "on the host"), ("ab", [1, 2], "page numbers")]:
        with pytest.raises(NB200Error, match=text):
            ops.pages_copy([pool], src, dst)
    with pytest.raises(NB200Error, match="outside"):
        ops.pages_copy([pool, pool[:3]], [4], [1])
    with pytest.raises(NB200Error, match="contiguous"):
        ops.pages_copy([pool.view(6, 4, 8).transpose(1, 2)], [0], [1])
    ops.pages_copy([], [0], [1])
    ops.pages_copy([pool], [], [])


# ---------------- the cache in 4 bits ----------------
def quantised(x):
    """(codes, s, m) of rows [..., D] by the definition, in 64 bits but for the roundings that it names."""
    x = x.float().unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    m, s = lo.half(), ((hi - lo) * torch.tensor(1.0 / 15.0, device=x.device)).half()
    c = torch.where(s[..., None] > 0, ((x.double() - m.double()[..., None]) / torch.where(s > 0, s, 1).double()[..., None]).round(), 0.0).clamp(0, 15)
    fine = (x.abs() <= 32768).all(-1)
    return c, torch.where(fine, s, math.nan), torch.where(fine, m, math.nan)


def stands_for(x):
    c, s, m = quantised(x)
    return (c * s.double()[..., None] + m.double()[..., None]).flatten(-2)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.double().nan_to_num(0), b.double().nan_to_num(0))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,heads,tokens", [(32, 1, 1), (64, 3, 33), (96, 2, 70), (128, 8, 300), (160, 1, 5), (224, 2, 3), (256, 4, 129)])
def test_kv4_rows(kind, dim, heads, tokens):
    g, pages = gen(dim), tokens // 32 + 3
    k, v = ((torch.randn(tokens, heads, dim, device="cuda", generator=g) * 2 + torch.randn(1, heads, dim, device="cuda", generator=g) * 5).to(DT[kind]) for _ in "kv")
    pool = torch.randint(0, 255, (pages, heads, 40 * dim), dtype=torch.uint8, device="cuda", generator=g)
    before = pool.clone()
    places = torch.randperm(pages * 32, device="cuda", generator=g)[:tokens].int()
    slots = places.clone()
    slots[1::3] = -1                                     # padding
    slots[2::7] = pages * 32                             # and places that the pool has not
    ops.kv4_write(pool, k, v, slots)
    live = (slots >= 0) & (slots < pages * 32)
    gk, gv = ops.kv4_read(pool, slots)
    assert same(gk, stands_for(k).float() * live[:, None, None]) and same(gv, stands_for(v).float() * live[:, None, None])
    # half the range's sixteenth, the pair's roundings beside it
    span = (k.float().unflatten(-1, (-1, 32)).amax(-1) - k.float().unflatten(-1, (-1, 32)).amin(-1))[..., None]
    far = (gk - k.float()).unflatten(-1, (-1, 32)).abs()[live]
    assert (far <= (span / 30 + span * 2.0 ** -10 + k.float().abs().amax() * 2.0 ** -11 + 1e-6)[live]).all()
    # nothing else has changed: written again over the old bytes, the pool is what it was
    rest = torch.ones(pages * 32, dtype=torch.bool, device="cuda")
    rest[slots[live].long()] = False
    others = torch.nonzero(rest)[:, 0].int()
    a, b = ops.kv4_read(pool, others), ops.kv4_read(before, others)
    assert same(a[0], b[0]) and same(a[1], b[1])
    for t in (torch.bfloat16, torch.float16):
        assert same(ops.kv4_read(pool, places, t)[1], ops.kv4_read(pool, places)[1].to(t))


def test_kv4_rows_at_the_borders_of_codes():
    """Numbers that lie on, just below and just above the borders between two codes."""
    s, m = 0.25, -2.0
    base = m + s * (torch.arange(16, dtype=torch.float64) + 0.5)
    x = torch.zeros(6, 1, 64, dtype=torch.float32)
    for i, step in enumerate((0, 1, -1, 3)):
        near_by = base.float()
        for _ in range(abs(step)):
            near_by = torch.nextafter(near_by, torch.tensor(math.inf if step > 0 else -math.inf))
        x[i, 0, :16], x[i, 0, 16:32] = near_by.clamp(m, m + 15 * s), torch.linspace(m, m + 15 * s, 16)
    x[4, 0] = 1.2345678                                   # a group of one number
    x[5, 0, :32] = torch.linspace(-1e-7, 1e-7, 32)        # below fp16's smallest step
    x[..., 32:] = x[..., :32].flip(-1) * 3.7
    x = x.cuda()
    pool = ops.kv4_cache(1, 1, 64)
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    ops.kv4_write(pool, x, x.flip(0).contiguous(), slots)
    k, v = ops.kv4_read(pool, slots)
    assert same(k, stands_for(x).float()) and same(v, stands_for(x.flip(0)).float())


def test_kv4_rows_of_all_magnitudes():
    e = torch.linspace(-40, 16, 4000, device="cuda")
    x = torch.randn(4000, 1, 32, device="cuda", generator=gen(2)) * torch.exp2(e)[:, None, None]
    x[5, 0, 3], x[6, 0, 3], x[7, 0, 3], x[8, 0, 3], x[9] = math.nan, math.inf, -math.inf, 40000.0, 32768.0
    pool, slots = ops.kv4_cache(125, 1, 32), torch.arange(4000, dtype=torch.int32, device="cuda")
    ops.kv4_write(pool, x, -x, slots)
    k, v = ops.kv4_read(pool, slots)
    assert same(k, stands_for(x).float()) and same(v, stands_for(-x).float())
    assert k[5:9].isnan().all() and (k[9] == 32768).all()


def test_kv4_rows_strides_and_refusals():
    pool = ops.kv4_cache(3, 2, 64)
    big = torch.randn(5, 6, 2, 70, device="cuda", generator=gen(8))
    k, v = big[:, 0, :, 3:67], big[:, 2, :, 6:70]                  # rows and heads strides apart, not on 16 bytes
    slots = torch.tensor([95, 0, 33, -1, 64], dtype=torch.int32, device="cuda")
    ops.kv4_write(pool, k, v, slots)
    gk, gv = ops.kv4_read(pool, slots)
    live = (slots >= 0)[:, None, None]
    assert same(gk, stands_for(k).float() * live) and same(gv, stands_for(v).float() * live)
    wide = torch.zeros(3, 3, 2560, dtype=torch.uint8, device="cuda")[:, :2]          # a pool's pages a stride apart
    ops.kv4_write(wide, k, v, slots)
    assert torch.equal(wide, pool)
    turned = k.permute(2, 1, 0).contiguous().permute(2, 1, 0)                  # coordinates that are not neighbours
    ops.kv4_write(wide, turned, v, slots)
    assert torch.equal(wide, pool)
    ops.kv4_write(pool, k[:0], v[:0], slots[:0])
    for args, text in [((pool, k[..., :32], v, slots), "k is"), ((pool, k, v.bfloat16(), slots), "one shape and type"), ((pool, k, v, slots[:2]), "a slot for each"), ((pool, k, v, slots.long()), "slots"),
                       ((pool[..., :100], k, v, slots), "a pool is"), ((pool.transpose(0, 1), k, v, slots), "contiguous|k is"), ((pool, k.cpu(), v, slots), "CUDA")]:
        with pytest.raises(NB200Error, match=text):
            ops.kv4_write(*args)
    with pytest.raises(NB200Error, match="multiples of 32"):
        ops.kv4_cache(1, 1, 48)


def rows_of(pool, table, n):
    """Keys and values [n, heads, dim] of one sequence, in 64 bits."""
    at = torch.arange(n, device="cuda")
    page = table[at // 32].long()
    slots = torch.where((page >= 0) & (page < pool.shape[0]), page * 32 + at % 32, -1).int()
    k, v = ops.kv4_read(pool, slots)
    return k.double(), v.double(), slots >= 0


def attention_reference(q, pool, table, lens, scale, window=0, block=0, softcap=0.0, sinks=None):
    """(out, tolerance) in 64 bits, from what kv4_read says the rows stand for.  With d the largest error of a score -- keys and queries off by 2^-11 each, the fp32 sum of D
    products beside it -- weights are off by the factor exp(2 d), rounded by 2^-11, and so are the values."""
    B, T, H, D = q.shape
    G = pool.shape[1]
    out, tol = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda"), torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = max(0, min(int(lens[b]), 32 * table.shape[1]))
        if not n:
            continue
        k, v, known = rows_of(pool, table[b], n)
        pos = n - T + torch.arange(T, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (j <= pos) & known[None]
        if window:
            seen &= j > pos - window
        if block:
            seen &= j // block == pos.clamp(min=0) // block
        for h in range(H):
            kk, vv = k[:, h // (H // G)], v[:, h // (H // G)]
            qq = q[b, :, h].double()
            s = qq @ kk.nan_to_num(0).T * scale
            off = (qq.abs() @ kk.nan_to_num(0).abs().T * abs(scale) * (2 * 2.0 ** -11 + D * 2.0 ** -24)).masked_fill(~seen, 0).amax(1, keepdim=True)
            if softcap:
                s, off = softcap * torch.tanh(s / softcap), off + softcap * 2.0 ** -21
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True)
            extra = 0.0
            if sinks is not None:
                top = torch.maximum(top, sinks[h].double())
                extra = (sinks[h].double() - top).exp()
            e = (s - top.clamp(min=-1e300)).exp()
            l = e.sum(1, keepdim=True) + extra
            p = torch.where(seen.any(1, keepdim=True), e / l, 0.0)
            poison = (seen & (kk.isnan().any(1) | vv.isnan().any(1))[None]).any(1)
            o = p @ vv.nan_to_num(0)
            out[b, :, h] = torch.where(poison[:, None], math.nan, o)
            tol[b, :, h] = (p @ vv.nan_to_num(0).abs()) * (torch.expm1(2 * off) + 2.0 ** -10 + 2.0 ** -18)
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -24
    return out, tol + (out.nan_to_num(0).abs() + tol) * half + 1e-30


def filled(g, pages, heads, dim, spread=1.0):
    pool = ops.kv4_cache(pages, heads, dim)
    k, v = (torch.randn(pages * 32, heads, dim, device="cuda", generator=g) * spread + torch.randn(1, heads, dim, device="cuda", generator=g) * 0.5 for _ in "kv")
    ops.kv4_write(pool, k, v, torch.arange(pages * 32, dtype=torch.int32, device="cuda"))
    return pool


def check_attention(q, pool, table, lens, scale=None, **kw):
    got = ops.kv4_attention(q, pool, table, lens, scale=scale, **kw)
    want, tol = attention_reference(q, pool, table, lens, q.shape[3] ** -0.5 if scale is None else scale, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    near(got, want, tol, "attention")
    assert torch.equal(ops.kv4_attention(q, pool, table, lens, scale=scale, **kw).view(torch.uint8), got.view(torch.uint8))
    return got


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (6, 2), (16, 1), (40, 2)])
def test_kv4_attention_of_single_tokens(kind, dim, heads, kv_heads):
    g = gen(dim + heads)
    lens = torch.tensor([1, 0, 31, 32, 33, 300, 1000], dtype=torch.int32, device="cuda")
    pool = filled(g, 7 * 32 + 3, kv_heads, dim)
    table = torch.randperm(7 * 32 + 3, device="cuda", generator=g)[:7 * 32].view(7, 32).int()
    q = (torch.randn(7, 1, heads, dim, device="cuda", generator=g) * 1.5).to(DT[kind])
    check_attention(q, pool, table, lens)


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("heads,tokens", [(4, 1), (4, 2), (16, 1), (5, 3)])
@pytest.mark.parametrize("width", [1, 5, 14])
def test_kv4_attention_of_short_contexts(dim, heads, tokens, width):
    g = gen(dim + width)
    pool = filled(g, 3 * width, 1, dim)
    table = torch.randperm(3 * width, device="cuda", generator=g).view(3, width).int()
    table[1, width // 2] = 3 * width + 5          # (a page that is none of the pool's)
    lens = torch.tensor([32 * width, 32 * width - 7, 1], dtype=torch.int32, device="cuda")
    q = torch.randn(3, tokens, heads, dim, device="cuda", generator=g).bfloat16()
    check_attention(q, pool, table, lens)
    check_attention(q, pool, table, lens, window=50, softcap=9.0, sinks=torch.randn(heads, device="cuda", generator=g))


@pytest.mark.parametrize("batch,width,tokens", [(9, 24, 1), (17, 31, 1), (20, 60, 1), (32, 40, 1), (33, 40, 2), (64, 20, 1), (65, 20, 1)])
def test_kv4_attention_of_many_sequences(batch, width, tokens):
    """Lengths of all kinds, equal ones, none at all, below zero and beyond the table among them, whatever order their blocks run in."""
    g = gen(batch)
    pool = filled(g, 100, 8, 32)
    table = torch.randint(0, 100, (batch, width), device="cuda", generator=g).int()          # (sequences may share pages)
    lens = torch.randint(1, 32 * width + 1, (batch,), device="cuda", generator=g).int()
    lens[1:batch:5] = 32 * width
    lens[2:batch:7] = lens[0]
    lens[3], lens[4], lens[7], lens[batch - 1] = 0, -3, 32 * width + 100, 2 ** 31 - 1
    q = torch.randn(batch, tokens, 16, 32, device="cuda", generator=g).bfloat16()
    check_attention(q, pool, table, lens)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,heads,kv_heads,tokens,context", [(128, 8, 8, 2, 50), (128, 16, 4, 3, 700), (64, 16, 4, 40, 40), (64, 4, 2, 129, 1500), (256, 4, 1, 70, 300), (32, 5, 1, 77, 99), (96, 8, 2, 33, 65), (128, 8, 2, 200, 201)])
def test_kv4_attention_of_portions(kind, dim, heads, kv_heads, tokens, context):
    g = gen(tokens)
    width = (context + 31) // 32
    pool = filled(g, 2 * width, kv_heads, dim)
    table = torch.randperm(2 * width, device="cuda", generator=g).view(2, width).int()
    lens = torch.tensor([context, max(1, context - tokens // 2 - 5)], dtype=torch.int32, device="cuda")          # (the second's first queries may lie before its start)
    q = torch.randn(2, tokens, heads, dim, device="cuda", generator=g).to(DT[kind])
    check_attention(q, pool, table, lens)


@pytest.mark.parametrize("tokens", [1, 5, 90])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=33), dict(window=100000), dict(block=16), dict(block=100), dict(block=64, window=20), dict(softcap=5.0), dict(softcap=20.0, window=77), dict(scale=0.0), dict(scale=-0.3)])
@pytest.mark.parametrize("sinks", [False, True])
def test_kv4_attention_masks_caps_and_sinks(tokens, kw, sinks):
    g = gen(7)
    pool = filled(g, 40, 2, 64, 2.0)
    table = torch.randperm(40, device="cuda", generator=g).view(2, 20).int()
    lens = torch.tensor([600, 129], dtype=torch.int32, device="cuda")
    q = torch.randn(2, tokens, 6, 64, device="cuda", generator=g).bfloat16()
    s = torch.tensor([0.0, -3.0, 5.0, 100.0, -math.inf, 1.0], device="cuda") if sinks else None
    check_attention(q, pool, table, lens, sinks=s, **kw)


@pytest.mark.parametrize("tokens", [1, 3, 60])
def test_kv4_attention_sees_nothing_that_it_should_not(tokens):
    """Bytes behind a sequence's end, pages of other numbers and rows before the window are full of NaN; page numbers outside the pool are not followed."""
    g, dim = gen(11), 128
    pool = filled(g, 30, 2, dim)
    good = pool.clone()
    table = torch.arange(20, device="cuda").view(2, 10).int()
    lens = torch.tensor([75, 200], dtype=torch.int32, device="cuda")
    pool[20:] = 255
    nan = torch.full((32, 2, dim), math.nan, device="cuda")
    ops.kv4_write(pool, nan[:21], nan[:21], torch.arange(75, 96, dtype=torch.int32, device="cuda"))          # behind the first sequence's end
    pool[3:10] = 255
    pool[17:20] = 255
    q = torch.randn(2, tokens, 4, dim, device="cuda", generator=g).bfloat16()
    if tokens <= 8:
        got = check_attention(q, pool, table, lens, window=40)
        assert got.isfinite().all()
    # the second sequence ends inside its seventh page: its last 24 rows are no one's
    pool = good.clone()
    ops.kv4_write(pool, nan[:24], nan[:24], torch.arange(10 * 32 + 200, 10 * 32 + 224, dtype=torch.int32, device="cuda"))
    got = check_attention(q, pool, table, lens)
    assert got.isfinite().all()
    lost = table.clone()
    lost[0, 1], lost[1, 4], lost[1, 0] = 30, -1, 1 << 30
    check_attention(q, pool, lost, lens)
    lost[:] = -5
    assert (check_attention(q, pool, lost, lens) == 0).all()


@pytest.mark.parametrize("tokens", [1, 6, 50])
@pytest.mark.parametrize("which", ["k", "v"])
def test_kv4_attention_shows_nan_where_it_is_seen(tokens, which):
    g, dim = gen(12), 64
    pool = filled(g, 8, 1, dim)
    row = torch.randn(1, 1, dim, device="cuda", generator=g)
    bad = row.clone()
    bad[0, 0, 40] = math.inf
    place = torch.tensor([3 * 32 + 5], dtype=torch.int32, device="cuda")
    ops.kv4_write(pool, bad if which == "k" else row, bad if which == "v" else row, place)
    q = torch.randn(1, tokens, 3, dim, device="cuda", generator=g).bfloat16()
    table = torch.arange(8, device="cuda").view(1, 8).int()
    for n in (101, 102, 125, 256):
        got = check_attention(q, pool, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
        pos = n - tokens + torch.arange(tokens, device="cuda")
        assert torch.equal(got.isnan().flatten(2).all(2)[0], pos >= 101) and torch.equal(got.isnan().flatten(2).any(2)[0], pos >= 101)
        check_attention(q, pool, table, torch.tensor([n], dtype=torch.int32, device="cuda"), window=30)


def test_kv4_attention_of_queries_of_all_magnitudes():
    g = gen(13)
    pool = filled(g, 8, 2, 128)
    table, lens = torch.arange(8, device="cuda").view(1, 8).int(), torch.tensor([250], dtype=torch.int32, device="cuda")
    for scale in (1e-30, 1e-6, 1.0, 3e4, 1e20):
        q = torch.randn(1, 2, 4, 128, device="cuda", generator=g) * scale
        check_attention(q, pool, table, lens, scale=0.1 / scale)
        check_attention(q.bfloat16(), pool, table, lens, scale=0.1 / scale)
    q[0, 0, 1, 5] = math.nan
    assert ops.kv4_attention(q, pool, table, lens)[0, 0, 1].isnan().all()
    assert (check_attention(torch.zeros(1, 2, 4, 128, device="cuda"), pool, table, lens)).isfinite().all()


def test_kv4_attention_far_into_a_long_context():
    """One sequence of 200001 tokens, pages scattered over a pool: the keys of a row shared by many blocks."""
    g, heads, dim = gen(14), 2, 128
    width = 200001 // 32 + 1
    pool = torch.randint(0, 255, (width, heads, 40 * dim), dtype=torch.uint8, device="cuda", generator=g)
    n = dim // 32
    pairs = torch.tensor([0.25, -2.0], dtype=torch.float16, device="cuda").view(torch.uint8).repeat(32 * n)
    pool[..., 512 * n:640 * n], pool[..., 1152 * n:] = pairs, pairs
    table = torch.randperm(width, device="cuda", generator=g).view(1, width).int()
    for tokens in (1, 9):
        q = torch.randn(1, tokens, 8, dim, device="cuda", generator=g).bfloat16()
        check_attention(q, pool, table, torch.tensor([200001], dtype=torch.int32, device="cuda"), scale=0.02)


def test_kv4_pools_beyond_32_bits():
    pages, heads, dim = 140_000, 8, 128          # 5.7 GB
    pool = ops.kv4_cache(pages, heads, dim)
    g = gen(15)
    k, v = (torch.randn(64, heads, dim, device="cuda", generator=g) for _ in "kv")
    slots = torch.arange((pages - 2) * 32, pages * 32, dtype=torch.int32, device="cuda")
    ops.kv4_write(pool, k, v, slots)
    got = ops.kv4_read(pool, slots)
    assert same(got[0], stands_for(k).float()) and same(got[1], stands_for(v).float()) and int(pool[:pages - 2].max()) == 0
    check_attention(torch.randn(1, 1, 16, dim, device="cuda", generator=g).bfloat16(), pool, torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda"), torch.tensor([60], dtype=torch.int32, device="cuda"))


def test_kv4_attention_strides_and_refusals():
    g = gen(16)
    pool, table, lens = filled(g, 6, 2, 64), torch.arange(12, device="cuda").view(2, 6).int()[:, :3] % 6, torch.tensor([90, 200], dtype=torch.int32, device="cuda")
    big = torch.randn(2, 4, 5, 9, 70, device="cuda", generator=g).bfloat16()
    q = big[:, :2, 1, 1:9:2, 3:67]
    got = check_attention(q, pool, table, lens)          # (200 tokens do not fit three pages: the length counts as 96)
    assert torch.equal(got, ops.kv4_attention(q.contiguous(), pool, table.contiguous(), lens))
    assert torch.equal(got, ops.kv4_attention(q.transpose(1, 3).contiguous().transpose(1, 3), pool, table, lens))
    assert ops.kv4_attention(q[:0], pool, table[:0], lens[:0]).shape == (0, 2, 4, 64) and ops.kv4_attention(q[:, :0], pool, table, lens).shape == (2, 0, 4, 64)
    assert (ops.kv4_attention(q, pool, table[:, :0], lens) == 0).all()
    for args, kw, text in [((q[..., :32], pool, table, lens), {}, "q is"), ((q.half(), pool, table, lens), {}, "q is"), ((q[:, :, :3], pool, table, lens), {}, "evenly"),
                           ((q, pool, table.long(), lens), {}, "table"), ((q, pool, table[:1], lens), {}, "table"), ((q, pool, table, lens.long()), {}, "lens"),
                           ((q, pool, table, lens), dict(window=-1), "window"), ((q, pool, table, lens), dict(softcap=-1.0), "softcap"), ((q, pool, table, lens), dict(sinks=torch.zeros(3, device="cuda")), "sinks"),
                           ((q, pool, table, lens), dict(scale=math.nan), "scale"), ((q, pool, table, lens), dict(scale=1e60), "scale"), ((q, pool, table, lens), dict(window=1 << 40), "window"),
                           ((q, pool, table, lens), dict(block=1.5), "block"), ((q, pool.cpu(), table, lens), {}, "CUDA"), ((q, pool, table, lens.cpu()), {}, "CUDA")]:
        with pytest.raises(NB200Error, match=text):
            ops.kv4_attention(*args, **kw)
    wide = ops.kv4_cache(2, 1, 160)
    with pytest.raises(NB200Error, match="no attention kernel"):
        ops.kv4_attention(torch.zeros(1, 1, 1, 160, device="cuda"), wide, table[:1], lens[:1])


# ---------------- together, on streams and in graphs ----------------
def run_of_all(st):
    """A step of a served batch: a forked page, the new tokens' rows, their attention, the scores of what follows."""
    ops.pages_copy([st["pool"]], [0, 0], [5, 6])
    ops.kv4_write(st["pool"], st["k"], st["v"], st["slots"])
    out = ops.kv4_attention(st["q"], st["pool"], st["table"], st["lens"])
    return (out, *ops.token_logprobs(out.flatten(1) @ st["w"], st["tokens"], top=4))


def state_of_all(seed):
    g = gen(seed)
    st = dict(pool=filled(g, 9, 2, 64))
    st["k"], st["v"] = (torch.randn(3, 2, 64, device="cuda", generator=g).bfloat16() for _ in "kv")
    st["table"] = torch.tensor([[0, 1], [5, 2], [6, 3]], dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor([40, 33, 64], dtype=torch.int32, device="cuda")
    at = st["lens"] - 1
    st["slots"] = (st["table"].gather(1, (at // 32)[:, None].long())[:, 0] * 32 + at % 32).int()
    st["q"] = torch.randn(3, 1, 8, 64, device="cuda", generator=g).bfloat16()
    st["w"] = torch.randn(512, 3001, device="cuda", generator=g).bfloat16()
    st["tokens"] = torch.tensor([5, 3000, 17], device="cuda")
    return st


def test_a_step_of_all_operators():
    st = state_of_all(20)
    prompt = ops.kv4_read(st["pool"], torch.arange(32, dtype=torch.int32, device="cuda"))
    out, lp, h, tl, ids = run_of_all(st)
    fork = ops.kv4_read(st["pool"], torch.arange(160, 192, dtype=torch.int32, device="cuda"))
    assert same(prompt[0], fork[0]) and same(prompt[1], fork[1])
    got = ops.kv4_read(st["pool"], st["slots"])
    assert same(got[0], stands_for(st["k"]).float()) and same(got[1], stands_for(st["v"]).float())
    want, tol = attention_reference(st["q"], st["pool"], st["table"], st["lens"], 64 ** -0.5)
    near(out, want, tol, "attention")
    check_logprobs(out.flatten(1) @ st["w"], st["tokens"], 4)


def test_captured_and_replayed():
    """Two graphs that share a memory pool, replayed in turn and beside eager calls, give the eager calls' bits."""
    a, b = state_of_all(21), state_of_all(22)
    want = [[t.clone() for t in run_of_all(s)] for s in (a, b)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run_of_all(s))
        graphs.append(graph)
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(outs[i], want[i]))
        assert torch.equal(run_of_all(a)[0], want[0][0])


def test_on_two_streams_at_once():
    states = [state_of_all(30 + i) for i in range(4)]
    want = [[t.clone() for t in run_of_all(s)] for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    got = [None] * 4
    for _ in range(20):
        for i, (s, stream) in enumerate(zip(states, streams)):
            with torch.cuda.stream(stream):
                got[i] = run_of_all(s)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(p.view(torch.uint8), r.view(torch.uint8)) for p, r in zip(x, y))


FIRST_CALLS = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from nano_b200 import ops
import test_gpu_device_ops as t
g = t.gen(7)
pool = ops.kv4_cache(40, 2, 64)
table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
k, v = (torch.randn(1280, 2, 64, device="cuda", generator=g) for _ in "kv")
slots = torch.arange(1280, dtype=torch.int32, device="cuda")
q = torch.randn(1, 300, 8, 64, device="cuda", generator=g).bfloat16()
lens = torch.tensor([1275], dtype=torch.int32, device="cuda")
w = torch.randn(512, 40001, device="cuda", generator=g).bfloat16()
x, tokens = torch.zeros(1, 40001, device="cuda"), torch.tensor([5], device="cuda")

def run():
    ops.kv4_write(pool, k, v, slots)
    one = ops.kv4_attention(q[:, -1:], pool, table, lens)
    many = ops.kv4_attention(q, pool, table, lens)
    ops.pages_copy([pool], [0], [39])
    return one, many, *ops.token_logprobs(x, tokens, top=5), *ops.token_logprobs(x.bfloat16(), tokens), *ops.kv4_read(pool, slots[:64])

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
got = [y.clone() for y in got]
pool.zero_()
assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, run()))
print("the same")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=os.path.dirname(here), tests=here)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]
