"""What lies in places of a cache in 4 bits that no query of a sequence sees -- behind its end, before its window, in its block's neighbours -- does not reach the result: whatever the bytes, the bits
are those of the same call over zeros there.  Tokens are given raw bytes, not rows that kv4_write has made: random ones, finite pairs whose c s + m leaves fp16, steps that the weights have no
room for, numbers that make scores large, and NaN."""
import pytest
import torch

from nano_b200 import ops
from test_gpu_device_ops import attention_reference, check_attention, filled, gen, near

pytestmark = pytest.mark.gpu

FORMS = [dict(), dict(window=40), dict(window=1), dict(block=48), dict(softcap=30.0), dict(softcap=3.0, window=77), dict(window=130, block=100, scale=-0.3)]


def unseen(table, lens, tokens, window=0, block=0, **_):
    """Places [batch, width * 32] that no query of their sequence sees."""
    at = torch.arange(32 * table.shape[1], device="cuda")[None]
    end, oldest = lens[:, None].long(), (lens[:, None].long() - tokens).clamp(min=0)
    low = torch.zeros_like(oldest)
    if window:
        low = torch.maximum(low, oldest - window + 1)
    if block:
        low = torch.maximum(low, oldest // block * block)
    return (at >= end) | (at < low)


def tokens_of(pool, dim):
    """Views [pages, heads, 32, ...] of a pool's key codes, key pairs, value codes and value pairs."""
    n = dim // 32
    cut = [0, 512 * n, 640 * n, 1152 * n, 1280 * n]
    part = [pool[..., a:b].unflatten(-1, (32, (b - a) // 32)) for a, b in zip(cut, cut[1:])]
    return part[0], part[1].view(torch.float16), part[2], part[3].view(torch.float16)


def put(pool, dim, places, kind, g):
    """The tokens at `places` [pages, 32] hold `kind` in all heads."""
    at = places[:, None].expand(-1, pool.shape[1], -1)
    count = int(at.sum())
    pair = {"zeros": (0.0, 0.0), "large": (60000.0, 60000.0), "small": (-60000.0, -60000.0), "steps": (3.0, 0.5), "far": (40.0, -300.0), "nan": (float("nan"), 1.0), "inf": (float("inf"), float("-inf"))}
    for x in tokens_of(pool, dim):
        if kind == "random":
            raw = x.view(torch.uint8)
            raw[at] = torch.randint(0, 256, (count, raw.shape[-1]), dtype=torch.uint8, device="cuda", generator=g)
        elif x.dtype == torch.uint8:
            x[at] = 0 if kind == "zeros" else 255
        else:
            x[at] = torch.tensor(pair[kind], dtype=torch.float16, device="cuda").repeat(x.shape[-1] // 2)


@pytest.mark.parametrize("kind", ["random", "large", "small", "steps", "far", "nan", "inf"])
@pytest.mark.parametrize("dim,heads,kv_heads,tokens", [(128, 4, 2, 60), (64, 6, 2, 150), (32, 5, 1, 30), (96, 4, 2, 20), (128, 4, 2, 1), (128, 8, 2, 3), (64, 8, 2, 4), (32, 5, 1, 1), (96, 2, 2, 1), (96, 6, 2, 3),
                                                          (256, 4, 1, 1), (256, 4, 1, 4), (256, 6, 2, 50)])
def test_bytes_that_nobody_sees(dim, heads, kv_heads, tokens, kind):
    g = gen(dim + tokens)
    pages = 40
    table = torch.randperm(pages, device="cuda", generator=g)[:36].view(3, 12).int()
    lens = torch.tensor([75, 333, 31], dtype=torch.int32, device="cuda")
    clean = filled(g, pages, kv_heads, dim)
    # Beside what attention_reference counts, a value c s + m is p s, rounded to 11 bits, times c and p times m: off by 2^-11 of c s, which is no larger than a group's range, even where c s + m is 0
    extra = 2.0 ** -11 * 1.01 * max(float(x.max() - x.min()) for x in ops.kv4_read(clean, torch.arange(pages * 32, dtype=torch.int32, device="cuda")))
    q = torch.randn(3, tokens, heads, dim, device="cuda", generator=g).bfloat16()
    sinks = torch.randn(heads, device="cuda", generator=g)
    for i, kw in enumerate(FORMS):
        kw = dict(kw, sinks=sinks) if i % 2 else kw
        places = torch.ones(pages, 32, dtype=torch.bool, device="cuda")
        places[table.flatten().long()] = unseen(table, lens, tokens, **kw).view(-1, 32)
        pool = clean.clone()
        put(pool, dim, places, "zeros", g)
        want = ops.kv4_attention(q, pool, table, lens, **kw)
        right, tol = attention_reference(q, pool, table, lens, **dict(dict(scale=dim ** -0.5), **kw))
        near(want, right, tol + extra, "attention over zeros")
        put(pool, dim, places, kind, g)
        got = ops.kv4_attention(q, pool, table, lens, **kw)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), (kw, (got != want).sum().item(), got.isnan().sum().item())


@pytest.mark.parametrize("tokens", [1, 40])
def test_pages_before_the_window_may_be_gone(tokens):
    """A page all of whose tokens lie before the window may be another sequence's by now, or no page at all."""
    g, dim = gen(5), 128
    pool = filled(g, 20, 2, dim)
    table = torch.arange(20, device="cuda").view(2, 10).int()
    lens = torch.tensor([317, 300], dtype=torch.int32, device="cuda")
    q = torch.randn(2, tokens, 4, dim, device="cuda", generator=g).bfloat16()
    want = check_attention(q, pool, table, lens, window=64)
    first = (lens.long() - tokens - 63) // 32
    gone = torch.arange(10, device="cuda")[None] < first[:, None]
    for other in (-1, 20, 1 << 30, 0):
        got = ops.kv4_attention(q, pool, torch.where(gone, other, table).int(), lens, window=64)
        assert torch.equal(got, want), other
