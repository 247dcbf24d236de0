"""Copies of pages in pools that share memory: refused where a page that is written in one lies over a page that is touched in another -- blocks run in any order, so the result would be whichever
came first -- and copied where pages only lie side by side."""
import itertools
import random

import pytest
import torch

from nano_b200 import engine as E

import ctypes as C
import numpy as np

EINVAL, ENODEV, BASE = -1, -3, 1 << 40          # BASE: an address that is never followed; what is not refused ends for want of a device


def call(pools, src, dst):
    """pools: (offset, page bytes, stride, pages) each"""
    n = len(pools)
    col = lambda i, t: (t * n)(*[p[i] for p in pools])
    s, d = np.asarray(src, np.uint32), np.asarray(dst, np.uint32)
    return E.lib().nb200_dev_pages_copy((C.c_void_p * n)(*[BASE + p[0] for p in pools]), col(1, C.c_uint64), col(2, C.c_uint64), col(3, C.c_uint32), n, E._p(s, E.u32p), E._p(d, E.u32p), s.size, None)


def meets(pools, src, dst):
    """by the bytes: is one that some pool's copy writes touched by another pool's copy.  The same pool twice is one pool"""
    pools = list({p[:3]: p for p in pools}.values())
    touch = []
    for o, b, s, _ in pools:
        touch.append((set(o + p * s + i for p in src for i in range(b)), set(o + p * s + i for p in dst for i in range(b))))
    return any(w & (r2 | w2) for (_, w), (r2, w2) in itertools.permutations(touch, 2))


@pytest.mark.skipif(E.device_count() > 0, reason="box has a GPU: addresses would be followed")
def test_refused_where_pages_meet_and_only_there():
    x = (0, 64, 64, 9)
    for pools, src, dst in [([x, (64, 64, 64, 9)], [0, 1], [5, 4]), ([x, (64, 64, 64, 9)], [0], [1]), ([x, (32, 64, 64, 9)], [0], [5]), ([(0, 128, 128, 9), x], [0, 1], [2, 5]), ([x, (512, 64, 64, 9)], [0], [8])]:
        assert meets(pools, src, dst)
        for order in (pools, pools[::-1]):
            assert call(order, src, dst) == EINVAL and b"overlap" in E.lib().nb200_last_error()
    for pools, src, dst in [([x, x], [0], [5]), ([x, x[:3] + (8,)], [0, 0], [5, 6]), ([x, (64, 64, 64, 9)], [0], [5]), ([x, (64, 64, 64, 9)], [0, 1], [6, 8]), ([(64 * i, 64, 256, 9) for i in (2, 0, 3, 1)], [0, 3], [1, 2]),
                            ([(0, 64, 200, 9), (64, 136, 200, 9)], [0], [8]), ([x, (10, 0, 0, 9)], [0], [5])]:
        assert not meets(pools, src, dst)
        assert call(pools, src, dst) == ENODEV, (pools, E.lib().nb200_last_error())
    rnd, seen = random.Random(1), {EINVAL: 0, ENODEV: 0}
    for _ in range(3000):
        pools = []
        for _ in range(rnd.randint(2, 4)):
            b = rnd.randint(1, 8)
            pools.append((rnd.randint(0, 60), b, rnd.choice([b, b + rnd.randint(0, 9), 12, 24]) if b <= 8 else b, 6))
        if any(p[2] < p[1] for p in pools):
            continue
        order = rnd.sample(range(6), 4)
        src, dst = order[:2], order[2:2 + rnd.randint(1, 2)]
        src = src[:len(dst)]
        want = EINVAL if meets(pools, src, dst) else ENODEV
        assert call(pools, src, dst) == want, (pools, src, dst)
        seen[want] += 1
    assert min(seen.values()) > 200, seen


@pytest.mark.gpu
def test_pools_of_one_tensor():
    from nano_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(0, 255, (12, 3, 4000), dtype=torch.uint8, device="cuda", generator=g)
    for pools in ([x[:, i] for i in (1, 0, 2)], [x, x], [x[:-1], x[1:]], [x.view(36, 4000)], [x[:, 0, :100], x[:, 0, 100:], x[:, 2]]):
        was = x.clone()
        want = was.clone()
        at = [p.storage_offset() for p in pools]
        for p, o in zip(pools, at):
            torch.as_strided(want, p.shape, p.stride(), o)[[5, 8]] = torch.as_strided(was, p.shape, p.stride(), o)[[0, 0]]
        ops.pages_copy(pools, [0, 0], [5, 8])
        assert torch.equal(x, want)
        x.copy_(was)
    was = x.clone()
    for pools, src, dst in [([x[:-1], x[1:]], [0], [1]), ([x[:-1], x[1:]], [0, 1], [5, 4]), ([x, x.view(36, 4000)], [0], [2]), ([x[:, 0], x.flatten(1)[:, 2000:6000]], [0], [7])]:
        with pytest.raises(E.NB200Error, match="overlap"):
            ops.pages_copy(pools, src, dst)
    assert torch.equal(x, was)
