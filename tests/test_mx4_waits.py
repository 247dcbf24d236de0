"""A tile whose depth is shared by the blocks of a cluster (k_mx4_few, products in microscaled 4-bit floating point), played through on the CPU in random orders with waits that run out: its results are the
whole sum or NaN, never a number made of something else, although a block's part lies where copies of its own that come late still land.  The steps are restated here; the order that they
rely on is looked for in the source."""
import math
import os
import random
import re

import pytest

from conftest import ROOT

SOURCE = re.sub(r"//.*", "", open(os.path.join(ROOT, "nano_b200", "csrc", "mx4_tc.cu")).read())
SUMMERS, STAGES, CODES = 4, 3, 1000.0          # warps that read sums out; what bytes of codes look like as a number


class Block:
    def __init__(self, part, steps, late):
        self.part, self.steps, self.late = part, steps, late          # late: steps whose copies come after everybody has stopped waiting for them
        self.ring, self.landed, self.sums, self.done, self.lost = [None] * SUMMERS, set(), 0, False, 0.0


class Cluster:
    def __init__(self, rnd, ks, steps, late, flagged):          # late: by block
        self.rnd, self.flagged = rnd, flagged
        self.blocks = [Block(q, steps, late.get(q, set())) for q in range(ks)]
        self.arrived, self.out, self.patience = [0, 0], {}, rnd.randint(5, 30) if late else math.inf

    def pause(self, most):
        for _ in range(self.rnd.randint(0, most)):
            yield

    def copies(self, b):
        """The stages in turn; a late copy lands at any time before the block ends."""
        flying = []
        for i in range(b.steps):
            t = 0
            while i - b.sums >= STAGES:          # the products have not given the stage back
                yield
                t += 1
                if t > self.patience:
                    break
            if t > self.patience:
                break
            if i in b.late:
                flying.append(i)
            else:
                b.landed.add(i)
            yield
        while flying:          # into the memory of the stages, whatever is there by now
            yield from self.pause(100)
            b.landed.add(flying.pop())
            b.ring[self.rnd.randrange(SUMMERS)] = CODES

    def products(self, b):
        for i in range(b.steps):
            t = 0
            while i not in b.landed:
                yield
                t += 1
                if t > self.patience:
                    return
            b.sums += 1
            yield
        b.done = True

    def summer(self, b, w):
        t, ok = 0, True
        while not b.done:
            yield
            t += 1
            if t > 2 * self.patience:
                ok = False
                break
        if not ok:
            b.lost = math.nan
        yield from self.pause(5)
        b.ring[w] = float(b.sums) if ok else math.nan
        yield from self.meet(0)
        got, none = 0.0, 0.0
        for peer in self.blocks:
            yield
            none += peer.lost
            got += peer.ring[w]
        self.out[b.part, w] = got + (none if self.flagged else 0.0)
        yield from self.meet(1)

    def meet(self, k):
        self.arrived[k] += 1
        while self.arrived[k] < SUMMERS * len(self.blocks):
            yield

    def play(self):
        todo = [x for b in self.blocks for x in [self.copies(b), self.products(b)] + [self.summer(b, w) for w in range(SUMMERS)]]
        steps = 0
        while todo:
            k = self.rnd.randrange(len(todo))
            try:
                next(todo[k])
            except StopIteration:
                todo.pop(k)
            steps += 1
            assert steps < 1_000_000, "somebody waits for ever"


def results(seed, ks, steps, with_late, flagged=True):
    rnd = random.Random(seed)
    late = {}
    if with_late:
        for q in rnd.sample(range(ks), rnd.randint(1, ks)):
            late[q] = set(rnd.sample(range(steps), rnd.randint(1, steps)))
    c = Cluster(rnd, ks, steps, late, flagged)
    c.play()
    return c, ks * steps


@pytest.mark.parametrize("ks", [2, 4, 8])
@pytest.mark.parametrize("steps", [1, 3, 7])
def test_a_shared_tile_is_whole_or_nan(ks, steps):
    lost = 0
    for seed in range(60):
        c, whole = results(seed, ks, steps, with_late=True)
        for got in c.out.values():
            assert got == whole or math.isnan(got)
        if any(math.isnan(b.lost) for b in c.blocks):
            lost += 1
            assert c.out and all(math.isnan(got) for got in c.out.values())
        c, whole = results(seed, ks, steps, with_late=False)
        assert c.out and all(got == whole for got in c.out.values())
    assert lost > 10


def test_a_part_that_is_nan_does_not_suffice():
    """Without the word of the block itself, copies that land in the part hide it: what the flag is for."""
    assert any(got != whole and not math.isnan(got) for seed in range(200) for c, whole in [results(seed, 4, 3, with_late=True, flagged=False)] for got in c.out.values())


def test_the_flag_is_that_of_the_source():
    few = SOURCE[SOURCE.index("k_mx4_few(const"):SOURCE.index("struct Many")]
    said, met, read = few.index("lost_s = NAN"), few.index("cluster_sync_all()"), few.index("finish_parts<16>(p, smem_u32(mine), smem_u32(&lost_s)")
    assert few.index("lost_s = 0.0f") < few.index("__syncthreads();\n    tc_fence_after();") < few.index("soon_warp(done, 0)") < said < few.index("mine[(c + j) * kRows] = f[j]") < met < read
    assert few.index("cluster_sync_all()", met + 1) > read and few.index("if (bad_s)") > read
    assert "finish_parts<4>(p, smem_u32(mine), smem_u32(&lost_s)" in few
    finish = SOURCE[SOURCE.index("void finish_parts("):SOURCE.index("template <int TN> struct Few")]
    assert "none += ld_cluster_f32(peer_lost)" in finish and finish.index("f[i] += none") < finish.index("put_rows<J>")
