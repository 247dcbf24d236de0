"""The barriers of k_kv4_attn_tc (attention of long portions over a cache in 4 bits), played through on the CPU in random orders: no wait lets a warp pass before its time, no buffer is
written while somebody may still read it, and nobody waits for ever.  The steps of the three kinds of warps are restated here; which barrier is which is read from the source."""
import os
import random
import re

import pytest

from conftest import ROOT

SOURCE = re.sub(r"//.*", "", open(os.path.join(ROOT, "nano_b200", "csrc", "kv4_tc.cu")).read())
NAMES = {k: int(v) for k, v in re.findall(r"(\w+) = (\d+)", re.search(r"enum \{ (KFULL[^}]*)\}", SOURCE).group(1))}
KFULL, KFREE, VFULL, VFREE, SFULL, PREADY, ODONE, NBAR = (NAMES[k] for k in ("KFULL", "KFREE", "VFULL", "VFREE", "SFULL", "PREADY", "ODONE", "NBAR"))
MAKERS, SOFTMAX, PAGES = 7, 8, 4


class Barrier:
    """An mbarrier of `count` arrivals; a wait names the parity of the phase that is to be over."""
    def __init__(self, count):
        self.count, self.here, self.phase = count, 0, 0

    def arrive(self):
        self.here += 1
        assert self.here <= self.count
        if self.here == self.count:
            self.here, self.phase = 0, self.phase + 1

    def over(self, parity):
        return self.phase & 1 != parity


class Block:
    def __init__(self, tiles, rnd, moves):
        self.n, self.rnd, self.moves = tiles, rnd, moves          # moves: tiles at which the rows' reference moves
        self.bars = [Barrier(PAGES if k < KFREE or VFULL <= k < VFREE else SOFTMAX if PREADY <= k < ODONE else 1) for k in range(NBAR)]
        self.scores, self.weights, self.summed = [None, None], {}, -1
        self.keys, self.values, self.hidden, self.met = [None, None], [None, None], {}, {}

    def wait(self, bar, parity):
        while not self.bars[bar].over(parity):
            yield

    def pause(self, most):
        for _ in range(self.rnd.randint(0, most)):
            yield

    def make_scores(self, i):
        s = i & 1
        yield from self.wait(KFULL + s, i >> 1 & 1)
        assert self.keys[s] == (i, PAGES) and (self.scores[s] is None or (self.scores[s] == i - 2 and self.summed >= i - 2))
        self.scores[s] = i
        yield
        assert self.keys[s] == (i, PAGES)
        self.bars[KFREE + s].arrive()
        self.bars[SFULL + s].arrive()

    def products(self):
        for i in range(min(2, self.n)):
            yield from self.make_scores(i)
        for i in range(self.n):
            s = i & 1
            yield from self.wait(VFULL + s, i >> 1 & 1)
            yield from self.wait(PREADY + s, i >> 1 & 1)
            assert self.values[s] == (i, PAGES) and len(self.weights[i]) == SOFTMAX and self.scores[s] == i
            yield from self.pause(6)
            assert self.values[s] == (i, PAGES)
            self.summed = i
            self.bars[VFREE + s].arrive()
            self.bars[ODONE + s].arrive()
            if i + 2 < self.n:
                yield from self.wait(ODONE + s, i >> 1 & 1)
                yield from self.make_scores(i + 2)

    def maker(self, w):
        for q in range(w, 2 * PAGES * self.n, MAKERS):
            i, of_keys = q // (2 * PAGES), q % (2 * PAGES) < PAGES
            s = i & 1
            place, full, free = (self.keys, KFULL, KFREE) if of_keys else (self.values, VFULL, VFREE)
            if i >= 2:
                yield from self.wait(free + s, (i >> 1) - 1 & 1)
                assert of_keys or self.summed >= i - 2
            if place[s] is None or place[s][0] != i:
                assert place[s] is None or place[s] == (i - 2, PAGES)
                place[s] = (i, 0)
            if of_keys:
                self.hidden.setdefault(i & 3, {})[q % PAGES] = i
            yield
            place[s] = (i, place[s][1] + 1)
            self.bars[full + s].arrive()

    def softmax(self, w):
        half, quad, n = w >> 2, w & 3, self.n

        def whole(i):
            return self.scores[i & 1] == i and set(self.hidden[i & 3].values()) == {i}
        for i in range(n):
            yield from self.wait(SFULL + (i & 1), i >> 1 & 1)
            assert whole(i)
            self.met[half, quad] = i          # the named barrier of two warps
            while self.met.get((half ^ 1, quad), -1) < i:
                yield
            if i and i in self.moves:
                yield from self.wait(ODONE + (i - 1 & 1), i - 1 >> 1 & 1)
                assert self.summed == i - 1
            for _ in self.pause(3):
                yield
                assert whole(i)
            self.weights.setdefault(i, set()).add(w)
            yield
            self.bars[PREADY + (i & 1)].arrive()
        yield from self.pause(40)          # (a warp may come late to the end)
        if n > 1:
            yield from self.wait(ODONE + (n & 1), n - 2 >> 1 & 1)
        if n:
            yield from self.wait(ODONE + (n - 1 & 1), n - 1 >> 1 & 1)
        assert self.summed == n - 1


@pytest.mark.parametrize("tiles", [0, 1, 2, 3, 4, 5, 7, 10])
def test_no_order_of_steps_breaks_a_block(tiles):
    for seed in range(20):
        rnd = random.Random(1000 * tiles + seed)
        block = Block(tiles, rnd, set(range(tiles)) if seed % 3 == 0 else set(rnd.sample(range(tiles), tiles // 2)))
        warps = [block.products()] + [block.maker(w) for w in range(MAKERS)] + [block.softmax(w) for w in range(SOFTMAX)]
        pace = [rnd.choice([0.05, 1, 1, 5]) for _ in warps]
        left, steps = list(range(len(warps))), 0
        while left:
            k = rnd.choices(left, [pace[x] for x in left])[0]
            try:
                next(warps[k])
            except StopIteration:
                left.remove(k)
            steps += 1
            assert steps < 3_000_000, "warps wait for ever"


def test_the_waits_are_those_of_the_source():
    for text in ["kPages = kTile / kKv4Page", "kSoft = 8", "kProducers = 7", "soon(bar(KFULL + s), (i >> 1) & 1u)", "tc_commit(bar(KFREE + s)); tc_commit(bar(SFULL + s));",
                 "soon(bar(VFULL + s), (i >> 1) & 1u) && soon(bar(PREADY + s), (i >> 1) & 1u)", "tc_commit(bar(VFREE + s)); tc_commit(bar(ODONE + s));",
                 "if (i + 2u < n) ok = soon(bar(ODONE + s), (i >> 1) & 1u) && scores(i + 2u);", "i >= 2u && !soon_warp(bar(KFREE + s), ((i >> 1) - 1u) & 1u)",
                 "i >= 2u && !soon_warp(bar(VFREE + s), ((i >> 1) - 1u) & 1u)", "soon_warp(bar(SFULL + (i & 1u)), (i >> 1) & 1u)",
                 "soon_warp(bar(ODONE + ((i - 1u) & 1u)), ((i - 1u) >> 1) & 1u)", "mbar_arrive(bar(PREADY + (i & 1u)))", "soon_warp(bar(ODONE + (n & 1u)), ((n - 2u) >> 1) & 1u)",
                 "soon_warp(bar(ODONE + ((n - 1u) & 1u)), ((n - 1u) >> 1) & 1u)", "q += kProducers", "hide_s[i & 3u][pw] ="]:
        assert text in SOURCE, text
