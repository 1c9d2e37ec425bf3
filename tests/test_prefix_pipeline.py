"""The barriers of the shared part of la_prefix.cu, restated on the CPU: the
loading warp, the two product warps and the softmax of both tiles, run in random
orders over random segments. Every wait is for one phase of its barrier, told by
its parity alone; it may pass only when that phase is complete, what is read then
is what was meant, and the whole always ends."""
import random

import pytest

STAGES, PARTS = 4, 2


class Bar:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def passes(self, parity):
        return self.phase & 1 != parity


class Cta:
    def __init__(self, segments, rnd):
        """segments: (two row tiles, key tiles)."""
        self.segments, self.rnd = segments, rnd
        self.kv_full = [Bar(1) for _ in range(STAGES)]
        self.kv_empty = [Bar(2) for _ in range(STAGES)]
        self.q_full, self.q_empty = Bar(1), Bar(2)
        self.s_full, self.p_full = ([[Bar(1) for _ in range(PARTS)] for _ in range(2)] for _ in range(2))
        self.pv_done, self.o_full, self.o_empty = ([Bar(1) for _ in range(2)] for _ in range(3))
        self.stage, self.q = [None] * STAGES, None
        self.s = [[None] * PARTS for _ in range(2)]      # what S / P of each part holds
        self.o = [[] for _ in range(2)]                  # the products in O
        self.queue = [[], []]                            # of each product warp, done in its order
        self.result = {}

    def load(self):
        pos = kq = 0
        for g, (two, n) in enumerate(self.segments):
            yield self.q_empty, (kq & 1) ^ 1, kq
            kq += 1
            self.q = g
            self.q_full.arrive()
            lead = 2 - two
            for i in range(n + lead):
                for kind, tile in (("v", i - lead), ("k", i)):
                    if not 0 <= tile < n:
                        continue
                    st = pos % STAGES
                    yield self.kv_empty[st], (pos // STAGES & 1) ^ 1, pos // STAGES
                    self.stage[st] = (g, kind, tile)
                    self.kv_full[st].arrive()
                    pos += 1

    def product(self, t):
        pos = segs = o_uses = 0
        tiles = 0
        do = self.queue[t].append
        for g, (two, n) in enumerate(self.segments):
            yield self.q_full, segs & 1, segs + 1
            segs += 1
            lead = 2 - two
            for i in range(-lead, n):
                pv, more = i >= 0, i + lead < n
                vs, vph = pos % STAGES, pos // STAGES
                pos += pv
                ks, kph = pos % STAGES, pos // STAGES
                pos += more
                if pv:
                    yield self.kv_full[vs], vph & 1, vph + 1
                if more:
                    yield self.kv_full[ks], kph & 1, kph + 1
                if not two and (i & 1) != t:
                    if pv:
                        self.kv_empty[vs].arrive()
                    if more:
                        self.kv_empty[ks].arrive()
                    continue
                for part in range(PARTS):
                    first, last = i < lead and part == 0, part == PARTS - 1
                    if pv:
                        if first:
                            yield self.o_empty[t], (o_uses & 1) ^ 1, o_uses
                            o_uses += 1
                        yield self.p_full[t][part], tiles & 1, tiles + 1
                        do(lambda first=first, part=part, vs=vs, i=i, g=g: self.pv(t, part, vs, first, g, i))
                        do(self.pv_done[t].arrive)
                        if last:
                            if not more:
                                do(self.o_full[t].arrive)
                            do(self.kv_empty[vs].arrive)
                    if more:
                        do(lambda part=part, ks=ks, i=i, g=g: self.qk(t, part, ks, g, i + lead))
                        do(self.s_full[t][part].arrive)
                        if last:
                            do(self.kv_empty[ks].arrive)
                            if i + 2 * lead >= n:
                                do(self.q_empty.arrive)
                tiles += pv
            if not two and t >= n:
                self.q_empty.arrive()

    def qk(self, t, part, st, g, tile):
        assert self.stage[st] == (g, "k", tile) and self.q == g
        self.s[t][part] = ("s", g, tile)

    def pv(self, t, part, st, first, g, tile):
        assert self.stage[st] == (g, "v", tile) and self.s[t][part] == ("p", g, tile)
        if first:
            assert not self.o[t], "O was not stored"
        self.o[t].append((tile, part))

    def softmax(self, t):
        seen = segs = 0
        for g, (two, n) in enumerate(self.segments):
            mine = [i for i in range(n) if two or (i & 1) == t]
            for tile in mine:
                for part in range(PARTS):
                    yield self.s_full[t][part], seen // PARTS & 1, seen // PARTS + 1
                    assert self.s[t][part] == ("s", g, tile)
                    if (tile != mine[0] or part) and self.rnd.random() < 0.5:
                        yield self.pv_done[t], (seen - 1) & 1, seen
                        assert len(self.o[t]) == PARTS * mine.index(tile) + part
                    self.s[t][part] = ("p", g, tile)
                    self.p_full[t][part].arrive()
                    seen += 1
            if not mine:
                continue
            yield self.o_full[t], segs & 1, segs + 1
            segs += 1
            self.result[g, t], self.o[t] = self.o[t], []
            self.o_empty[t].arrive()

    def run(self):
        actors = {n: [a, None] for n, a in (("load", self.load()), ("p0", self.product(0)), ("p1", self.product(1)),
                                             ("s0", self.softmax(0)), ("s1", self.softmax(1)))}
        pace = {n: self.rnd.choice((0.02, 0.3, 1.0)) for n in [*actors, "t0", "t1"]}
        while actors or any(self.queue):
            able = [n for n, (_, w) in actors.items() if w is None or w[0].passes(w[1])]
            able += ["t%d" % t for t in range(2) if self.queue[t]]
            assert able, f"all wait: {list(actors)}"
            n = self.rnd.choices(able, [pace[x] for x in able])[0]
            if n[0] == "t":
                self.queue[int(n[1])].pop(0)()
                continue
            actor, w = actors[n]
            if w is not None:
                assert w[0].phase >= w[2], f"{n} passed a barrier too early"
            actors[n][1] = next(actor, False)
            if actors[n][1] is False:
                del actors[n]


@pytest.mark.parametrize("seed", range(300))
def test_barriers(seed):
    r = random.Random(seed)
    segments = [(r.randint(0, 1), r.choice((1, 1, 2, 3, r.randint(1, 12)))) for _ in range(r.randint(1, 9))]
    cta = Cta(segments, r)
    cta.run()
    for g, (two, n) in enumerate(segments):
        for t in range(2):
            tiles = [i for i in range(n) if two or (i & 1) == t]
            assert cta.result.get((g, t), []) == [(i, part) for i in tiles for part in range(PARTS)]
