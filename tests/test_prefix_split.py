"""The division of shared prefixes among CTAs, restated on the CPU: the
segments of la_prefix.cu cover every key tile of every item once, their partial
rows never meet and stay inside the workspace, and the rows that the combine
pass reads for a (batch row, query head) are those that were written for it."""
import random

import pytest

ROWS, KEYS = 128, 128


def shape(rows, keys, per_tile):
    row_tiles = -(-rows // per_tile)
    tiles = -(-keys // KEYS)
    pairs, single = (row_tiles + 1) >> 1, row_tiles & 1
    return tiles, pairs, single, (pairs - single) * tiles + ((tiles + 1) >> 1 if single else 0)


def part_of(x, T, G):
    return ((x + 1) * G - 1) // T


class Split:
    def __init__(self, groups, hkv, grp, grid, batch):
        """groups: (first, rows, keys)."""
        self.groups, self.hkv, self.grp, self.grid, self.batch = groups, hkv, grp, grid, batch
        self.per = ROWS // grp
        self.steps = [hkv * shape(n, k, self.per)[3] if k and n >= 2 else 0 for _, n, k in groups]
        self.T = sum(self.steps)
        self.G = max(1, min(self.T, grid))

    def part_row(self, g, h, r, c):
        first, rows, _ = self.groups[g]
        return 2 * self.grp * (self.hkv * first + h * rows + r * 2 * self.per) + 2 * ROWS * c

    def segments(self, c):
        """As walk_start and walk_next."""
        if c >= self.G or self.T == 0:
            return
        u0, u1 = c * self.T // self.G, (c + 1) * self.T // self.G
        left, before, g = u1 - u0, 0, 0
        while before + self.steps[g] <= u0:
            before += self.steps[g]
            g += 1
        tiles, pairs, single, per_head = shape(*self.groups[g][1:], self.per)
        h, y = divmod(u0 - before, per_head)
        r = min(y // tiles, pairs - 1)
        s = y - r * tiles
        while left > 0:
            first, rows, keys = self.groups[g]
            one = bool(single) and r == pairs - 1
            steps = (tiles + 1) >> 1 if one else tiles
            n = min(steps - s, left)
            t0 = 2 * s if one else s
            nt = min(2 * n, tiles - t0) if one else n
            seqs = min(rows - r * 2 * self.per, 2 * self.per)
            yield g, h, r, one, t0, nt, seqs, self.part_row(g, h, r, c)
            left -= n
            s += n
            if s == steps and left > 0:
                s, r = 0, r + 1
                if r == pairs:
                    r, h = 0, h + 1
                    if h == self.hkv:
                        h, g = 0, g + 1
                        while not self.steps[g]:
                            g += 1
                        tiles, pairs, single, per_head = shape(*self.groups[g][1:], self.per)

    def reads(self, b, hh):
        """Partial rows that the combine pass takes for row b, query head hh."""
        g = max(i for i, (f, _, _) in enumerate(self.groups) if f <= b)
        first, rows, keys = self.groups[g]
        tiles, pairs, single, per_head = shape(rows, keys, self.per)
        h, seq = hh // self.grp, b - first
        r = seq // (2 * self.per)
        inside = seq - r * 2 * self.per
        one = bool(single) and r == pairs - 1
        u0 = sum(self.steps[:g]) + h * per_head + r * tiles
        n = (tiles + 1) >> 1 if one else tiles
        pf, pl = part_of(u0, self.T, self.G), part_of(u0 + n - 1, self.T, self.G)
        tile = 0 if one else inside // self.per
        stride = (rows - r * 2 * self.per) * self.grp
        row0 = (self.part_row(g, h, r, pf) + tile * self.per * self.grp + (inside - tile * self.per) * self.grp
                + hh % self.grp)
        out = []
        for c in range(pl - pf + 1):
            out += [row0 + 2 * ROWS * c + x * stride for x in range(2 if one else 1)]
        return out


@pytest.mark.parametrize("seed", range(40))
def test_segments_and_partial_rows(seed):
    r = random.Random(seed)
    hkv, grp, grid = r.choice((1, 2, 4, 8)), r.randint(1, 8), r.choice((1, 7, 148))
    groups, first = [], 0
    for _ in range(r.choice((1, 1, 2, 5, 40))):
        rows = r.choice((0, 1, 2, 3, r.randint(1, 300)))
        groups.append((first, rows, r.choice((0, 16, 128, 129, r.randint(1, 40) * 48, r.randint(1, 9000)))))
        first += rows
    batch = first + r.choice((0, 3))
    s = Split(groups, hkv, grp, grid, batch)
    written, seen = {}, {}
    for c in range(grid):
        for g, h, rr, one, t0, nt, seqs, row0 in s.segments(c):
            assert nt > 0 and t0 + nt <= -(-groups[g][2] // KEYS)
            for i in range(t0, t0 + nt):
                assert seen.setdefault((g, h, rr, i), c) == c
                seen[g, h, rr, i] = c
            rows0 = min(seqs, s.per) * grp
            for t in range(2):
                n = (seqs - s.per if not one and t else min(seqs, s.per)) * grp
                assert 0 < n <= ROWS
                for i in range(n):
                    row = row0 + t * rows0 + i
                    assert row not in written and 0 <= row < 2 * batch * hkv * grp + 2 * ROWS * grid
                    seq, q = divmod(i, grp)
                    b = groups[g][0] + rr * 2 * s.per + (0 if one else t * s.per) + seq
                    written[row] = (b, h * grp + q)
    tiles = sum(hkv * -(-k // KEYS) * ((-(-n // s.per) + 1) >> 1) for _, n, k in groups if n >= 2 and k)
    assert len(seen) == tiles
    want = {}
    for row, at in written.items():
        want.setdefault(at, set()).add(row)
    for (b, hh), rows in want.items():
        got = s.reads(b, hh)
        assert len(got) == len(set(got)) and set(got) == rows
    assert {b for b, _ in want} == {b for f, n, k in groups if n >= 2 and k for b in range(f, f + n)}


@pytest.mark.parametrize("grid", [2, 3, 7, 8, 64, 131, 132, 147, 148])
def test_every_part_of_the_division_is_taken_once(grid):
    """take_part: with Q CTAs (an even number) that stream, the others' numbers
    are 0..grid-Q-1, theirs 0..Q-1, and neighbours 2i, 2i+1 have the same part."""
    pairs = grid // 2
    for Q in range(0, grid + 1 - (grid & 1) if grid > 2 else 2, 2):
        half, got = Q // 2, {True: [], False: []}
        for block in range(grid):
            pair = block // 2
            before = pair * half // pairs
            shared = pair >= pairs or (pair + 1) * half // pairs == before
            got[shared].append(block - 2 * min(before, half) if shared else 2 * before + (block & 1))
        assert sorted(got[False]) == list(range(Q)) and sorted(got[True]) == list(range(grid - Q)), (grid, Q)
