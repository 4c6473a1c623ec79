"""The work split of the 8-bit cache's attention kernel, restated in Python: for
random batches every step of every unit is taken exactly once, a CTA's parts of
a cut unit lie in consecutive workers, and the CTAs that share a unit are the
ones its ticket counts on."""
import random

import pytest

MERGE = 16  # steps that take a CTA as long as a merge across CTAs


class Split:
    def __init__(self, total, most):
        self.total, self.n = total, min(most, total)
        self.each = total // self.n
        self.rem = total - self.each * self.n

    def begin(self, g):
        return g * self.each + min(g, self.rem) if g < self.n else self.total

    def owner(self, x):
        wide = self.rem * (self.each + 1)
        return x // (self.each + 1) if x < wide else self.rem + (x - wide) // self.each


def _unit_at(steps, units, x):
    """(sequence, unit of it, step of that, first step of the unit)."""
    at = 0
    for b, s in enumerate(steps):
        if x < at + s * units:
            sub = (x - at) // s
            return b, sub, (x - at) % s, at + sub * s
        at += s * units
    raise AssertionError(x)


def _whole(split, steps, units):
    """Units of at most this many steps are not cut between CTAs."""
    most = (split.each + MERGE) // max(steps)  # units of the longest kind a CTA may have
    return max(steps) if len(steps) * units <= split.n * most else 2 * MERGE


def _border(split, steps, units, c):
    x = split.begin(c)
    if 0 < x and c < split.n:
        b, _, inside, _ = _unit_at(steps, units, x)
        if steps[b] <= _whole(split, steps, units):
            x += -inside if 2 * inside < steps[b] else steps[b] - inside
    return x


@pytest.mark.parametrize("warps", [8, 12])
@pytest.mark.parametrize("seed", range(18))
def test_every_step_is_taken_once_and_parts_join(seed, warps):
    rng = random.Random(seed)
    ctas = rng.choice([1, 3, 16, 37])
    units = rng.choice([1, 2, 8])
    longest = rng.choice([1, 6, 33, 90, 400])
    even = seed % 3 == 0
    steps = [longest if even else rng.randint(1, longest) for _ in range(rng.choice([1, 2, 9, 40]))]
    total = sum(steps) * units
    split = Split(total, ctas)
    taken = []
    parts_of = {}  # unit's first step -> [(cta, how many parts of it there)]
    borders = [_border(split, steps, units, c) for c in range(split.n + 1)]
    assert borders[0] == 0 and borders[-1] == total and borders == sorted(borders)
    for cta in range(split.n):
        lo, hi = borders[cta], borders[cta + 1]
        if lo == hi:
            continue
        share = Split(hi - lo, warps)
        entries = []  # (2 * worker + slot, unit, begins, ends)
        for w in range(warps):
            x, end = lo + share.begin(w), lo + share.begin(w + 1)
            while x < end:
                b, sub, inside, first = _unit_at(steps, units, x)
                stop = min(end, first + steps[b])
                taken.extend(range(x, stop))
                begins, ends = inside == 0, stop == first + steps[b]
                if not (begins and ends):
                    assert all(e[0] != 2 * w + begins for e in entries)
                    entries.append((2 * w + begins, first, begins, ends))
                x = stop
        entries.sort()
        runs = []
        for i, e in enumerate(entries):
            if e[2] or i == 0:
                runs.append([e])
            else:
                assert runs[-1][-1][1] == e[1]
                runs[-1].append(e)
        cut = {}
        for r in runs:
            assert len({e[1] for e in r}) == 1
            # entry i of a run behind its first is slot 0 of the i-th worker behind
            assert all(e[0] == 2 * (r[0][0] // 2 + i) for i, e in enumerate(r) if i)
            if not (r[0][2] and r[-1][3]):
                side = int(r[0][2])
                assert side not in cut
                cut[side] = r[0][1]
                parts_of.setdefault(r[0][1], []).append((cta, side))
    assert taken == list(range(total))
    for first, where in parts_of.items():
        b = _unit_at(steps, units, first)[0]
        assert steps[b] > _whole(split, steps, units)
        c0, c1 = split.owner(first), split.owner(first + steps[b] - 1)
        assert where == [(c, int(c == c0)) for c in range(c0, c1 + 1)]  # what the last of them merges
