"""A model of the ring protocol of the row kernel of attention over the 4-bit cache (csrc/oxq_kv4_attn.cu), run on random schedules: parity barriers,
two groups of four warps on alternate tiles, copies that land in any order.  It holds that no tile is overwritten before its four warps have left it
and that a warp that passes a wait finds its own tile there; a parity wait cannot tell a phase from the one two before, so the order of the steps matters."""
import random

import pytest

STAGES, LEAD = 5, 3


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.phase = 0

    def _check(self):
        if self.pending == 0 and self.tx == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def arrive(self, tx=0):
        assert self.pending > 0, "too many arrivals"
        self.tx += tx
        self.pending -= 1
        self._check()

    def land(self):
        self.tx -= 1
        self._check()

    def passed(self, parity):
        return (self.phase & 1) != parity


def run(seed, pieces, see_first=True, prime_after_all=True):
    rng = random.Random(seed)
    full, empty = [Barrier(1) for _ in range(STAGES)], [Barrier(4) for _ in range(STAGES)]
    holds, left, flying, meeting = [None] * STAGES, [4] * STAGES, [], {}
    pace = [rng.random() ** 3 + 0.01 for _ in range(8)]

    def sync(key, w):
        meeting.setdefault(key, set()).add(w)
        while len(meeting[key]) < 8:
            yield

    def bring(n):
        s = n % STAGES
        while not empty[s].passed(((n // STAGES) & 1) ^ 1):
            yield
        assert holds[s] is None or left[s] == 0, f"{n} overwrites {holds[s]}"
        holds[s], left[s] = n, 4
        full[s].arrive(1)
        flying.append(s)
        yield

    def warp(w):
        group, count = w >> 2, 0

        def prime(tiles):
            i = (2 * (w & 3) + 1 - group - count) & 7
            if i < tiles and i < LEAD:
                yield from bring(count + i)

        yield from sync("start", w)
        yield from prime(pieces[0])
        for k, tiles in enumerate(pieces):
            yield from sync(("rows", k), w)
            for i in range((group - count) & 1, tiles, 2):
                t = count + i
                mine = i + LEAD < tiles and ((t + LEAD) >> 1 & 3) == (w & 3)
                if mine and not see_first:
                    yield from bring(t + LEAD)
                while not full[t % STAGES].passed((t // STAGES) & 1):
                    yield
                assert holds[t % STAGES] == t and t % STAGES not in flying, f"{holds[t % STAGES]} in the place of {t}"
                if mine and see_first:
                    yield from bring(t + LEAD)
                yield
                left[t % STAGES] -= 1
                empty[t % STAGES].arrive()
            count += tiles
            more = k + 1 < len(pieces)
            if more and not prime_after_all:
                yield from prime(pieces[k + 1])
            yield from sync(("join", k), w)
            if more and prime_after_all:
                yield from prime(pieces[k + 1])

    warps, idle = {w: warp(w) for w in range(8)}, 0
    while warps:
        idle += 1
        assert idle < 100000, "stuck"
        if flying and rng.random() < 0.15:
            full[flying.pop(rng.randrange(len(flying)))].land()
            idle = 0
            continue
        w = rng.choices(list(warps), [pace[x] for x in warps])[0]
        try:
            next(warps[w])
        except StopIteration:
            del warps[w]


def _pieces(seed):
    rng = random.Random(seed + 9999)
    return [rng.choice([1, 1, 2, 3, 4, 5, 7, 9, 14, 30]) for _ in range(rng.randrange(1, 6))]


def test_the_ring_holds():
    for seed in range(150):
        run(seed, _pieces(seed))


def test_the_order_matters():
    """The model finds the fault of bringing a tile before the own one is seen and of priming a piece before all warps have left the last one."""
    with pytest.raises(AssertionError):
        for seed in range(400):
            run(seed, _pieces(seed), see_first=False, prime_after_all=False)
