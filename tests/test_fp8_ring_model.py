"""Model of the rings of the kernels over an 8-bit cache (csrc/attn/decode_fp8.cu: F8Ring; csrc/attn/fp8_cache.cu: the store's) when waits run out.

A loading warp and its consumers, mbarriers with arrivals, bytes and phase, and copies that take their time, some of them longer than a consumer waits.
Whatever order they run in, no barrier gets more arrivals than its phase takes, and no copy is on its way when the last warp has left.
"""
import random

import pytest

PATIENCE = 40                                            # turns until a wait runs out
LATEST = 60                                              # turns that a copy takes at most: it is late, not lost


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.phase = 0

    def _flip(self):
        if self.pending == 0 and self.tx == 0:
            self.phase ^= 1
            self.pending = self.count

    def arrive(self, tx=0):
        assert self.pending > 0, "more arrivals than the phase takes"
        self.pending -= 1
        self.tx += tx
        self._flip()

    def complete(self):
        self.tx -= 1
        self._flip()

    def done(self, parity):
        return self.phase != parity


def wait(barrier, parity, patience=PATIENCE):
    for _ in range(patience):
        if barrier.done(parity):
            return True
        yield
    return False


def run(seed, stages, consumers, tiles, leave, give_back, settle):
    """leave: consumers return when a wait has run out (the store's), or go on without waits.  give_back: they still free their stages."""
    rng = random.Random(seed)
    full, empty = [Barrier(1) for _ in range(stages)], [Barrier(consumers) for _ in range(stages)]
    copies = []                                          # [turns left, stage]

    def loader():
        s = phase = issued = 0
        for _ in range(tiles):
            if not (yield from wait(empty[s], phase ^ 1)):
                break
            full[s].arrive(tx=1)
            copies.append([rng.choice((1, 5, 20, LATEST)), s])
            issued = min(issued + 1, stages)
            s, phase = (0, phase ^ 1) if s + 1 == stages else (s + 1, phase)
            yield
        if settle:
            for i in range(1, issued + 1):
                at = s - i
                assert (yield from wait(full[at + stages if at < 0 else at], phase ^ 1 if at < 0 else phase, 4 * LATEST))

    def consumer():
        s, phase, ok = 0, 0, True
        for _ in range(tiles):
            ok = ok and (yield from wait(full[s], phase))
            if not ok and leave:
                return
            yield
            if ok or give_back:
                empty[s].arrive()
            s, phase = (0, phase ^ 1) if s + 1 == stages else (s + 1, phase)

    warps = [loader()] + [consumer() for _ in range(consumers)]
    while warps:
        w = rng.choice(warps)
        for c in copies[:]:
            c[0] -= 1 / len(warps)                       # on average a turn of every warp
            if c[0] <= 0:
                copies.remove(c)
                full[c[1]].complete()
        try:
            next(w)
        except StopIteration:
            warps.remove(w)
    assert not copies, "a copy is on its way to shared memory that is gone"


SHAPES = [(3, 2, 9), (2, 4, 1), (2, 4, 2), (2, 4, 7), (1, 4, 1), (8, 12, 14), (3, 12, 20)]


@pytest.mark.parametrize("stages,consumers,tiles", SHAPES)
@pytest.mark.parametrize("leave", [False, True])
def test_no_copy_outlives_its_warps(stages, consumers, tiles, leave):
    for seed in range(60):
        run(seed, stages, consumers, tiles, leave, give_back=False, settle=True)


@pytest.mark.parametrize("give_back,settle", [(True, True), (False, False)])
def test_the_model_finds_rings_that_do_not_settle_or_free_a_stage_under_a_copy(give_back, settle):
    broken = 0
    for seed in range(60):
        try:
            run(seed, 2, 4, 7, leave=False, give_back=give_back, settle=settle)
        except AssertionError:
            broken += 1
    assert broken
