"""The buffer rings of the expert mix's tensor-core kernel, as a model on the CPU: two warpgroups that take turns at filling
the operand stages, the tensor core that reads them, and waits by parity (a wait passes when the barrier's open phase has the
other parity, so also when it is two phases behind). Random schedules, with actors that are much slower than others, must never read or
overwrite the wrong tile, nor come to a stop; the rule "as many barriers as buffers" does at one buffer, and the model shows it."""
import random

import pytest

TILES = 21


class Fault(Exception):
    pass


class Barrier:
    def __init__(self):
        self.done = 0                     # completed phases

    def arrive(self):
        self.done += 1

    def passes(self, phase):              # try_wait.parity with the phase's parity
        return self.done & 1 != phase & 1


def run(stages, raw, slots, raw_slots, seed):
    """One CTA's tiles through a ring of `stages` operand buffers on `slots` barriers and (fp32 by TMA) `raw` raw buffers on
    `raw_slots` barriers; raw = 0: the warpgroups load themselves."""
    rng = random.Random(seed)
    full, empty = ([Barrier() for _ in range(slots)] for _ in range(2))
    raw_full, raw_empty = ([Barrier() for _ in range(raw_slots)] for _ in range(2))
    stage, raw_tile = [None] * stages, [None] * max(raw, 1)
    issued, in_flight, read = [], [], set()   # MMAs in order; loads in flight; tiles that the tensor core is done with

    def wait(bars, tile):
        return lambda: bars[tile % len(bars)].passes(tile // len(bars))

    def loader():
        for t in range(TILES):
            if t >= raw:
                yield wait(raw_empty, t - raw)
            raw_tile[t % raw] = None
            in_flight.append(t)
            yield None

    def landing():
        for _ in range(TILES):
            yield lambda: bool(in_flight)
            t = in_flight.pop(0)
            raw_tile[t % raw] = t
            raw_full[t % raw_slots].arrive()

    def see(t):
        if raw and raw_tile[t % raw] != t:
            raise Fault(f"tile {t} read from a raw buffer with {raw_tile[t % raw]}")

    def filler(wg):
        for t in range(wg, TILES, 2):
            if raw:
                yield wait(raw_full, t)
            see(t)                        # the pass for the largest magnitude
            yield None
            if t >= stages:
                yield wait(empty, t - stages)
            see(t)                        # the pass that writes the planes
            old = stage[t % stages]
            if old is not None and old not in read:
                raise Fault(f"tile {t} written over {old}")
            stage[t % stages] = t
            yield None
            full[t % slots].arrive()
            if raw:
                raw_empty[t % raw_slots].arrive()

    def issuer():
        for t in range(TILES):
            yield wait(full, t)
            issued.append(t)

    def tensor():
        for _ in range(TILES):
            yield lambda: bool(issued)
            t = issued[0]
            yield None
            if stage[t % stages] != t:
                raise Fault(f"products of tile {t} read {stage[t % stages]}")
            issued.pop(0)
            read.add(t)
            empty[t % slots].arrive()

    actors = [filler(0), filler(1), issuer(), tensor()] + ([loader(), landing()] if raw else [])
    weight = {a: 2.0 ** rng.uniform(-6, 0) for a in actors}
    blocked = {a: next(a) for a in actors}
    while blocked:
        ready = [a for a, c in blocked.items() if c is None or c()]
        if not ready:
            raise Fault("no actor can go on")
        a = rng.choices(ready, [weight[r] for r in ready])[0]
        try:
            blocked[a] = next(a)
        except StopIteration:
            del blocked[a]


@pytest.mark.parametrize("raw", [0, 1, 2, 4])
@pytest.mark.parametrize("stages", [1, 2, 3, 4])
def test_rings(stages, raw):
    """Four barriers for any number of stages, and four for any number of raw buffers."""
    for seed in range(300):
        run(stages, raw, 4, 4, seed)


@pytest.mark.parametrize("raw", [0, 2])
def test_the_model_finds_a_ring_of_one_stage_on_one_barrier(raw):
    with pytest.raises(Fault):
        for seed in range(300):
            run(1, raw, 1, raw or 1, seed)


@pytest.mark.parametrize("stages", [1, 2, 4])
def test_the_model_finds_one_raw_buffer_on_one_barrier(stages):
    with pytest.raises(Fault):
        for seed in range(300):
            run(stages, 1, 4, 1, seed)
