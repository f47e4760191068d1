"""The operand ring of the grouped maps' weight gradient, as a model on the CPU: loads, MMAs and the warp that clears the
rows behind a group's end, with waits by parity. Random schedules with actors much slower than others must not read a stage
before it is loaded and cleared, nor come to a stop. Without the clearing warp's arrival on the stages' empty barriers (the
MMAs' completion alone) a slow clearing warp falls two phases behind, and the model shows it."""
import random

import pytest

STAGES = 4


class Fault(Exception):
    pass


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.done = count, 0, 0

    def arrive(self):
        self.pending += 1
        if self.pending == self.count:
            self.pending, self.done = 0, self.done + 1

    def passes(self, phase):              # try_wait.parity with the phase's parity
        return self.done & 1 != phase & 1


def run(items, both, seed):
    """`items`: (blocks, whether the last one has a tail). `both`: the clearing warp arrives on the empty barriers too."""
    rng = random.Random(seed)
    blocks = [(i == n - 1 and tail) for n, tail in items for i in range(n)]   # per k-block: is there something to clear
    full = [Barrier(1) for _ in range(STAGES)]
    clear = [Barrier(1) for _ in range(STAGES)]
    empty = [Barrier(2 if both else 1) for _ in range(STAGES)]
    holds, cleared, issued, flying = [None] * STAGES, set(), [], []

    def producer():
        for b in range(len(blocks)):
            if b >= STAGES:
                yield lambda: empty[b % STAGES].passes(b // STAGES - 1)
            holds[b % STAGES] = None
            flying.append(b)
            yield None

    def landing():
        for _ in blocks:
            yield lambda: bool(flying)
            b = flying.pop(0)
            holds[b % STAGES] = b
            full[b % STAGES].arrive()

    def issuer():
        phase = [0] * STAGES
        for b, tail in enumerate(blocks):
            s = b % STAGES
            if tail:
                yield lambda: clear[s].passes(phase[s])
                phase[s] ^= 1
            else:
                yield lambda: full[s].passes(b // STAGES)
            issued.append(b)

    def tensor():
        for _ in blocks:
            yield lambda: bool(issued)
            b = issued[0]
            yield None
            if holds[b % STAGES] != b or (blocks[b] and b not in cleared):
                raise Fault(f"block {b} read from a stage with {holds[b % STAGES]}")
            issued.pop(0)
            empty[b % STAGES].arrive()

    def clearer():
        for b, tail in enumerate(blocks):
            s = b % STAGES
            yield lambda: full[s].passes(b // STAGES)
            if tail:
                if holds[s] != b:
                    raise Fault(f"block {b} cleared in a stage with {holds[s]}")
                cleared.add(b)
                clear[s].arrive()
            if both:
                empty[s].arrive()

    actors = [producer(), landing(), issuer(), tensor(), clearer()]
    weight = {a: 2.0 ** rng.uniform(-8, 0) for a in actors}
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


ITEMS = [[(1, True), (1, True), (3, True)], [(40, True)], [(17, False), (30, True), (2, True)], [(4, True), (8, True), (9, False)]]


@pytest.mark.parametrize("items", ITEMS, ids=str)
def test_weight_gradient_ring(items):
    for seed in range(400):
        run(items, True, seed)


def test_the_model_finds_a_clearing_warp_that_nothing_waits_for():
    with pytest.raises(Fault):
        for seed in range(400):
            run([(40, True)], False, seed)
