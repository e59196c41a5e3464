"""The stages of the 4-bit layer's tcgen05 kernel (csrc/int4tc.cuh) as a model on the CPU: its roles, barriers and waits by
parity, run in orders that no GPU promises to avoid: a role may be held back for as long as any other can go on. What is
checked: nobody reads a stage of x, or the sums taken of it, that holds another stage's, and every wait ends. The model's
earlier form (a refill that waits for the products alone, warps that wait for phases which nothing holds for them) has to
fail, or the model would see nothing."""
import random

import pytest

STAGES, BUFS, AHEAD = 4, 4, 3
SUMS = 2 * STAGES


class Bar:
    """An mbarrier: a phase completes with its count of arrivals; a wait by parity sees only the current phase's parity."""

    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left = self.count
            self.phase += 1

    def passed(self, parity):
        return (self.phase & 1) != parity


class Wrong(Exception):
    pass


def simulate(seed, units, zero, copies, n_it, gated=True, idle_leave=True):
    """units: of a stage (4, 2 or 1). Raises Wrong at a stale read, returns False where the waits never end."""
    rng = random.Random(seed)
    a_full, b_full, empty = [[Bar(n) for _ in range(STAGES)] for n in (2, 1 if copies else 3, 1)]
    sx_full = [Bar(3) for _ in range(SUMS)]
    d_full, d_empty = [[Bar(n) for _ in range(BUFS)] for n in (1, 2)]
    if units == 1:
        empty = d_full
    x = [[None] * 3 for _ in range(STAGES)]        # which stage's rows a slot holds, by the warp that sums them
    sums = [[None] * 3 for _ in range(SUMS)]
    queue = []                                     # copies and products under way: (steps that follow in any order, or in turn)
    products = []

    def unpack():                                  # two of the eight warps stand for all
        for it in range(n_it):
            if it >= STAGES:
                yield lambda: empty[it % STAGES].passed(((it // STAGES) & 1) ^ 1)
            a_full[it % STAGES].arrive()
            yield None

    def issue():
        unit = 0
        for it in range(n_it):
            st, ph = it % STAGES, (it // STAGES) & 1
            yield lambda: a_full[st].passed(ph)
            yield lambda: b_full[st].passed(ph)
            for _ in range(units):
                buf = unit % BUFS
                if unit >= BUFS:
                    yield lambda: d_empty[buf].passed(((unit // BUFS) & 1) ^ 1)
                products.append(("product", it, [d_full[buf]]))
                unit += 1
            if units > 1:
                products.append(("commit", it, [empty[st]]))
            yield None

    def tensor_core():
        done = 0
        total = n_it * (units + (units > 1))
        while done < total:
            yield lambda: len(products) > done
            kind, it, bars = products[done]
            if kind == "product" and x[it % STAGES] != [it] * 3:
                raise Wrong(f"products of stage {it} read {x[it % STAGES]}")
            for b in bars:
                b.arrive()
            done += 1
            yield None

    def copier():
        done = 0
        while done < n_it:
            yield lambda: len(queue) > done
            it = queue[done]
            for w in range(3):
                x[it % STAGES][w] = it
                yield None
            b_full[it % STAGES].arrive()
            done += 1

    def rows(w):                                   # warps 9, 10, 11
        if copies and not zero and w and idle_leave:
            return
        for nx in range(n_it + (AHEAD if zero else 0)):
            if nx < n_it:
                if nx >= STAGES and not (gated and zero and copies and w):
                    yield lambda: empty[nx % STAGES].passed(((nx // STAGES) & 1) ^ 1)
                    if gated and zero and copies:
                        old = nx - STAGES
                        yield lambda: sx_full[old % SUMS].passed((old // SUMS) & 1)
                if not copies:
                    x[nx % STAGES][w] = nx
                    b_full[nx % STAGES].arrive()
                elif w == 0:
                    queue.append(nx)
                yield None
            if not zero or nx < AHEAD:
                continue
            it = nx - AHEAD
            yield lambda: b_full[it % STAGES].passed((it // STAGES) & 1)
            if x[it % STAGES][w] != it:
                raise Wrong(f"warp {9 + w} sums stage {x[it % STAGES][w]} for {it}")
            sums[it % SUMS][w] = it
            sx_full[it % SUMS].arrive()
            yield None

    def add():                                     # two of the warps 12-15
        for unit in range(n_it * units):
            buf, it = unit % BUFS, unit // units
            yield lambda: d_full[buf].passed((unit // BUFS) & 1)
            if zero:
                yield lambda: sx_full[it % SUMS].passed((it // SUMS) & 1)
                if sums[it % SUMS] != [it] * 3:
                    raise Wrong(f"the sums of stage {it} are {sums[it % SUMS]}")
            d_empty[buf].arrive()
            yield None

    roles = [unpack(), unpack(), issue(), tensor_core(), rows(0), rows(1), rows(2), add(), add()]
    if copies:
        roles.append(copier())
    waits = [None] * len(roles)
    left = set(range(len(roles)))
    held, until = None, 0                          # a role that is held back while others can go on
    step = 0
    while left:
        ready = [i for i in left if waits[i] is None or waits[i]()]
        if not ready:
            return False
        if step >= until:
            held, until = rng.randrange(len(roles)), step + rng.choice((5, 40, 400))
        pick = [i for i in ready if i != held] or ready
        i = rng.choice(pick)
        try:
            waits[i] = next(roles[i])
        except StopIteration:
            left.discard(i)
        step += 1
    return True


FORMS = [(units, zero, copies) for units in (1, 2, 4) for zero in (False, True) for copies in (False, True)]


@pytest.mark.parametrize("units,zero,copies", FORMS)
def test_no_stale_stage_and_no_endless_wait(units, zero, copies):
    for seed in range(150):
        assert simulate(seed, units, zero, copies, 1 + seed % 27), f"a wait never ends (seed {seed})"


@pytest.mark.parametrize("units", [1, 2, 4])
def test_the_model_sees_a_refill_that_does_not_wait_for_the_sums(units):
    stale = 0
    for seed in range(150):
        try:
            simulate(seed, units, True, True, 24, gated=False)
        except Wrong:
            stale += 1
    assert stale > 0


@pytest.mark.parametrize("units", [1, 2, 4])
def test_the_model_sees_waits_for_phases_that_nothing_holds(units):
    assert not all(simulate(seed, units, False, True, 24, idle_leave=False) for seed in range(150))
