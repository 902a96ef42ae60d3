"""The hand-overs of the tensor-core kernels for 4-bit matrices (csrc/mxfp4_tc.cu, csrc/mxfp4_pair.cuh), as a model on the host: agents that
take their steps in random order and at different speeds, copies that land in any order, matrix instructions that are done in order.
A barrier is waited for by the parity of its phase, so a wait may pass on a phase two before the one it means: the model finds an agent
that reads what has not landed, an arrival at the wrong phase, and agents that wait for one another."""
import random
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "fastllm-py_b200" / "csrc"


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.pending, self.phase = count, count, 0, 0

    def _complete(self):
        if self.left == 0 and self.pending == 0:
            self.phase += 1
            self.left = self.count

    def arrive(self, copies=0):
        assert self.left > 0, "an arrival too many"
        self.left -= 1
        self.pending += copies
        self._complete()

    def land(self):
        self.pending -= 1
        self._complete()

    def over(self, parity):
        return (self.phase & 1) != parity


class Machine:
    """Runs generators (a yield is a step) until all are done; `flight`: copies, landed in any order; `issued`: in order."""

    def __init__(self, seed):
        self.random, self.flight, self.issued = random.Random(seed), [], []

    def run(self, agents):
        r = self.random
        weights = [r.choice((1, 1, 5, 20)) for _ in agents]
        slow, idle = r.choice((0.003, 0.03, 0.2)), 0
        live = list(zip(agents, weights))
        while live:
            assert idle < 6000, "agents wait for one another"
            idle += 1
            if self.flight and r.random() < slow:
                self.flight.pop(r.randrange(len(self.flight)))()
                idle = 0
            elif self.issued and r.random() < 0.3:
                self.issued.pop(0)()
                idle = 0
            else:
                i = r.choices(range(len(live)), [w for _, w in live])[0]
                try:
                    if next(live[i][0]):
                        idle = 0
                except StopIteration:
                    live.pop(i)
                    idle = 0


class Ring:
    def __init__(self, machine, stages, full, empty):
        self.machine, self.stages = machine, stages
        self.full, self.empty = [Barrier(full) for _ in range(stages)], [Barrier(empty) for _ in range(stages)]
        self.holds = [-1] * stages

    def fill(self, it):
        s = it % self.stages

        def land():
            self.holds[s] = it
            self.full[s].land()
        self.machine.flight.append(land)
        self.full[s].arrive(1)

    def producer(self, total):
        for it in range(total):
            while not self.empty[it % self.stages].over((it // self.stages & 1) ^ 1):
                yield False
            self.fill(it)
            yield True

    def read(self, it):
        assert self.holds[it % self.stages] == it, f"chunk {it} read, {self.holds[it % self.stages]} there"


def scales_of_pairs(seed, stages, groups, total, before):
    """The pair kernel of two 4-bit operands: `groups` of warps take the stages' scales in turn, one issues the matrix instructions.
    `before`: what a group waits for besides its own phase."""
    m = Machine(seed)
    ring, scales = Ring(m, stages, 1, 1), [Barrier(1) for _ in range(stages)]

    def group(g):
        for it in range(g, total, groups):
            s, ph = it % stages, it // stages & 1
            while before == "empty" and not ring.empty[s].over(ph ^ 1) or before == "full" and not ring.full[s].over(ph ^ 1):
                yield False
            while not ring.full[s].over(ph):
                yield False
            ring.read(it)
            scales[s].arrive()
            yield True

    def issuer():
        for it in range(total):
            s = it % stages
            while not scales[s].over(it // stages & 1):
                yield False
            ring.read(it)
            m.issued.append(ring.empty[s].arrive)
            yield True
    m.run([ring.producer(total), issuer()] + [group(g) for g in range(groups)])


def converted(seed, stages, places, total, token_stages=0):
    """The kernels that convert: two groups of warps take every other chunk from the ring to a place, one issues.  With a ring of their
    own for the tokens (pairs) the groups look for those too, and only they empty the codes' ring."""
    m = Machine(seed)
    ring = Ring(m, stages, 1, 1 if token_stages else 2)
    tokens = Ring(m, token_stages, 1, 1) if token_stages else None
    a_full, a_empty, place_holds = [Barrier(1) for _ in range(places)], [Barrier(1) for _ in range(places)], [-1] * places

    def group(g):
        for it in range(g, total, 2):
            s, p = it % stages, it % places
            while not ring.full[s].over(it // stages & 1):
                yield False
            ring.read(it)
            ring.empty[s].arrive()
            yield True
            while tokens and not tokens.full[it % token_stages].over(it // token_stages & 1):
                yield False
            if tokens:
                tokens.read(it)
            while not a_empty[p].over((it // places & 1) ^ 1):
                yield False
            place_holds[p] = it
            a_full[p].arrive()
            yield True

    def issuer():
        for it in range(total):
            p = it % places
            while not a_full[p].over(it // places & 1):
                yield False
            assert place_holds[p] == it
            (tokens or ring).read(it)

            def done(it=it, p=p):
                assert place_holds[p] == it, "a place was written while it was read"
                a_empty[p].arrive()
                (tokens or ring).empty[it % (token_stages or stages)].arrive()
            m.issued.append(done)
            yield True
    m.run([ring.producer(total), issuer(), group(0), group(1)] + ([tokens.producer(total)] if tokens else []))


def constant(file, name):
    return eval(re.search(rf"#define {name} (\([^\n/]*\)|\d+)", (CSRC / file).read_text()).group(1))


def test_the_model_finds_phases_taken_for_one_another():
    """What the kernel would do without the wait for the stage's use before, and with one for a phase that may be passed twice."""
    for before in (None, "full"):
        with pytest.raises(AssertionError):
            for seed in range(300):
                scales_of_pairs(seed, 5, 4, 40, before)


def test_scales_of_pairs():
    stages = constant("mxfp4_pair.cuh", "MXQP_STAGES")
    source = (CSRC / "mxfp4_pair.cuh").read_text()
    assert "!mxt_wait(&empty_bar[s], ph ^ 1u, abort_flag) || !mxt_wait(&full_bar[s], ph, abort_flag)" in source
    for seed in range(200):
        scales_of_pairs(seed, stages, 4, 40, "empty")


@pytest.mark.parametrize("tokens", range(16, 129, 16))
def test_conversion_on_tiles(tokens):
    ring, most = constant("mxfp4_tc.cu", "MXT_RING"), constant("mxfp4_tc.cu", "MXT_MAX_STAGES")
    stages = min(most, ring // (tokens * 256 + 2 * (8192 + 1024)))
    for seed in range(50):
        converted(seed, stages, 3 if tokens <= 64 else 2, 40)


@pytest.mark.parametrize("tokens", range(32, 193, 32))
def test_conversion_on_pairs(tokens):
    ring, most = constant("mxfp4_pair.cuh", "MXP_X_RING"), constant("mxfp4_pair.cuh", "MXP_X_STAGES")
    for seed in range(50):
        converted(seed, constant("mxfp4_pair.cuh", "MXP_W_STAGES"), 2, 40, min(most, ring // (tokens * 128)))
