"""How a CTA pair's operand ring ends after a wait's limit: every copy has landed before the memory is given up.

The plan of ``csrc/pair_ring.cuh`` is compiled for the host and run against a model of the ring: two CTAs with one or two
producers each and the leader's MMA warp, which take their steps in any order and stop anywhere, and copies that land
whenever they like.  No GPU takes part; on one, a wait of these kernels runs out only when something else is broken.
"""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "td_benchmark_b200" / "csrc"
LEADER, PEER = 0, 1


@pytest.fixture(scope="module")
def end_of_stage(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no C++ compiler")
    tmp = tmp_path_factory.mktemp("pair_ring")
    (tmp / "shim.cpp").write_text(
        '#include "pair_ring.cuh"\n'
        'extern "C" void plan(uint32_t s, uint32_t stages, uint32_t leader, uint32_t peer, int32_t* out) {\n'
        "  const b2m::StageEnd e = b2m::end_of_stage(b2m::uses_of_stage(s, stages, leader),\n"
        "                                            b2m::uses_of_stage(s, stages, peer));\n"
        "  out[0] = e.arm, out[1] = e.take_off, out[2] = e.wait, out[3] = (int32_t)e.parity;\n}\n")
    subprocess.run([cxx, "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(tmp / "shim.cpp"), "-o",
                    str(tmp / "shim.so")], check=True)
    lib = ctypes.CDLL(str(tmp / "shim.so"))

    def plan(s, stages, leader, peer):
        out = (ctypes.c_int32 * 4)()
        lib.plan(*(ctypes.c_uint32(v) for v in (s, stages, leader, peer)), out)
        return bool(out[0]), bool(out[1]), bool(out[2]), out[3]

    return plan


class Barrier:
    """One arrival and a byte count complete a phase."""

    def __init__(self):
        self.phase, self.pending, self.tx = 0, 1, 0

    def change(self, arrivals=0, tx=0):
        self.pending, self.tx = self.pending - arrivals, self.tx + tx
        assert self.pending >= 0
        if self.pending == 0 and self.tx == 0:
            self.phase, self.pending = self.phase + 1, 1

    def done(self, parity):
        return self.phase % 2 != parity


class Pair:
    def __init__(self, rng, stages, producers=2):
        self.rng, self.stages, self.producers = rng, stages, producers
        self.full = [Barrier() for _ in range(stages)]
        self.empty = [[0] * stages for _ in range(2)]      # stages released, as each CTA knows
        self.released = []                                 # (CTA, stage) on their way
        self.flight = []                                   # (CTA, stage, bytes on the leader's barrier, index)
        self.landed = [set(), set()]
        self.issued = {(c, w): 0 for c in range(2) for w in range(2)}
        self.next = {(c, w): w for c in range(2) for w in range(2)}
        self.bytes = [[0] * stages for _ in range(2)]
        self.mma = 0
        total = rng.randrange(1, 5 * stages)
        self.tail = [rng.random() < 0.25 for _ in range(total)]
        self.size = [rng.randrange(1, 9) * 16 for _ in range(total)]

    def produce(self, c, w):
        i = self.next[c, w]
        s = i % self.stages
        if i >= len(self.size) or self.empty[c][s] < i // self.stages:
            return False
        if c == LEADER:
            self.full[s].change(1, 0 if self.tail[i] else 2 * self.size[i])
        self.bytes[c][s] = 0 if self.tail[i] else self.size[i]
        self.flight.append((c, s, self.bytes[c][s], i))
        self.next[c, w] = i + self.producers
        for of in (w, 1) if self.producers == 1 else (w,):      # one producer: its count stands for both kinds of stage
            self.issued[c, of] = i + 1
        return True

    def multiply(self):
        i = self.mma
        s = i % self.stages
        if i >= len(self.size) or self.full[s].phase <= i // self.stages:
            return False
        if self.tail[i] and not all(i in got for got in self.landed):
            return False
        self.mma += 1
        self.released += [(c, s) for c in range(2)]        # reaches the CTAs one after the other
        return True

    def land(self, at):
        c, s, counted, i = self.flight.pop(at)
        if counted:
            self.full[s].change(0, -counted)
        self.landed[c].add(i)

    def run_until_all_stopped(self):
        actors = [("p", c, w) for c in range(2) for w in range(self.producers)] + [("m",)]
        stop = self.rng.choice([0.01, 0.05, 0.2])
        while actors:
            if self.released and self.rng.random() < 0.5:
                c, s = self.released.pop(self.rng.randrange(len(self.released)))
                self.empty[c][s] += 1
            if self.flight and self.rng.random() < self.rng.choice([0.1, 0.6]):
                self.land(self.rng.randrange(len(self.flight)))
            a = self.rng.choice(actors)
            moved = self.multiply() if a[0] == "m" else self.produce(a[1], a[2])
            if self.rng.random() < stop or (not moved and self.rng.random() < 0.1):
                actors.remove(a)

    def counted_in_flight(self, s):
        return [f for f in self.flight if f[1] == s and f[2]]


def _settle(ring, plan):
    """What the leader does; False when it goes on while a copy that it counts is in flight."""
    for s in range(ring.stages):
        arm, take_off, wait, parity = plan(s, ring.stages, ring.issued[LEADER, s & 1], ring.issued[PEER, s & 1])
        bar = ring.full[s]
        if arm:
            bar.change(1, ring.bytes[PEER][s])
        if take_off:
            bar.change(0, -ring.bytes[LEADER][s])
        while wait and not bar.done(parity):
            left = ring.counted_in_flight(s)
            assert left, "the wait can never end"
            ring.land(ring.flight.index(ring.rng.choice(left)))
        if ring.counted_in_flight(s):
            return False
    return True


@pytest.mark.parametrize("producers", [1, 2])
@pytest.mark.parametrize("stages", [2, 4, 6])
def test_every_copy_lands_wherever_the_ctas_stop(end_of_stage, stages, producers):
    ahead = {"leader": 0, "peer": 0, "even": 0}
    for seed in range(4000):
        ring = Pair(random.Random(seed), stages, producers)
        ring.run_until_all_stopped()
        for w in range(2):
            lead, peer = ring.issued[LEADER, w], ring.issued[PEER, w]
            ahead["leader" if lead > peer else "peer" if peer > lead else "even"] += 1
        assert _settle(ring, end_of_stage), seed
    assert min(ahead.values()) > 100                      # every kind of end was met


def test_the_model_shows_a_leader_that_waits_for_its_own_stages_only():
    """The plan that knows the leader's count alone: it waits for ever, or leaves the peer's copies in flight."""
    def own_stages(s, stages, leader, peer):
        uses = (leader - 1 - s) // stages + 1 if leader > s else 0
        return False, False, uses > 0, (uses - 1) & 1

    left = stuck = 0
    for seed in range(500):
        ring = Pair(random.Random(seed), 6)
        ring.run_until_all_stopped()
        try:
            left += not _settle(ring, own_stages)
        except AssertionError:
            stuck += 1
    assert left and stuck
