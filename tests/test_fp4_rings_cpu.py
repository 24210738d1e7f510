"""The rings of fp4_grad_kernel (bsq_fp4_grad.cu) as a model: decoding warps that wait by the parity of barriers, copies that land in any order, one issuer of MMAs.
No run can be relied on to show a wait that takes one round for another; random schedules of the model do.  The lengths are read from the source."""
import bisect
import itertools
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitsqueeze-llm_b200", "csrc", "bsq_fp4_grad.cu")


def lengths(mt):
    with open(SOURCE) as f:
        text = f.read()
    found = []
    for name in ("ring_of", "groups_of", "raw_ring_of"):
        two, one = re.search(r"constexpr int %s\(int mt\) \{ return mt == 2 \? (\d+) : (\d+); \}" % name, text).groups()
        found.append(int(two if mt == 2 else one))
    return tuple(found)


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.done = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.done, self.pending = self.done + 1, self.count

    def passes(self, parity):
        """mbarrier.try_wait.parity: whether the round of that parity is not the one under way."""
        return (self.done & 1) != parity


def schedule(ring, groups, raw_ring, stages, seed, warps=4):
    """One random schedule; None, or what went wrong.  Every schedule has its own speeds, a hundredfold apart: with equal ones nobody falls far enough behind
    for a round to be taken for another, and the hazards hardly show."""
    rnd = random.Random(seed)
    full, empty = [Barrier(warps + 2) for _ in range(ring)], [Barrier(1) for _ in range(ring)]      # full: expectation, bytes of dY, warps
    raw_full, raw_empty = [Barrier(1) for _ in range(raw_ring)], [Barrier(warps) for _ in range(raw_ring)]
    raw_next = a_next = mma = 0
    decoders = [[g, False] for g in range(groups) for _ in range(warps)]
    actors = list(itertools.accumulate([10 ** rnd.uniform(-1, 1) for _ in range(4)] + [10 ** rnd.uniform(0, 1)]))
    speeds = list(itertools.accumulate(10 ** rnd.uniform(-1, 1) for _ in decoders))
    decoded, raw_moving, a_moving, raw_here, a_here, late = {}, [], [], set(), set(), rnd.random()
    for _ in range(stages * 40000):
        if mma >= stages:
            return None
        who = bisect.bisect(actors, rnd.random() * actors[-1])
        if who == 0 and raw_next < stages:                            # copies of B
            place, use = raw_next % raw_ring, raw_next // raw_ring
            if use == 0 or raw_empty[place].passes((use & 1) ^ 1):
                if raw_empty[place].done < use:
                    return "a place is filled that has not been read"
                raw_moving.append(raw_next)
                raw_next += 1
        elif who == 1:                                                # copies land, often not in order
            for moving, here, bars, n in ((raw_moving, raw_here, raw_full, raw_ring), (a_moving, a_here, full, ring)):
                if moving and rnd.random() < 0.5:
                    stage = moving.pop(rnd.randrange(len(moving)) if rnd.random() < late else 0)
                    here.add(stage)
                    bars[stage % n].arrive()
        elif who == 2 and a_next < stages:                            # copies of dY
            place, use = a_next % ring, a_next // ring
            if use == 0 or empty[place].passes((use & 1) ^ 1):
                if empty[place].done < use:
                    return "dY overwrites a stage that is being read"
                full[place].arrive()
                a_moving.append(a_next)
                a_next += 1
        elif who == 3:                                                # the issuer of MMAs
            place, use = mma % ring, mma // ring
            if full[place].passes(use & 1):
                if decoded.get(mma, 0) != warps or mma not in a_here:
                    return "MMAs of a stage that is not there"
                empty[place].arrive()
                mma += 1
        elif who == 4:
            warp = decoders[bisect.bisect(speeds, rnd.random() * speeds[-1])]
            stage, has = warp
            if stage >= stages:
                continue
            if not has:
                if raw_full[stage % raw_ring].passes((stage // raw_ring) & 1):
                    if stage not in raw_here:
                        return "decoded before the copy has landed"
                    warp[1] = True
            else:
                place, use = stage % ring, stage // ring
                if use == 0 or empty[place].passes((use & 1) ^ 1):
                    if empty[place].done < use:
                        return "decoded into a stage that is being read"
                    decoded[stage] = decoded.get(stage, 0) + 1
                    full[place].arrive()
                    raw_empty[stage % raw_ring].arrive()
                    warp[0], warp[1] = stage + groups, False
    return "stuck"


@pytest.mark.parametrize("mt", [1, 2])
def test_no_wait_takes_one_round_for_another(mt):
    ring, groups, raw_ring = lengths(mt)
    assert groups <= ring and raw_ring % groups == 0
    wrong = {schedule(ring, groups, raw_ring, 60, seed) for seed in range(60)} - {None}
    assert not wrong


@pytest.mark.parametrize("ring,groups,raw_ring,stages", [(3, 4, 6, 60), (5, 4, 6, 400)])
def test_the_model_finds_the_lengths_that_failed(ring, groups, raw_ring, stages):
    assert {schedule(ring, groups, raw_ring, stages, seed) for seed in range(40)} - {None, "stuck"}
