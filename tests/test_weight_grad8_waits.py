"""How the warps of a team meet at a range's last rows in the weight gradient from 8 bits (csrc/weight_grad8.cu): the team's waits replayed
on the CPU under random interleavings, with a wait that runs out somewhere.  A warp whose wait has run out leaves, so that the others must
not wait for it without a limit."""
import os
import random
import re

import pytest

from tests.test_warp_waits import WAIT, _offences

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tile_fusion_b200", "csrc")
WARPS = 4


class _Barrier:
    """An mbarrier of `count` arrivals; a wait of parity p passes while the phase under way has the other parity."""

    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def _replay(turns, bounded, seed, run_out):
    """A team of four warps with `turns` slices, the last of them without all its rows, and the warp that issues products.  True where all
    come to their end.  `bounded`: how the team meets; else in a barrier without a limit."""
    full, empty, tail = _Barrier(WARPS), _Barrier(1), _Barrier(WARPS)
    met = [0]  # arrivals at the barrier without a limit

    def warp():
        for turn in range(turns):
            if turn and not (yield empty, (turn - 1) & 1):
                return
            if turn == turns - 1:
                for k in range(2):
                    if bounded:
                        tail.arrive()
                        if not (yield tail, k):
                            return
                    else:
                        met[0] += 1
                        yield None, WARPS * (k + 1)
            full.arrive()

    def products():
        for turn in range(turns):
            if not (yield full, turn & 1):
                return
            empty.arrive()

    rng = random.Random(seed)
    roles = [warp() for _ in range(WARPS)] + [products()]
    waits = [next(r, None) for r in roles]
    dead, step = False, 0
    while any(w is not None for w in waits):
        step += 1
        able = []
        for i, w in enumerate(waits):
            if w is None:
                continue
            if w[0] is None:
                if met[0] >= w[1]:
                    able.append((i, True))
            elif w[0].passes(w[1]):
                able.append((i, True))
            elif dead or step >= run_out:
                able.append((i, False))
        if not able:
            if any(w is not None and w[0] is not None for w in waits):  # bounded waits are left: one of them runs out
                run_out = step
                continue
            return False
        i, ok = rng.choice(able)
        dead = dead or not ok
        try:
            waits[i] = roles[i].send(ok)
        except StopIteration:
            waits[i] = None
    return True


@pytest.mark.parametrize("turns", [1, 2, 3, 6])
def test_a_team_never_waits_for_a_warp_that_left(turns):
    runs = [(seed, run_out) for seed in range(400) for run_out in (1, 3, 5, 8, 13, 10 ** 9)]
    assert all(_replay(turns, True, seed, run_out) for seed, run_out in runs)
    if turns > 1:
        assert not all(_replay(turns, False, seed, run_out) for seed, run_out in runs)  # what a barrier without a limit comes to


def test_no_barrier_without_a_limit_among_warps_that_may_leave():
    """Named barriers have no limit: the one there is (few classes: the warps that bring tiles) is passed by all of its warps, since none leaves."""
    found = {}
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            n = len(re.findall(r"\"bar\.(?:sync|red|arrive)", f.read()))
        if n:
            found[name] = n
    assert found == {"ce_few.cu": 1}


@pytest.mark.parametrize("source", ["plane_gemm.cu", "ce_few.cu", "weight_grad8.cu"])
def test_a_warp_leaves_as_one(source):
    """As for the other kernels (test_warp_waits.py): nothing is decided by a wait's result before the warp has voted on it."""
    with open(os.path.join(CSRC, source)) as f:
        text = f.read()
    assert WAIT.search(text) and _offences(text) == []
