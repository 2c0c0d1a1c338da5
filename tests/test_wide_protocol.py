"""Model check (CPU) of how the softmax warps of the wide attention kernel leave (go-infer_b200/csrc/wide_attn.cu).

Eight warps walk a CTA's units and tiles.  They wait for barriers in memory, each wait with a time limit of its
own, and meet at one named barrier, which has none.  A wait may expire for one warp in the moment in which it is
over for another, or because another role gave up, so its outcomes differ from warp to warp.  Claim: whatever the
outcomes, no warp waits at the named barrier for one that is gone: a warp whose wait expired stays until the next
vote there, and the vote sends all away.  The model replays the warps' steps over random outcomes; the same steps
with a warp that leaves by itself must get stuck, which shows that the check has teeth.
"""
import random

import pytest

WARPS = 8


def warp(units, wait, votes):
    """One softmax warp: yields its `ok` at each meeting and is sent the vote; returns when it leaves."""
    ok = True
    for tiles in units:
        yield True  # the unit is shown
        if tiles:
            yield True  # the queries' maxima
            yield True  # they are read
        for i in range(tiles + 1 if tiles else 0):
            if i < tiles:
                ok = ok and wait()  # s_full
                if votes:
                    ok = yield ok
                    if not ok:
                        break
                else:
                    if not ok:
                        break
                    yield True
            if i > 0:
                ok = ok and wait()  # o_full
                if not ok:
                    if votes:
                        continue
                    break
        if votes:
            ok = yield ok
            if not ok:
                return False
        else:
            if not ok:
                return False
            yield True
        yield True  # everything shown is read
    return ok


def play(seed, votes, fail=0.1):
    """Whether the warps end together; False when one waits for a warp that is gone."""
    rng = random.Random(seed)
    units = [rng.choice([0, 1, 2, 5]) for _ in range(rng.randint(1, 6))]
    stop = [False]

    def wait():
        if rng.random() < (0.5 if stop[0] else fail):  # after the first expiry the others' are over, or see the stop
            stop[0] = True
            return False
        return True

    warps = [warp(units, wait, votes) for _ in range(WARPS)]
    send = [None] * WARPS
    while True:
        met, left = [], []
        for w, x in zip(warps, send):
            try:
                met.append(w.send(x))
            except StopIteration as e:
                left.append(e.value)
        if not met:
            return len(set(left)) == 1 and left[0] == (not stop[0])
        if left:
            return False
        send = [all(met)] * WARPS


@pytest.mark.parametrize("fail", [0.0, 0.001, 0.02, 0.3])
def test_warps_leave_together(fail):
    assert all(play(seed, True, fail) for seed in range(3000))


def test_a_warp_that_leaves_by_itself_leaves_others_waiting():
    stuck = sum(not play(seed, False, 0.01) for seed in range(3000))
    assert stuck > 100 and all(play(seed, False, 0.0) for seed in range(200))
