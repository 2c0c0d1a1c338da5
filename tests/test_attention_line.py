"""CPU replay of how the attention kernels cut their line of tiles, and of where the merge looks for the parts."""
import random

import pytest

from _line import Line

SHAPES = [(8, 16, 8, 444, 4), (32, 16, 8, 296, 4), (128, 128, 4, 148, 1)]  # rows, positions, unit cost, CTAs, least


def owner(q_start, n_seqs, token):
    """The merge's sequence of a token: the last that starts at or before it and has it, or -1."""
    b = max((i for i in range(n_seqs) if q_start[i] <= token), default=0)
    return b if q_start[b] <= token < q_start[b + 1] else -1


@pytest.mark.parametrize("rows,tt,cost,ctas,least", SHAPES)
def test_the_merge_reads_what_the_tiles_left(rows, tt, cost, ctas, least):
    """Every tile of every unit is in one run; the parts that the merge reads are those that the runs wrote."""
    rng = random.Random(rows)
    for _ in range(40):
        n = rng.randint(1, 12)
        fresh = [rng.choice([0, 1, 1, rng.randint(1, 90)]) for _ in range(n)]
        lens = [rng.choice([0, rng.randint(0, 50), rng.randint(0, 3000)]) for _ in range(n)]
        start = [rng.randint(0, 3)]
        for f in fresh:
            start.append(start[-1] + f)
        tokens, group, kv = start[-1] + rng.randint(0, 2), rng.choice([1, 3, 8]), rng.choice([1, 2])
        for prefix in (0, rng.randint(1, 2000)):
            line = Line(start, lens, tokens, group, kv, rows, tt, cost, ctas, least, prefix)
            wrote, tiles = {}, {}
            for cta in range(ctas):
                for b, h, row0, tile0, count, _ in line.units(cta):
                    tiles.setdefault((b, h, row0), []).extend(range(tile0, tile0 + count))
                    if count < line.spans[b][1]:
                        slot = (cta, 0 if tile0 > 0 else 1)
                        assert slot not in wrote
                        wrote[slot] = (b, h, row0)
            for (b, h, row0), got in tiles.items():
                assert got == list(range(line.spans[b][1]))
            assert len(tiles) == sum(rt * kv for rt, _, _ in line.spans)
            for token in range(tokens):
                b = owner(start, n, token)
                if b < 0:
                    continue
                b = 0 if prefix else b
                for h in range(kv):
                    r, where = line.parts(token, h, group - 1, b)
                    row0 = (token - line.seqs[b][0]) * group + group - 1 - r
                    if len(where) > 1:
                        assert all(wrote[x] == (b, h, row0) for x in where)


def test_a_q_start_that_does_not_ascend_stays_inside():
    """The prefix pass covers rows q_start[0] .. q_start[n] only; a token of a sequence that lies outside has no
    place on its line.  With the merge's check every part lies in the workspace; without it some do not."""
    rng = random.Random(1)
    outside = 0
    for _ in range(300):
        n, tokens = rng.randint(1, 6), 600
        start = [rng.randint(-5, tokens + 5) for _ in range(n + 1)]
        line = Line(start, [9] * n, tokens, 4, 2, 8, 16, 8, 444, 4, prefix=700)
        own = Line(start, [9] * n, tokens, 4, 2, 8, 16, 8, 444, 4)
        for token in range(0, tokens, 7):
            b = owner(start, n, token)
            if b < 0:
                continue
            s, fresh, _ = own.seqs[b]
            assert s <= token < s + fresh
            s, fresh, _ = line.seqs[0]
            for h in range(2):
                good = all(0 <= i < 444 for i, _ in line.parts(token, h, 0)[1]) and token >= s
                assert good or not s <= token < s + fresh
                outside += not good
    assert outside > 50
