"""The sharing out of attention_tree's work over its blocks (csrc/attention_tree.cuh), restated: every tile of every unit is taken once, the
pieces of a cut unit follow one another from the block that begins it to the one that its note names, and a block has at most one piece that it does
not begin and one that it does not end."""
import random

import pytest


def blocks_for(grid, work, extra):
    return min(grid, max(work // (extra + 2), 1))


def share(grid, work, b, extra):
    n = blocks_for(grid, work, extra)
    if b >= n or work == 0:
        return 0, 0
    each, more = divmod(work, n)
    begin = b * each + min(b, more)
    return begin, begin + each + (1 if b < more else 0)


def block_of(grid, work, p, extra):
    n = blocks_for(grid, work, extra)
    each, more = divmod(work, n)
    edge = more * (each + 1)
    return p // (each + 1) if p < edge else more + (p - edge) // each


def work_of(tiles, items, kvh, items_per_unit, extra):
    return kvh * (tiles * items + extra * -(-items // items_per_unit))


def piece(requests, kvh, items_per_unit, p, end, extra):
    """requests: (tiles, items) each.  -> (request, kv head, item, t0, t1, tiles, next, last)."""
    at = 0
    for s, (tiles, items) in enumerate(requests):
        mine = work_of(tiles, items, kvh, items_per_unit, extra)
        if p < at + mine:
            break
        at += mine
    whole = items_per_unit * tiles + extra
    head, in_head = divmod(p - at, mine // kvh)
    unit = in_head // whole
    item = unit * items_per_unit
    two = items_per_unit == 2 and item + 1 < items
    off, size = in_head - unit * whole, (2 if two else 1) * tiles + extra
    off_end = min(size, off + end - p)
    t0, t1 = max(off - extra, 0), max(off_end - extra, 0)
    if two:
        t0, t1 = (t0 + 1) // 2, (t1 + 1) // 2
    nxt = p + off_end - off
    return s, head, item, t0, t1, tiles, end if end - nxt <= extra else nxt, p - off + size - (2 if two else 1)


@pytest.mark.parametrize("extra", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("items_per_unit", [1, 2])
@pytest.mark.parametrize("seed", range(60))
def test_every_tile_once(items_per_unit, seed, extra):
    rng = random.Random(seed)
    grid, kvh = rng.choice([1, 2, 3, 7, 148, 296]), rng.choice([1, 2, 8])
    requests = [(rng.choice([1, 1, 2, 3, rng.randrange(1, 60)]), rng.choice([0, 1, 1, 2, 3, 5])) for _ in range(rng.randrange(1, 12))]
    work = sum(work_of(t, i, kvh, items_per_unit, extra) for t, i in requests)
    taken = {}
    for b in range(grid):
        begin, end = share(grid, work, b, extra)
        p, mine = begin, []
        while p < end:
            x = piece(requests, kvh, items_per_unit, p, end, extra)
            if x[3] == x[4]:
                assert not mine, "an empty piece behind the first"
            else:
                mine.append(x)
            p = x[6]
        assert bool(mine) == (begin < end)
        assert sum(x[3] > 0 for x in mine) <= 1 and sum(x[4] < x[5] for x in mine) <= 1
        assert all(x[3] == 0 for x in mine[1:]) and all(x[4] == x[5] for x in mine[:-1])
        for s, head, item, t0, t1, tiles, _, last in mine:
            taken.setdefault((s, head, item), []).append((b, t0, t1, tiles, last))
    want = {(s, h, i) for s, (_, items) in enumerate(requests) for h in range(kvh) for i in range(0, items, items_per_unit)}
    assert set(taken) == want
    for parts in taken.values():
        assert parts[0][1] == 0 and parts[-1][2] == parts[0][3]
        assert [p[0] for p in parts] == list(range(parts[0][0], parts[-1][0] + 1))
        assert all(a[2] == b[1] for a, b in zip(parts, parts[1:]))
        assert block_of(grid, work, parts[0][4], extra) == parts[-1][0]
