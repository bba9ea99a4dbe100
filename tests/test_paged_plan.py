"""The partition of the paged attention on the CPU: every stage of every tile is taken once, nothing is written behind the workspace, and the
grid has a workgroup for every piece."""
import random

import pytest

from oracle.paged_plan import STAGE, Plan


def check(p: Plan, lengths):
    # workgroups and pieces are one to one
    items = [p.item_of(w) for w in range(p.grid)]
    taken = sorted(i for i in items if i is not None)
    assert taken == list(range(p.pieces)), "workgroups do not cover the pieces"
    assert p.pieces <= p.grid
    # the stages of a tile, in order and without a gap; slots are distinct, and where the join looks
    seen, slots = {}, set()
    for i in range(p.pieces):
        b, head, tile, x, s0, s1, slot = p.piece(i)
        assert s0 < s1 and x < p.n[b] and tile < p.tiles[b] <= p.rt
        seen.setdefault((b, head, tile), []).append((x, s0, s1))
        if slot is not None:
            assert slot == p.join_slot(b, head, tile, x) and slot not in slots
            slots.add(slot)
    assert len(seen) == p.Hkv * sum(p.tiles)
    for (b, _, _), runs in seen.items():
        runs.sort()
        assert [r[0] for r in runs] == list(range(p.n[b])) and runs[0][1] == 0 and runs[-1][2] == p.stages[b]
        assert all(a[2] == c[1] for a, c in zip(runs, runs[1:]))
    assert len(slots) == p.used_slots
    if p.used_slots:
        assert p.ws_bytes and max(slots) < p.slots, "a slot behind the workspace"


def lengths_of(rng, B, most):
    kind = rng.random()
    if kind < 0.25:
        return [most] * B
    if kind < 0.5:
        return [max(1, int(most * (1 - (b * 0.618034) % 1))) for b in range(B)]
    if kind < 0.75:
        return [rng.choice((0, 1, rng.randint(0, most), most)) for _ in range(B)]
    return [rng.randint(0, 300) if rng.random() < 0.9 else most for _ in range(B)]


@pytest.mark.parametrize("seed", range(8))
def test_random_calls(seed):
    rng = random.Random(seed)
    ways = set()
    for _ in range(60):
        cus = rng.choice((8, 32, 64, 256))          # (few compute units reach every branch with little work)
        B = rng.choice((1, 2, 3, 8, 33, 64, 65, 130))
        Hkv = rng.choice((1, 2, 5, 8))
        G = rng.choice((1, 2, 4, 7))
        Lq = rng.choice((1, 1, 2, 9, 33, 61, 200))
        d = rng.choice((64, 128, 256))
        most = rng.choice((100, 513, 1400, 5000, 20000, 60000)) // (4 if B > 60 else 1)
        lengths = lengths_of(rng, B, most)
        counts = None if rng.random() < 0.5 else [rng.randint(-1, Lq + 1) for _ in range(B)]
        max_len = rng.choice((most, most, most // 2, 2 * most))
        p = Plan(lengths, counts, Hkv * G, Hkv, Lq, d, rng.random() < 0.5, max_len, cus, rng.random() < 0.9)
        if p.pieces > 30000:
            continue
        check(p, lengths)
        ways.add(p.way)
    assert {"uncut", "one round"} <= ways and len(ways) >= 4, ways


def test_slots_at_their_bound():
    """Lengths made to be cut worst: every tile one stage over a multiple of the share."""
    for staged in (False, True):
        for cus in (8, 64, 256):
            for share in (2, 3, 5, 9):
                for B in (64, 200, 900):
                    lengths = [STAGE * share + 1] * B + [STAGE * 4000]
                    check(Plan(lengths, None, 4 if not staged else 40, 1, 1 if not staged else 3, 128, False, STAGE * 4000, cus), lengths)


def test_known_plans():
    """One long sequence: as many pieces as the rounds hold.  Short ones: not cut.  A sequence that is cut cuts all."""
    p = Plan([131071], None, 32, 8, 1, 128, True, 131071, 256)
    assert p.cut and p.way == "one round" and p.pieces <= p.target and p.n == [64]
    p = Plan([500, 3, 0], None, 8, 2, 1, 128, False, 512, 256)
    assert not p.cut and p.n == [1, 1, 1] and p.ws_bytes == 0
    p = Plan([300, 5000], None, 8, 2, 1, 128, False, 5000, 256)
    assert p.cut and p.n[0] == 3 and p.first_slot == [0, 6]
