"""The oracle of forked and compacted pages, by hand and by what must hold (CPU)."""

import random

from oracle.pages import compact, fork


def test_one_prompt_goes_on_as_three():
    tables = [[5, 2, 7, 1, -1], [-1] * 5, [-1] * 5]
    new, lens, lacking, moves = fork(tables, [9, 0, 0], [0, 0, 0], 10, 4, held=[0])
    assert new == [[5, 2, 7, 1, -1], [5, 2, 3, 4, -1], [5, 2, 6, 8, -1]]
    assert lens == [9, 9, 9] and lacking == 0 and moves == [(7, 3, 1), (7, 6, 1)]


def test_rows_end_and_pages_run_out():
    tables = [[0, 1], [2, 3]]
    assert fork(tables, [4, 4], [1, 1], 4, 4) == ([[2, 3], [2, 0]], [4, 4], 0, [])
    new, lens, lacking, _ = fork([[0, 1, 2], [3, 4, 5], [-1] * 3], [2, 2, 0], [0, 0, 1], 6, 4)
    assert new == [[0, 1, 2], [-1] * 3, [3, 4, 5]] and lens == [2, 0, 2] and lacking == 3
    assert fork(tables, [4, 4], [-1, 9], 4, 4)[:3] == ([[-1, -1], [-1, -1]], [0, 0], 0)


def test_forked_rows_own_what_they_write():
    rng = random.Random(4)
    for _ in range(200):
        B, W, bs, nb = rng.randint(1, 6), rng.randint(1, 6), rng.choice([1, 2, 4]), 60
        ids = rng.sample(range(nb), B * W)
        tables = [ids[b * W:(b + 1) * W] for b in range(B)]
        lens, parents = [rng.randint(0, W * bs) for _ in range(B)], [rng.randint(-1, B - 1) for _ in range(B)]
        new, new_lens, lacking, moves = fork(tables, lens, parents, nb, bs)
        assert lacking == 0
        writable = [e for row, n in zip(new, new_lens) for j, e in enumerate(row) if e >= 0 and (j + 1) * bs > n]
        assert len(set(writable)) == len(writable)
        assert not {d for _, d, _ in moves} & {s for s, _, _ in moves}
        content = {d: (s, k) for s, d, k in moves}
        for b, p in enumerate(parents):
            for j in range(-(-new_lens[b] // bs)):
                e = new[b][j]
                assert e == tables[p][j] or content[e] == (tables[p][j], min(bs, new_lens[b] - j * bs))


def test_compact():
    assert compact([[9, 4, -1], [4, 7, 2]], 10, held=[0, 8]) == (
        [[1, 4, -1], [4, 3, 2]], [0, -1, 2, -1, 4, -1, -1, 3, 8, 1], 9, [(9, 1), (7, 3)])
    assert compact([[-1]], 3) == ([[-1]], [-1] * 3, 0, [])
    rng = random.Random(5)
    for _ in range(200):
        nb = rng.randint(1, 40)
        used, held = rng.sample(range(nb), rng.randint(0, nb)), rng.sample(range(nb), rng.randint(0, nb // 3))
        tables, ids, top, moves = compact([used + [-1]], nb, held)
        assert len({e for e in tables[0] if e >= 0}) == len(used)
        assert all(ids[h] == h for h in held)
        count = len(set(used) | set(held))
        assert top == count or max(held, default=-1) == top - 1 >= count
        assert all(d < s for s, d in moves)
