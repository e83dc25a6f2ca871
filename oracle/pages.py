"""CPU oracle of forked and compacted cache pages — TEST INFRASTRUCTURE ONLY.

Plain lists, from the definitions in include/naivspec.h (nsv_fork_pages,
nsv_compact_pages).  No reference counterpart.
"""

from __future__ import annotations


def fork(tables, lens, parents, num_blocks, block_size, held=()):
    """(tables, lens, lacking, moves [(src, dst, keys)])."""
    B, W = len(tables), len(tables[0]) if tables else 0
    parents = [p if 0 <= p < B else -1 for p in parents]
    old = [[e if 0 <= e < num_blocks else -1 for e in row] for row in tables]
    new = [[-1] * W for _ in range(B)]
    wants = {}
    for b, p in enumerate(parents):
        if p < 0:
            continue
        for j, e in enumerate(old[p]):
            whole = (j + 1) * block_size <= max(lens[p], 0)
            if e >= 0 and not whole and p in parents[:b]:
                wants.setdefault(b, []).append(j)
            else:
                new[b][j] = e
    kept = {e for row in new for e in row} | set(held)
    free = [i for i in range(num_blocks) if i not in kept]
    new_lens = [max(lens[p], 0) if p >= 0 else 0 for p in parents]
    asked, moves = 0, []
    for b, columns in sorted(wants.items()):
        asked += len(columns)
        if asked > len(free):
            new[b], new_lens[b] = [-1] * W, 0
            continue
        for j, f in zip(columns, free[asked - len(columns):asked]):
            new[b][j] = f
            keys = min(block_size, new_lens[b] - j * block_size)
            if keys > 0:
                moves.append((old[parents[b]][j], f, keys))
    return new, new_lens, max(0, asked - len(free)), moves


def compact(tables, num_blocks, held=()):
    """(tables, new_ids, top, moves [(src, dst)])."""
    old = [[e if 0 <= e < num_blocks else -1 for e in row] for row in tables]
    used = {e for row in old for e in row if e >= 0}
    at = {e: e for e in used | set(held)}
    moves = []
    holes = [i for i in range(num_blocks) if i not in at]
    for e, hole in zip(sorted(used - set(held), reverse=True), holes):
        if hole < e:
            at[e] = hole
            moves.append((e, hole))
    ids = [at.get(i, -1) for i in range(num_blocks)]
    return [[at[e] if e >= 0 else -1 for e in row] for row in old], ids, max(ids, default=-1) + 1, moves
