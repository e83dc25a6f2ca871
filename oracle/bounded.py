"""CPU oracle for the operators of a bounded paged cache.

TEST INFRASTRUCTURE ONLY, as the rest of this package.

float64 numpy, from the definitions:
  * window attention: the row at position p sees the keys j <= p, j < context,
    on a mapped page, with j > p - window or j < sinks;
  * key weights: for each (key, kv head) the softmax weights of the rows and
    of the kv head's query heads, summed; set for the keys at or behind the
    position of the sequence's first row, added for older ones;
  * eviction: min(length, budget) keys of each (sequence, kv head) stay: the
    first ``sinks``, the last ``recent`` and of the rest those with the most
    weight (ties: the lowest position; NaN is less than every number), moved
    to the front in the order of their positions.

The reference has none of them; the attention without a window is pinned
against oracle.attention (tests/test_oracle_bounded.py).
"""

from __future__ import annotations

import numpy as np


def visible(positions, keys, window=None, sinks: int = 0) -> np.ndarray:
    """[rows, keys]: whether the row at a position sees the key at an index."""
    p, j = np.asarray(positions)[:, None], np.asarray(keys)[None, :]
    seen = j <= p
    if window is not None:
        seen &= (j > p - window) | (j < sinks)
    return seen


def attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, positions, scale, num_kv_heads: int,
              window=None, sinks: int = 0):
    """Returns (out [T, H, D], the same over |V| [T, H, D], the largest
    scale * sum |q| |k| of a row [T, H], weights {b: [Hkv, n]}): the second and third bound what
    roundings of the weights and of the scores do to the first."""
    q = np.asarray(q, dtype=np.float64)
    T, H, D = q.shape
    bs, G = k_cache.shape[1], H // num_kv_heads
    out, out_abs, mag, weights = np.zeros_like(q), np.zeros_like(q), np.zeros((T, H)), {}
    for b in range(block_tables.shape[0]):
        n = max(0, min(int(context_lens[b]), block_tables.shape[1] * bs))
        rows = [r for r in range(int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1])) if positions[r] >= 0]
        weights[b] = np.zeros((num_kv_heads, n))
        j = np.arange(n)
        page = np.asarray(block_tables)[b, j // bs].astype(np.int64)
        j = j[page >= 0]
        page = page[page >= 0]
        seen = visible([positions[r] for r in rows], j, window, sinks)
        used = seen.any(0)
        j, page, seen = j[used], page[used], seen[:, used]
        if not rows or not j.size:
            continue
        for h in range(H):
            hk = h // G
            K, V = (np.asarray(c[page, j % bs, hk], dtype=np.float64) for c in (k_cache, v_cache))
            s = np.where(seen, (q[rows, h] @ K.T) * scale, -np.inf)
            top = s.max(axis=1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
            p = p / np.maximum(p.sum(axis=1, keepdims=True), 1e-300)
            out[rows, h], out_abs[rows, h] = p @ V, p @ np.abs(V)
            mag[rows, h] = (np.abs(q[rows, h]) @ np.abs(K).T * seen).max(axis=1) * scale
            weights[b][hk, j] += p.sum(axis=0)
    return out, out_abs, mag, weights


def add_weights(key_weights, sums, block_tables, first) -> np.ndarray:
    """key_weights [num_blocks, Hkv, bs] after a call whose sequences'
    sums[b] [Hkv, n] cover the keys 0 .. n - 1 up to the last row, and whose
    first rows lie at first[b]."""
    new = np.array(key_weights, dtype=np.float64)
    bs = new.shape[2]
    for b, w in sums.items():
        for j in range(w.shape[1]):
            page = int(block_tables[b, j // bs])
            if page >= 0:
                old = new[page, :, j % bs] if j < first[b] else 0.0
                new[page, :, j % bs] = old + w[:, j]
    return new


def evict(k_cache, v_cache, key_weights, block_tables, context_lens, budget: int, sinks: int = 0, recent: int = 0,
          out_block_tables=None):
    """Returns (k_cache, v_cache, key_weights, lens, kept [B, Hkv, budget])."""
    old = [np.array(x) for x in (k_cache, v_cache, key_weights)]
    new = [x.copy() for x in old]
    bs, hkv = k_cache.shape[1:3]
    out = block_tables if out_block_tables is None else out_block_tables
    B = block_tables.shape[0]
    lens, all_kept = np.zeros(B, dtype=np.int64), np.full((B, hkv, budget), -1, dtype=np.int32)
    for b in range(B):
        n = max(0, min(int(context_lens[b]), block_tables.shape[1] * bs))
        lens[b] = min(n, budget)
        for h in range(hkv):
            j = np.arange(n)
            w = old[2][block_tables[b, j // bs], h, j % bs].astype(np.float64)
            w = np.where(np.isnan(w), -np.inf, w)
            if n <= budget:
                kept = j
            else:
                middle = j[sinks:n - recent]
                best = sorted(middle, key=lambda i: (-w[i], i))[:budget - sinks - recent]
                kept = np.concatenate([j[:sinks], np.sort(np.array(best, dtype=np.int64)), j[n - recent:]])
            all_kept[b, h, :len(kept)] = kept
            if n <= budget and out_block_tables is None:
                continue
            i = np.arange(len(kept))
            src, to = block_tables[b, kept // bs], out[b, i // bs]
            for x, y in zip(old[:2], new[:2]):
                y[to, i % bs, h] = x[src, kept % bs, h]
            new[2][to, h, i % bs] = old[2][src, h, kept % bs]
    return (*new, lens, all_kept)
