"""The bounded cache's oracle against the verify oracle and brute force."""

import math

import numpy as np
import pytest

from naivllm_amd.utils import synth
from oracle import attention as ora
from oracle import bounded as ob


def _attend(vb, **kw):
    return ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q, vb.positions,
                        1.0 / math.sqrt(vb.head_dim), vb.num_kv_heads, **kw)


def test_without_a_window_it_is_the_verify_oracle():
    vb = synth.verify_batch(3, [70, 9, 40], [4, 2, 3], num_heads=4, num_kv_heads=2, head_dim=16, block_size=8,
                            pad_rows=[1, 0, 0])
    vb.block_tables[2, 1] = -1
    want = ora.verify_attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q,
                                vb.positions, 1.0 / 4, 4, 2)
    out, _, _, sums = _attend(vb)
    np.testing.assert_allclose(out, want, atol=1e-13)
    # every row's weights sum to one
    rows = [3, 2, 3]
    for b in range(3):
        np.testing.assert_allclose(sums[b].sum(axis=1), 2 * rows[b], atol=1e-12)
    wide, *_ = _attend(vb, window=70, sinks=0)
    np.testing.assert_allclose(wide, want, atol=1e-13)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 2), (30, 0), (3, 50)])
def test_window_by_brute_force(window, sinks):
    vb = synth.verify_batch(4, [37], [3], num_heads=2, num_kv_heads=1, head_dim=8, block_size=4)
    out, _, _, sums = _attend(vb, window=window, sinks=sinks)
    total = np.zeros(37)
    for r in range(3):
        p = 34 + r
        for h in range(2):
            keys = [j for j in range(37) if j <= p and (j > p - window or j < sinks)]
            page = lambda j: (vb.block_tables[0, j // 4], j % 4, 0)  # noqa: E731
            e = [math.exp(float(vb.q[r, h] @ vb.k_cache[page(j)]) / math.sqrt(8)) for j in keys]
            o = sum(x / sum(e) * vb.v_cache[page(j)] for x, j in zip(e, keys))
            np.testing.assert_allclose(out[r, h], o, atol=1e-12)
            total[keys] += np.array(e) / sum(e)
    np.testing.assert_allclose(sums[0][0], total, atol=1e-12)


def test_added_weights_set_new_keys_and_leave_the_rest():
    tables = np.array([[2, 0, -1]])
    old = np.arange(12.0).reshape(3, 1, 4)
    new = ob.add_weights(old, {0: np.full((1, 7), 10.0)}, tables, [5])
    assert new[2, 0].tolist() == [18, 19, 20, 21]      # keys 0..3: added
    assert new[0, 0].tolist() == [10, 10, 10, 3]       # key 4 added, 5 and 6 set, 7 kept
    assert new[1, 0].tolist() == old[1, 0].tolist()    # a page of nobody


def test_eviction_keeps_first_newest_and_heaviest():
    k = np.arange(8.0).reshape(2, 4, 1, 1)
    w = np.array([[[0, 5, 1, 5]], [[5, 0, np.nan, 0]]], dtype=np.float64)
    tables = np.array([[0, 1]])
    k2, v2, w2, lens, kept = ob.evict(k, k + 100, w, tables, [8], 4, sinks=1, recent=1)
    assert lens.tolist() == [4] and kept[0, 0].tolist() == [0, 1, 3, 7]  # of three equal ones the first two
    assert k2[0, :, 0, 0].tolist() == [0, 1, 3, 7] and k2[1].tolist() == k[1].tolist()
    assert w2[0, 0].tolist() == [0, 5, 5, 0] and v2[0, :, 0, 0].tolist() == [100, 101, 103, 107]
    *_, lens, kept = ob.evict(k, k, w, tables, [3], 4, sinks=1, recent=1)
    assert lens.tolist() == [3] and kept[0, 0].tolist() == [0, 1, 2, -1]
    *_, kept = ob.evict(k, k, w, tables, [8], 7)  # NaN goes first
    assert kept[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 7]
