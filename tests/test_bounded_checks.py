"""What the bounded cache's operators refuse, and the host's work lists:
nothing here launches a kernel."""

import ctypes

import numpy as np
import pytest
import torch

from naivllm_amd import _lib
from naivllm_amd.layers.attention import (evict_kvcache, few_rows_serve_prefill, paged_attention_weights,
                                          paged_attention_window, prefill_key_weights)


def test_row_attention_codes():
    h = _lib.lib()

    def window(B=2, T=2, H=16, Hkv=8, D=128, bs=16, mb=4, mq=1, dt=1, window=8, sinks=0, ws=None, size=0, ptr=16):
        return h.nsv_window_attention(ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, 0.1, B, T, H, Hkv, D, bs, mb, mq, dt, window,
                                      sinks, None, ws, size, None)

    def weights(B=2, T=2, H=16, Hkv=8, D=128, bs=16, mb=4, mq=1, dt=1, w=16, ws=None, size=0):
        return h.nsv_weights_attention(16, 16, 16, 16, w, 16, 16, 16, 16, 0.1, B, T, H, Hkv, D, bs, mb, mq, dt, ws, size,
                                       None)

    for call in (window, weights):
        assert call(B=0) == 0 and call(T=0) == 0         # nothing to do
        assert call(B=-1) == call(T=-1) == call(H=0) == call(mb=0) == call(mq=0) == call(dt=2) == -1
        assert call(H=12) == call(D=96) == call(bs=24) == call(mq=65) == call(mb=1 << 27) == -2
        assert call() == -3 and call(ws=16, size=64) == -3  # no workspace, a small one
    assert window(window=0) == window(window=-3) == window(sinks=-1) == -1
    assert window(ptr=8) == window(ptr=None) == -1          # not on 16 bytes; null
    assert weights(w=None) == -1
    assert h.nsv_window_attention_workspace_size(2, 16, 8, 96, 16, 4, 1, 1, 8, 0) == 0
    assert h.nsv_window_attention_workspace_size(2, 16, 8, 128, 16, 4, 1, 1, 8, 0) > 0


def test_evict_codes():
    h = _lib.lib()

    def evict(B=1, Hkv=2, D=64, bs=16, mb=4, ob=0, dt=1, budget=8, sinks=0, recent=0, out=None, k=16, ws=None):
        return h.nsv_evict_kv(k, 16, 16, 16, 16, out, 16, 16, B, Hkv, D, bs, mb, ob, dt, budget, sinks, recent, ws, 64,
                              None)

    assert evict(B=0) == 0
    assert evict(B=-1) == evict(budget=0) == evict(sinks=-1) == evict(recent=-1) == evict(dt=3) == evict(k=None) == -1
    assert evict(sinks=5, recent=4) == evict(k=24) == -1
    assert evict(out=16, ob=0) == evict(out=16, ob=1, budget=40) == -1  # no room for what stays
    assert evict(D=40) == evict(bs=24) == evict(mb=1 << 27) == -2
    assert evict(mb=600, budget=8192) == evict(mb=600, budget=8192, ws=16) == -3  # rows by way of a workspace
    assert h.nsv_evict_workspace_size(1, 2, 64, 16, 600, 0, 1, 8192) == 2 * 2 * 8192 * 128
    assert h.nsv_evict_workspace_size(1, 2, 64, 16, 600, 1, 1, 8192) == 0
    assert h.nsv_evict_workspace_size(16, 8, 128, 256, 128, 0, 1, 2048) == 0


def test_prefill_key_weights_codes():
    h = _lib.lib()

    def call(n=1, m=1, H=4, Hkv=2, D=128, bs=16, mb=4, part=16, q=16):
        return h.nsv_prefill_key_weights(q, 16, 16, 16, 16, 16, n, 16, m, 0.1, H, Hkv, D, bs, mb, part, None)

    assert call(n=0) == call(m=0) == 0
    assert call(n=-1) == call(H=0) == call(mb=0) == call(q=None) == call(q=8) == -1
    assert call(H=3) == call(D=96) == call(bs=10) == -2
    assert call(part=None) == -3


def _cpu_case():
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    return dict(query=torch.zeros((2, 4, 64), dtype=torch.bfloat16), k_cache=cache, v_cache=cache,
                tables=torch.zeros((2, 2), dtype=torch.int32), lens=torch.tensor([3, 4]),
                cu=torch.tensor([0, 1, 2], dtype=torch.int32), positions=torch.tensor([2, 3]),
                weights=torch.zeros((4, 2, 16)))


def test_operators_refuse_the_cpu():
    c = _cpu_case()
    meta = (c["tables"], c["lens"], c["cu"], c["positions"], 0.1, 4, 2, 64, 16, 16)
    with pytest.raises(ValueError, match="GPU"):
        paged_attention_window(c["query"], c["k_cache"], c["v_cache"], *meta, window=4)
    with pytest.raises(ValueError, match="GPU"):
        paged_attention_weights(c["query"], c["k_cache"], c["v_cache"], c["weights"], *meta)
    with pytest.raises(ValueError, match="GPU"):
        evict_kvcache(c["k_cache"], c["v_cache"], c["weights"], c["tables"], c["lens"], 2)
    plan = type("Plan", (), dict(num_heads=4, num_kv_heads=2, rows=2))
    with pytest.raises(ValueError, match="GPU"):
        prefill_key_weights(c["query"], c["k_cache"], c["weights"], plan, None, 0.1, 64, c["tables"])


@pytest.mark.parametrize("window,sinks", [(0, 0), (-1, 0), (2.5, 0), (4, -1), (4, 0.5)])
def test_windows_that_are_none(window, sinks):
    c = _cpu_case()
    meta = (c["tables"], c["lens"], c["cu"], c["positions"], 0.1, 4, 2, 64, 16, 16)
    with pytest.raises(ValueError, match="window|sinks"):
        paged_attention_window(c["query"], c["k_cache"], c["v_cache"], *meta, window=window, sinks=sinks)


def test_few_rows_rule():
    assert few_rows_serve_prefill([24, 3], 16, 8) and not few_rows_serve_prefill([25], 16, 8)
    assert few_rows_serve_prefill([1], 40, 1) and not few_rows_serve_prefill([], 16, 8)


def _lists(build, words, ql, kl):
    n = len(ql)
    counts = (ctypes.c_int32 * 4)()
    q, k = (ctypes.c_int64 * n)(*ql), (ctypes.c_int64 * n)(*kl)
    small = np.zeros(1, dtype=np.int32)
    assert build(q, k, n, small.ctypes.data, 1, counts) == -3  # (too small: the counts all the same)
    buf = np.zeros(words(counts), dtype=np.int32)
    assert build(q, k, n, buf.ctypes.data, buf.size, counts) == 0
    return buf, list(counts)


@pytest.mark.parametrize("H,Hkv", [(16, 8), (32, 8), (3, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 4), (100, 300), (5000, 7)])
@pytest.mark.parametrize("cus", [256, 8])
def test_window_tiles_cover_every_visible_key_once(H, Hkv, window, sinks, cus):
    ql, kl = [700, 1, 130, 64], [700, 900, 4130, 64]
    buf, (nt, nm, rows, slots) = _lists(
        lambda q, k, n, at, w, c: _lib.lib().nsv_prefill_window_tiles(q, k, n, H, Hkv, 16, cus, window, sinks, at, w, c),
        lambda c: 8 * c[0] + 4 * c[1], ql, kl)
    tiles = buf[:8 * nt].reshape(nt, 8)
    seen = {}
    for seq, row0, nr, pos, _, begin, end, slot in tiles.tolist():
        first = max(0, pos - window + 1) if window else 0
        head = sinks if window and first > sinks else 0
        gap = first - head if head or (window and first > sinks) else 0
        assert 0 < nr <= rows and begin % 64 == 0 and begin < end
        for r in range(nr):
            keys = seen.setdefault((seq, row0 + r), [])
            for v in range(begin, end):
                j = v if v < head else v + gap
                p = pos + r
                if j <= p and (not window or j > p - window or j < sinks):
                    keys.append(j)
    row = 0
    for seq, (q, k) in enumerate(zip(ql, kl)):
        for p in range(k - q, k):
            want = [j for j in range(p + 1) if not window or j > p - window or j < sinks]
            assert sorted(seen[(seq, row)]) == want, (seq, p)
            row += 1


def test_window_tiles_of_no_window_are_the_prefill_tiles():
    ql, kl = [700, 1, 130], [700, 900, 4130]
    words = lambda c: 8 * c[0] + 4 * c[1]  # noqa: E731
    a, ca = _lists(lambda q, k, n, at, w, c: _lib.lib().nsv_prefill_tiles(q, k, n, 16, 8, 16, 256, at, w, c), words, ql, kl)
    b, cb = _lists(lambda q, k, n, at, w, c: _lib.lib().nsv_prefill_window_tiles(q, k, n, 16, 8, 16, 256, 0, 0, at, w, c),
                   words, ql, kl)
    assert ca == cb and (a == b).all()
    bad = (ctypes.c_int64 * 1)(5), (ctypes.c_int64 * 1)(5)
    counts = (ctypes.c_int32 * 4)()
    assert _lib.lib().nsv_prefill_window_tiles(*bad, 1, 16, 8, 16, 256, -1, 0, a.ctypes.data, a.size, counts) == -1
    assert _lib.lib().nsv_prefill_window_tiles(*bad, 1, 16, 8, 16, 256, 4, -1, a.ctypes.data, a.size, counts) == -1


@pytest.mark.parametrize("H,Hkv,cus", [(16, 8, 256), (4, 1, 8), (3, 3, 256)])
def test_key_weight_units_cover_every_pair_once(H, Hkv, cus):
    ql, kl = [700, 1, 130, 64], [700, 900, 1130, 64]
    buf, (nu, ns, _, _) = _lists(
        lambda q, k, n, at, w, c: _lib.lib().nsv_key_weights_units(q, k, n, H, Hkv, cus, at, w, c),
        lambda c: 8 * c[0] + 6 * c[1], ql, kl)
    units, sums = buf[:8 * nu].reshape(nu, 8), buf[8 * nu:].reshape(ns, 6)
    G, at = H // Hkv, 0
    for seq, key0, keys, unit, count, fresh in sums.tolist():
        assert unit == at and keys <= 256 and fresh == kl[seq] - ql[seq]
        at += count
        first = max(0, key0 - fresh)  # rows before it see none of the block's keys
        tiles = G * -(-(ql[seq] - first) // 64)
        spans = units[unit:unit + count]
        assert (spans[:, 0] == seq).all() and (spans[:, 1] == key0).all() and (spans[:, 2] == keys).all()
        assert (spans[:, 3] == sum(ql[:seq])).all() and (spans[:, 4] == ql[seq]).all() and (spans[:, 5] == fresh).all()
        assert spans[0, 6] == 0 and spans[-1, 7] == tiles and (spans[1:, 6] == spans[:-1, 7]).all()
        assert (spans[:, 6] < spans[:, 7]).all()
    assert at == nu
    covered = [[(k0, n) for s, k0, n, *_ in sums.tolist() if s == b] for b in range(4)]
    assert [sum(n for _, n in c) for c in covered] == kl
