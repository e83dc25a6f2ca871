"""prefill_attention with a window, its statistics, and prefill_key_weights
against the oracle."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import KeyWeightsPlan, PrefillPlan, prefill_attention, prefill_key_weights
from naivllm_amd.utils import synth
from oracle import bounded as ob
from tests.bounded_util import EPS32, as_device, check_attention, weight_error
from tests.gpu_util import to_device

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _batch(seed, new, prefix, H=4, Hkv=2, D=128, block_size=64):
    return synth.verify_batch(seed, [p + n for p, n in zip(prefix, new)], new, num_heads=H, num_kv_heads=Hkv, head_dim=D,
                              block_size=block_size)


def _run(vb, window, sinks, paged=True, stats=None):
    t = to_device(vb)
    new, ends = np.diff(vb.cu_seqlens_q).tolist(), vb.context_lens.tolist()
    bs = vb.block_size if paged else None
    plan = PrefillPlan(new, ends, vb.num_heads, vb.num_kv_heads, bs, DEV, window=window, sinks=sinks)
    k, v, tables = t["k_cache"], t["v_cache"], t["block_tables"]
    if not paged:
        rows = [np.array([vb.block_tables[b, j // vb.block_size] * vb.block_size + j % vb.block_size for j in range(n)])
                for b, n in enumerate(ends)]
        at = torch.from_numpy(np.concatenate(rows)).to("cuda")
        k, v, tables = k.flatten(0, 1)[at], v.flatten(0, 1)[at], None
    out = prefill_attention(t["query"], k, v, plan, 1.0 / np.sqrt(vb.head_dim), vb.head_dim, tables, stats=stats)
    torch.cuda.synchronize()
    return out, t


def _oracle(vb, window=None, sinks=0):
    return ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q, vb.positions,
                        1.0 / np.sqrt(vb.head_dim), vb.num_kv_heads, window, sinks)


def _check(vb, window, sinks, paged=True):
    want, want_abs, mag, _ = _oracle(vb, window or None, sinks)
    out, _ = _run(vb, window, sinks, paged)
    keys = min(int(vb.context_lens.max()), (window or 1 << 30) + sinks)
    check_attention(out, want, want_abs, mag, "bf16", keys, f"window {window} sinks {sinks}")


@pytest.mark.parametrize("window", [1, 3, 63, 64, 65, 200, 330, 5000])
@pytest.mark.parametrize("sinks", [0, 1, 4, 64, 130])
def test_windows(window, sinks):
    print(f"case: prompt window {window} sinks {sinks}", flush=True)
    _check(_batch(51, [500, 1, 77, 130], [0, 0, 300, 65]), window, sinks)


@pytest.mark.parametrize("H,Hkv,D", [(2, 1, 128), (3, 1, 64), (8, 8, 64), (8, 2, 64), (5, 1, 128), (16, 8, 128)])
@pytest.mark.parametrize("paged", [True, False])
def test_head_layouts(H, Hkv, D, paged):
    print(f"case: prompt heads {H}/{Hkv} dim {D} paged {paged}", flush=True)
    _check(_batch(52, [300, 40], [0, 0], H, Hkv, D, 16), 100, 5, paged)


@pytest.mark.parametrize("block_size", [1, 16, 1024])
def test_page_sizes_and_long_prefixes(block_size):
    print(f"case: prompt page {block_size}", flush=True)
    _check(_batch(53, [150, 20], [3000, 5], 2, 1, 64, block_size), 2500, 5)
    _check(_batch(53, [150, 20], [3000, 5], 2, 1, 64, block_size), 60, 5)


def test_many_rows_of_eight_wave_tiles():
    print("case: prompt 2600 rows, window 1700", flush=True)
    vb = _batch(54, [2600], [40], 2, 1, 128, 64)
    _check(vb, 1700, 4)


def test_keys_that_no_row_sees_are_not_read():
    print("case: prompt NaN between sinks and windows", flush=True)
    vb = _batch(55, [40], [900], 4, 2, 128, 32)
    want, want_abs, mag, _ = _oracle(vb, 128, 6)
    for j in list(range(6, 900 - 127)) + list(range(940, 960)):
        page = int(vb.block_tables[0, j // 32])
        vb.k_cache[page, j % 32] = vb.v_cache[page, j % 32] = np.nan
    vb.block_tables[0, 1:20] = -1
    out, _ = _run(vb, 128, 6)
    check_attention(out, want, want_abs, mag, "bf16", 134, "NaN outside")


def test_unmapped_pages():
    print("case: prompt holes", flush=True)
    vb = _batch(56, [200, 50, 30], [100, 0, 40], 4, 2, 128, 16)
    vb.block_tables[0, [0, 9, 18]] = -1
    vb.block_tables[1, :] = -1
    vb.block_tables[2, 3:] = -1
    _check(vb, 20, 4)
    _check(vb, 1000, 0)


def test_a_window_of_every_key_is_no_window():
    vb = _batch(57, [700], [100], 4, 2, 128, 64)
    a, _ = _run(vb, 0, 0)
    b, _ = _run(vb, 800, 0)
    assert torch.equal(a, b)


def _check_key_weights(vb, seed=5):
    want, want_abs, mag, sums = _oracle(vb)
    stats = torch.full((len(vb.q), vb.num_heads, 2), float("nan"), device="cuda")
    out, t = _run(vb, 0, 0, stats=stats)
    check_attention(out, want, want_abs, mag, "bf16", int(vb.context_lens.max()), "out")
    nb, bs = vb.k_cache.shape[:2]
    old = synth.normal(seed, 3, nb * vb.num_kv_heads * bs).reshape(nb, vb.num_kv_heads, bs).astype(np.float32) ** 2
    weights = as_device(old)
    new, ends = np.diff(vb.cu_seqlens_q).tolist(), vb.context_lens.tolist()
    plan = KeyWeightsPlan(new, ends, vb.num_heads, vb.num_kv_heads, bs, DEV)
    prefill_key_weights(t["query"], t["k_cache"], weights, plan, stats, 1.0 / np.sqrt(vb.head_dim), vb.head_dim,
                        t["block_tables"])
    torch.cuda.synchronize()
    want_w = ob.add_weights(old, sums, vb.block_tables, [e - n for n, e in zip(new, ends)])
    got = weights.cpu().numpy().astype(np.float64)
    rows = max(new) * vb.num_heads // vb.num_kv_heads
    # every weight's own error, as many additions as rows (fewer: lanes and parts), the addition to the old value
    bound = (weight_error(mag.max(), max(ends), vb.head_dim) + (rows + 2) * EPS32) * np.abs(want_w) + 1e-30
    assert (np.abs(got - want_w) <= bound).all(), f"worst by {(np.abs(got - want_w) / bound).max():.2f}"
    same = want_w == old
    assert (got[same] == old[same]).all()


@pytest.mark.parametrize("H,Hkv,D", [(2, 1, 128), (3, 1, 64), (8, 8, 64), (16, 8, 128)])
@pytest.mark.parametrize("block_size", [16, 256])
def test_key_weights(H, Hkv, D, block_size):
    print(f"case: prompt weights {H}/{Hkv} {D} page {block_size}", flush=True)
    _check_key_weights(_batch(58, [300, 1, 64, 257], [0, 0, 70, 300], H, Hkv, D, block_size))


def test_key_weights_of_many_blocks_and_parts():
    print("case: prompt weights 2100 rows behind 600 keys", flush=True)
    _check_key_weights(_batch(59, [2100], [600], 2, 1, 128, 64))


def test_key_weights_unmapped_pages():
    print("case: prompt weights holes", flush=True)
    vb = _batch(60, [200, 50], [100, 0], 4, 2, 128, 16)
    vb.block_tables[0, [0, 9, 18]] = -1
    vb.block_tables[1, :] = -1
    _check_key_weights(vb)


def test_a_row_of_nan_stays_alone():
    print("case: prompt, a NaN row", flush=True)
    vb = _batch(61, [200, 50], [100, 0], 4, 2, 128, 16)
    scale, tables = 1.0 / np.sqrt(128), None
    results = []
    for bad in (False, True):
        t = to_device(vb)
        tables = t["block_tables"]
        if bad:
            t["query"][150, 3] = float("nan")
        plan, adder = (PrefillPlan([200, 50], [300, 50], 4, 2, 16, DEV), KeyWeightsPlan([200, 50], [300, 50], 4, 2, 16, DEV))
        stats = torch.empty((250, 4, 2), device="cuda")
        out = prefill_attention(t["query"], t["k_cache"], t["v_cache"], plan, scale, 128, tables, stats=stats)
        w = torch.ones((vb.k_cache.shape[0], 2, 16), device="cuda")
        prefill_key_weights(t["query"], t["k_cache"], w, adder, stats, scale, 128, tables)
        j = np.arange(300)
        results.append((out, w[torch.from_numpy(vb.block_tables[0, j // 16]).long().cuda(), :, torch.from_numpy(j % 16).cuda()]))
    (good, w_good), (got, w_got) = results
    assert got[150, 3].isnan().all() and w_got[:251, 1].isnan().all()
    got[150, 3] = good[150, 3] = 0
    w_got[:251, 1] = w_good[:251, 1] = 0
    assert torch.equal(got, good) and torch.equal(w_got, w_good)
