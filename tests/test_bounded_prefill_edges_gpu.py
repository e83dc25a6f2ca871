"""The prompts' bounded operators at their edges."""

import numpy as np
import pytest
import torch

from naivllm_amd import _lib
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


def _lse2(vb, scale, window, sinks):
    """log2 of every row's sum of exponentials [T, H], and the scores' magnitudes."""
    lse, mag = np.full((len(vb.q), vb.num_heads), -np.inf), np.zeros((len(vb.q), vb.num_heads))
    G = vb.num_heads // vb.num_kv_heads
    for b, n in enumerate(vb.context_lens):
        j, rows = np.arange(n), slice(vb.cu_seqlens_q[b], vb.cu_seqlens_q[b + 1])
        seen = ob.visible(vb.positions[rows], j, window or None, sinks)
        page = vb.block_tables[b, j // vb.block_size]
        for h in range(vb.num_heads):
            K = vb.k_cache[page, j % vb.block_size, h // G]
            s = np.where(seen, vb.q[rows, h] @ K.T * scale, -np.inf) * np.log2(np.e)
            top = s.max(1)
            lse[rows, h] = top + np.log2(np.exp2(s - top[:, None]).sum(1))
            mag[rows, h] = (np.abs(vb.q[rows, h]) @ np.abs(K).T * seen).max(1) * abs(scale)
    return lse, mag


@pytest.mark.parametrize("new,prefix,H,Hkv,window,sinks,waves,cut", [
    ([500, 1, 77, 130], [0, 0, 300, 65], 4, 2, 100, 4, 4, False),
    ([40], [1500], 2, 1, 900, 3, 4, True),         # keys cut over workgroups
    ([1100] * 4, [2200] * 4, 16, 8, 1700, 4, 8, False),
    ([900], [3000], 2, 1, 1700, 70, 8, True),
    ([300, 90], [0, 200], 3, 1, 0, 0, 4, False)])  # no window
def test_statistics_of_the_library_entry(new, prefix, H, Hkv, window, sinks, waves, cut):
    """nsv_prefill_window_attention leaves every row's (m, r), under a window
    as without one, beside its outputs."""
    print(f"case: statistics {new} window {window}", flush=True)
    vb = _batch(101, new, prefix, H, Hkv)
    t = to_device(vb)
    ends, scale = vb.context_lens.tolist(), 1.0 / np.sqrt(128)
    plan = PrefillPlan(new, ends, H, Hkv, 64, DEV, window=window, sinks=sinks)
    assert (plan.nmerges > 0) == cut and plan.tile_rows * (2 if H // Hkv % 2 == 0 else 1) == 32 * waves
    out = torch.empty_like(t["query"])
    stats = torch.full((sum(new), H, 2), float("nan"), device="cuda")
    part = torch.empty(max(1, plan.slots) * H * plan.tile_rows * 130, device="cuda")
    at = plan.work.data_ptr()
    rc = _lib.lib().nsv_prefill_window_attention(
        out.data_ptr(), t["query"].data_ptr(), t["k_cache"].data_ptr(), t["v_cache"].data_ptr(),
        t["block_tables"].data_ptr(), at, plan.ntiles, plan.tile_rows, at + plan.ntiles * 32, plan.nmerges, scale, H, Hkv,
        128, 64, vb.block_tables.shape[1], window, sinks, stats.data_ptr(), part.data_ptr(),
        torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0
    check_attention(out, *ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q,
                                       vb.positions, scale, Hkv, window or None, sinks)[:3], "bf16", max(ends))
    want, mag = _lse2(vb, scale, window, sinks)
    m, r = stats.cpu().numpy().astype(np.float64).transpose(2, 0, 1)
    # the sum's relative error is a weight's; m is rounded once, r twice (its sum's and its own)
    bound = np.log2(np.e) * (weight_error(mag, max(ends), 128) + 4 * EPS32) + EPS32 * (np.abs(m) + mag * np.log2(np.e))
    assert (np.abs(m - np.log2(r) - want) <= bound).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 3)])
@pytest.mark.parametrize("scale", [0.0, -0.09, 2.0])
def test_scales_of_every_sign(window, sinks, scale):
    """As the few-row operators': at 0 a row's keys weigh the same, below it
    the smallest products weigh most."""
    print(f"case: prompt scale {scale} window {window}", flush=True)
    vb = _batch(102, [300, 40, 5], [0, 900, 33])
    vb.block_tables[0, 1] = -1
    t = to_device(vb)
    want, want_abs, mag, sums = ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens,
                                             vb.cu_seqlens_q, vb.positions, scale, 2, window or None, sinks)
    mag = np.abs(mag)
    new, ends = [300, 40, 5], vb.context_lens.tolist()
    plan = PrefillPlan(new, ends, 4, 2, 64, DEV, window=window, sinks=sinks)
    stats = None if window else torch.empty((345, 4, 2), device="cuda")
    out = prefill_attention(t["query"], t["k_cache"], t["v_cache"], plan, scale, 128, t["block_tables"], stats=stats)
    check_attention(out, want, want_abs, mag, "bf16", max(ends), f"scale {scale}")
    if window:
        return
    old = synth.normal(9, 3, vb.k_cache.shape[0] * 2 * 64).reshape(-1, 2, 64).astype(np.float32) ** 2
    weights = as_device(old)
    prefill_key_weights(t["query"], t["k_cache"], weights, KeyWeightsPlan(new, ends, 4, 2, 64, DEV), stats, scale, 128,
                        t["block_tables"])
    want_w = ob.add_weights(old, sums, vb.block_tables, [0, 900, 33])
    bound = (weight_error(mag.max(), max(ends), 128) + (300 * 2 + 2) * EPS32) * np.abs(want_w) + 1e-30
    assert (np.abs(weights.cpu().numpy() - want_w) <= bound).all()


def test_a_row_of_nan_whose_keys_are_cut():
    """NaN for the row, its statistics and the weights of the keys it sees,
    also where several workgroups share its keys; nothing for other rows."""
    print("case: prompt, a NaN row over cut keys", flush=True)
    vb = _batch(103, [40], [1500], 2, 1)
    plan = PrefillPlan([40], [1540], 2, 1, 64, DEV)
    assert plan.nmerges > 0
    results = []
    for bad in (False, True):
        t = to_device(vb)
        if bad:
            t["query"][17, 1] = float("nan")
        stats, w = torch.empty((40, 2, 2), device="cuda"), torch.ones((vb.k_cache.shape[0], 1, 64), device="cuda")
        out = prefill_attention(t["query"], t["k_cache"], t["v_cache"], plan, 0.09, 128, t["block_tables"], stats=stats)
        prefill_key_weights(t["query"], t["k_cache"], w, KeyWeightsPlan([40], [1540], 2, 1, 64, DEV), stats, 0.09, 128,
                            t["block_tables"])
        j = np.arange(1540)
        results.append((out, w[torch.from_numpy(vb.block_tables[0, j // 64]).long().cuda(), 0,
                               torch.from_numpy(j % 64).cuda()], stats))
    (good, w_good, s_good), (got, w_got, s_got) = results
    assert s_got[17, 1, 1].isnan() and got[17, 1].isnan().all() and w_got[:1518].isnan().all()
    got[17, 1] = good[17, 1] = 0
    s_got[17, 1] = s_good[17, 1] = 0
    assert torch.equal(got, good) and torch.equal(s_got, s_good) and torch.equal(w_got[1518:], w_good[1518:])
