"""The bounded cache's operators over pools whose later pages lie past 2^32
bytes from their start."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import (KeyWeightsPlan, PrefillPlan, evict_kvcache, paged_attention_weights,
                                          paged_attention_window, prefill_attention, prefill_key_weights)
from naivllm_amd.utils import synth
from oracle import bounded as ob
from tests.bounded_util import as_device, check_attention, weight_error

pytestmark = pytest.mark.gpu
BS, HKV, H, D = 256, 8, 16, 128
PAGES = 9000  # of 512 KiB: 4.4 GiB for K, and for V


@pytest.fixture(scope="module")
def pool():
    """The last pages hold two sequences' keys; the others are not read."""
    vb = synth.verify_batch(101, [700, 300], [40, 40], num_heads=H, num_kv_heads=HKV, head_dim=D, block_size=BS)
    used = vb.block_tables[vb.block_tables >= 0]
    k, v = (torch.empty((PAGES, BS, HKV, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tables = vb.block_tables.copy()
    for p in used:
        far = PAGES - 1 - int(p)
        k[far], v[far] = as_device(vb.k_cache[p], "bf16"), as_device(vb.v_cache[p], "bf16")
        tables[vb.block_tables == p] = far
    yield vb, k, v, torch.from_numpy(tables).cuda(), tables
    del k, v
    torch.cuda.empty_cache()


def _weights_of(weights, tables, n, b):
    j = np.arange(n)
    return weights[tables[b, j // BS], :, j % BS].cpu().numpy()


def test_few_rows_and_prompts(pool):
    print("case: far pages", flush=True)
    vb, k, v, tables, np_tables = pool
    scale = 1.0 / np.sqrt(D)
    q = as_device(vb.q, "bf16")
    lens = torch.from_numpy(vb.context_lens).cuda()
    # three rows of each sequence
    rows = np.r_[37:40, 77:80]
    cu, pos = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda"), torch.from_numpy(vb.positions[rows]).cuda()
    meta = (tables, lens, cu, pos, scale, H, HKV, D, BS, 16)
    few = (vb.q[rows], vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, np.array([0, 3, 6]), vb.positions[rows],
           scale, HKV)
    want, want_abs, mag, _ = ob.attention(*few, 100, 4)
    out = paged_attention_window(q[rows], k, v, *meta, window=100, sinks=4, max_q_len=3)
    check_attention(out, want, want_abs, mag, "bf16", 110, "window")
    weights = torch.zeros((PAGES, HKV, BS), device="cuda")
    want, want_abs, mag, sums = ob.attention(*few)
    out = paged_attention_weights(q[rows], k, v, weights, *meta, max_q_len=3)
    check_attention(out, want, want_abs, mag, "bf16", 700, "weights")
    share = weight_error(mag.max(), 700, D) + 20 * 2.0 ** -24
    for b, n in enumerate((700, 300)):
        got = _weights_of(weights, np_tables, n, b)
        assert (np.abs(got - sums[b].T) <= share * sums[b].T + 1e-30).all()
    # all rows as a prompt's
    new, ends = [40, 40], [700, 300]
    dev = torch.device("cuda", 0)
    every = (vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q, vb.positions, scale, HKV)
    want, want_abs, mag, _ = ob.attention(*every, 100, 4)
    out = prefill_attention(q, k, v, PrefillPlan(new, ends, H, HKV, BS, dev, window=100, sinks=4), scale, D, tables)
    check_attention(out, want, want_abs, mag, "bf16", 110, "window prompt")
    stats = torch.empty((80, H, 2), device="cuda")
    want, want_abs, mag, sums = ob.attention(*every)
    out = prefill_attention(q, k, v, PrefillPlan(new, ends, H, HKV, BS, dev), scale, D, tables, stats=stats)
    check_attention(out, want, want_abs, mag, "bf16", 700, "prompt")
    weights.zero_()
    prefill_key_weights(q, k, weights, KeyWeightsPlan(new, ends, H, HKV, BS, dev), stats, scale, D, tables)
    share = weight_error(mag.max(), 700, D) + 100 * 2.0 ** -24
    for b, n in enumerate((700, 300)):
        got = _weights_of(weights, np_tables, n, b)
        assert (np.abs(got - sums[b].T) <= share * sums[b].T + 1e-30).all()


def test_eviction(pool):
    print("case: far pages evicted", flush=True)
    vb, k, v, tables, np_tables = pool
    weights = torch.rand((PAGES, HKV, BS), device="cuda")
    old = [_weights_of(weights, np_tables, n, b) for b, n in enumerate((700, 300))]
    lens, kept = evict_kvcache(k, v, weights, tables, torch.from_numpy(vb.context_lens).cuda(), 280, sinks=4, recent=20)
    kept = kept.cpu().numpy()
    for b, n in enumerate((700, 300)):
        for h in range(HKV):
            middle = sorted(range(4, n - 20), key=lambda j: (-old[b][j, h], j))[:256]
            want = np.array(sorted([*range(4), *middle, *range(n - 20, n)]))
            assert (kept[b, h] == want).all()
            for cache, mine in ((k, vb.k_cache), (v, vb.v_cache)):
                i = np.arange(280)
                got = cache[tables[b].long().cpu()[i // BS].cuda(), torch.from_numpy(i % BS).cuda(), h]
                src = as_device(mine[vb.block_tables[b, want // BS], want % BS, h], "bf16")
                assert torch.equal(got, src)
    assert lens.tolist() == [280, 280]
