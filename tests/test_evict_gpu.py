"""evict_kvcache against the oracle, bit for bit."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import evict_kvcache
from naivllm_amd.utils import synth
from oracle import bounded as ob

pytestmark = pytest.mark.gpu


def _case(seed, lens, Hkv=2, D=64, block_size=16, dtype=torch.bfloat16, levels=None, spare=0):
    """Caches, weights (levels: that many distinct values) and tables."""
    pages = [-(-n // block_size) for n in lens]
    nb = sum(pages) + 3 + spare
    perm = synth.randperm(seed, 1, nb)
    tables = np.full((len(lens), max(pages + [1])), -1, dtype=np.int32)
    at = 0
    for b, p in enumerate(pages):
        tables[b, :p] = perm[at:at + p]
        at += p
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((nb, block_size, Hkv, D), generator=gen).to(dtype) for _ in range(2))
    w = torch.randn((nb, Hkv, block_size), generator=gen) ** 2
    if levels:
        w = (w * levels).floor() / levels
    return k, v, w, tables, perm[at:].astype(np.int32)


def _check(k, v, w, tables, lens, budget, sinks=0, recent=0, out_tables=None):
    lens = np.array(lens, dtype=np.int64)
    to_np = lambda x: x.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32).numpy()  # noqa: E731
    want = ob.evict(to_np(k), to_np(v), w.numpy(), tables, lens, budget, sinks, recent, out_tables)
    gk, gv, gw = (x.cuda() for x in (k, v, w))
    out = None if out_tables is None else torch.from_numpy(out_tables).cuda()
    new_lens, kept = evict_kvcache(gk, gv, gw, torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda(), budget,
                                   sinks=sinks, recent=recent, out_block_tables=out)
    torch.cuda.synchronize()
    assert (kept.cpu().numpy() == want[4]).all(), "kept"
    assert (new_lens.cpu().numpy() == want[3]).all(), "lens"
    for name, got, x in (("k", to_np(gk.cpu()), want[0]), ("v", to_np(gv.cpu()), want[1])):
        assert (got == x).all(), name
    assert (gw.cpu().numpy().view(np.int32) == want[2].view(np.int32)).all(), "weights"


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 0, 0), (100, 4, 30), (100, 60, 40),
                                                 (300, 17, 0), (5000, 4, 4)])
def test_budgets(budget, sinks, recent):
    print(f"case: evict budget {budget} sinks {sinks} recent {recent}", flush=True)
    lens = [700, 1, 100, 101, 0, 2333]
    _check(*_case(71, lens)[:4], lens, budget, sinks, recent)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hkv,D,block_size", [(1, 64, 1), (8, 128, 256), (3, 128, 16), (2, 96, 4), (1, 32, 8)])
def test_layouts(dtype, Hkv, D, block_size):
    print(f"case: evict {Hkv} heads dim {D} page {block_size} {dtype}", flush=True)
    lens = [600, 1030]
    _check(*_case(72, lens, Hkv, D, block_size, dtype)[:4], lens, 257, 3, 20)


@pytest.mark.parametrize("levels", [1, 4])
def test_equal_weights_keep_the_lower_positions(levels):
    print(f"case: evict {levels} levels", flush=True)
    lens = [3000, 900]
    k, v, w, tables, _ = _case(73, lens, levels=levels)
    _check(k, v, w, tables, lens, 500, 4, 50)
    _check(k, v, torch.zeros_like(w), tables, lens, 500, 4, 50)


def test_weights_of_every_kind_have_one_order():
    print("case: evict special weights", flush=True)
    lens = [800]
    k, v, w, tables, _ = _case(74, lens)
    values = torch.tensor([0.0, -0.0, float("nan"), float("inf"), float("-inf"), -1.0, 1e-45, -1e-45, 3e38, 1.0])
    w = values[torch.randint(0, len(values), w.shape, generator=torch.Generator().manual_seed(1))]
    for budget in (30, 100, 250, 500, 790):
        _check(k, v, w, tables, lens, budget, 2, 5)


def test_pages_apart_leave_the_old_ones():
    print("case: evict apart", flush=True)
    lens = [700, 20, 300]
    k, v, w, tables, free = _case(75, lens, spare=60)
    out = np.full((3, 20), -1, dtype=np.int32)
    out[0, :13], out[1, :2], out[2, :13] = free[:13], free[13:15], free[15:28]
    _check(k, v, w, tables, lens, 200, 4, 30, out)


@pytest.mark.parametrize("Hkv,D", [(2, 64), (1, 128)])
def test_many_rows_of_few_sequences(Hkv, D):
    print(f"case: evict by way of staging rows {Hkv} {D}", flush=True)
    lens = [9000, 5000, 8193]
    _check(*_case(78, lens, Hkv, D, 64)[:4], lens, 5000, 4, 100)


def test_a_long_context():
    print("case: evict 70000 keys", flush=True)
    lens = [70000, 40000]
    _check(*_case(76, lens, 1, 32, 64, levels=64)[:4], lens, 3001, 4, 100)


def test_a_table_narrower_than_the_context():
    lens = [400]
    k, v, w, tables, _ = _case(77, lens)
    _check(k, v, w, tables[:, :20].copy(), lens, 100, 4, 10)


@pytest.mark.parametrize("apart", [False, True])
def test_many_keys_stay_on_small_pages(apart):
    """More places than the workgroup lists at a time, more pages than it holds."""
    print(f"case: evict 25000 of 30000 keys, pages of 4, apart {apart}", flush=True)
    lens = [30000, 8193, 25001]
    k, v, w, tables, free = _case(79, lens, 1, 32, 4, levels=1000, spare=6250 * 3)
    out = free[:6250 * 3].reshape(3, 6250).copy() if apart else None
    _check(k, v, w, tables, lens, 25000, 4, 100, out)


def test_weights_off_their_alignment():
    print("case: evict, weights at an odd address", flush=True)
    k, v, w, tables, _ = _case(80, [3000, 700])
    odd = torch.empty(w.numel() + 1, device="cuda")[1:].view(w.shape)
    odd.copy_(w)
    aligned = w.cuda()
    results = []
    for weights in (aligned, odd):
        gk, gv = k.cuda(), v.cuda()
        _, kept = evict_kvcache(gk, gv, weights, torch.from_numpy(tables).cuda(),
                                torch.tensor([3000, 700], device="cuda"), 333, sinks=3, recent=40)
        results.append((gk, gv, weights, kept))
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("block_size,apart", [(64, False), (16, True), (2, False)])
def test_long_contexts_of_many_kept_keys(block_size, apart):
    print(f"case: evict 50000 -> 20001 keys, pages of {block_size}, apart {apart}", flush=True)
    lens = [50000, 33000, 20002]
    pages = -(-20001 // block_size)
    k, v, w, tables, free = _case(81, lens, 1, 32, block_size, levels=500, spare=3 * pages)
    _check(k, v, w, tables, lens, 20001, 4, 100, free[:3 * pages].reshape(3, pages).copy() if apart else None)
