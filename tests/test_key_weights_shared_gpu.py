"""Key weights of pages that one sequence of a call fills and others read: a
step's prompts may share a prefix that the first of them computes."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import (Attention, KeyWeightsPlan, PrefillPlan, paged_attention_weights, prefill_attention,
                                          prefill_key_weights)
from naivllm_amd.utils import synth
from naivllm_amd.utils.context import reset_context, set_context
from oracle import bounded as ob
from tests.bounded_util import as_device, weight_error
from tests.gpu_util import to_device

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _shared(seed, lens, rows, owner, pages, **kw):
    """Every sequence's first pages are those of sequence ``owner``."""
    vb = synth.verify_batch(seed, lens, rows, block_size=16, **kw)
    for b in range(len(lens)):
        vb.block_tables[b, :pages] = vb.block_tables[owner, :pages]
    return vb


def _check(vb, owner, add, seed=5):
    """add(tensors, weights) against the oracle's sums, the owner's first."""
    first = [int(vb.positions[vb.cu_seqlens_q[b]]) for b in range(len(vb.context_lens))]
    _, _, mag, sums = ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q,
                                   vb.positions, 1.0 / np.sqrt(vb.head_dim), vb.num_kv_heads)
    order = [owner] + [b for b in sums if b != owner]
    nb, bs = vb.k_cache.shape[:2]
    old = synth.normal(seed, 3, nb * vb.num_kv_heads * bs).reshape(nb, vb.num_kv_heads, bs).astype(np.float32) ** 2
    want = ob.add_weights(old, {b: sums[b] for b in order}, vb.block_tables, first)
    got = as_device(old)
    add(to_device(vb), got)
    torch.cuda.synchronize()
    rows = int(np.diff(vb.cu_seqlens_q).max()) * vb.num_heads // vb.num_kv_heads
    # a weight's own error, the additions of a sequence's rows, one addition per sequence
    share = weight_error(mag.max(), int(vb.context_lens.max()), vb.head_dim) + (rows + len(first) + 2) * 2.0 ** -24
    assert (np.abs(got.cpu().numpy() - want) <= share * want + 1e-30).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("owner", [0, 5])
@pytest.mark.parametrize("H,Hkv,rows", [(16, 8, 9), (40, 1, 2)])  # stored scores; keys read again
def test_few_rows(dtype, owner, H, Hkv, rows):
    print(f"case: shared new keys {dtype} {H}/{Hkv} owner {owner}", flush=True)
    lens = [120 + 7 * b for b in range(6)]
    lens[owner] = 32                              # two pages, its rows' own keys in the second
    vb = _shared(131, lens, [rows] * 6, owner, 2, num_heads=H, num_kv_heads=Hkv, dtype=dtype)
    _check(vb, owner, lambda t, w: paged_attention_weights(
        t["query"], t["k_cache"], t["v_cache"], w, t["block_tables"], t["context_lens"], t["cu_seqlens_q"], t["positions"],
        1 / np.sqrt(128), H, Hkv, 128, 16, 64, max_q_len=rows))


@pytest.mark.parametrize("owner", [0, 3])
def test_prompts(owner):
    print(f"case: prompts behind a prefix of the same step, owner {owner}", flush=True)
    new, prefix = [60, 300, 33, 70], [192] * 4
    new[owner], prefix[owner] = 400, 0
    vb = _shared(132, [n + p for n, p in zip(new, prefix)], new, owner, 12, num_heads=4, num_kv_heads=2)

    def add(t, w):
        ends = vb.context_lens.tolist()
        stats = torch.empty((sum(new), 4, 2), device="cuda")
        scale = 1 / np.sqrt(128)
        prefill_attention(t["query"], t["k_cache"], t["v_cache"], PrefillPlan(new, ends, 4, 2, 16, DEV), scale, 128,
                          t["block_tables"], stats=stats)
        prefill_key_weights(t["query"], t["k_cache"], w, KeyWeightsPlan(new, ends, 4, 2, 16, DEV), stats, scale, 128,
                            t["block_tables"])

    _check(vb, owner, add)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("owner", [0, 2])
def test_the_layer_over_a_step_that_shares_its_prefix(dtype, owner):
    """One prompt computes a prefix, two of the same step have it behind them."""
    print(f"case: layer, shared prefix {dtype} owner {owner}", flush=True)
    new, prefix = [33, 90, 100], [128] * 3
    new[owner], prefix[owner] = 300, 0
    vb = _shared(133, [n + p for n, p in zip(new, prefix)], new, owner, 8, num_heads=4, num_kv_heads=2, dtype=dtype)
    layer = Attention(4, 128, 1.0, 2, 16)

    def add(t, w):
        layer.k_cache, layer.v_cache, layer.key_weights = t["k_cache"], t["v_cache"], w
        at = torch.from_numpy(np.concatenate([
            vb.block_tables[b, np.arange(p, p + n) // 16].astype(np.int64) * 16 + np.arange(p, p + n) % 16
            for b, (n, p) in enumerate(zip(new, prefix))])).cuda()
        k, v = t["k_cache"].flatten(0, 1)[at], t["v_cache"].flatten(0, 1)[at]
        set_context(True, cu_seqlens_q=t["cu_seqlens_q"], slot_mapping=at, context_lens=t["context_lens"],
                    block_tables=t["block_tables"], seqlens_q=new, seqlens_k=vb.context_lens.tolist())
        try:
            layer(t["query"], k, v)
        finally:
            reset_context()

    _check(vb, owner, add)


@pytest.mark.filterwarnings("ignore:Synchronization debug mode")
@pytest.mark.parametrize("new", [[100], [100, 40, 70]])
def test_a_layer_of_a_step_waits_for_nothing_and_can_be_captured(new):
    """fp32: the step's lists are made by its first layer."""
    print(f"case: fp32 layer captured {new}", flush=True)
    vb = synth.verify_batch(134, new, new, block_size=16, num_heads=4, num_kv_heads=2, dtype="f32")
    t = to_device(vb)
    layers = [Attention(4, 128, 1.0, 2, 16) for _ in range(2)]
    for layer in layers:
        layer.k_cache, layer.v_cache = t["k_cache"], t["v_cache"]
        layer.key_weights = torch.full((vb.k_cache.shape[0], 2, 16), float("nan"), device="cuda")
    k = v = torch.empty((sum(new), 2, 128), device="cuda")
    set_context(True, cu_seqlens_q=t["cu_seqlens_q"], context_lens=t["context_lens"], block_tables=t["block_tables"],
                seqlens_q=new, seqlens_k=new)
    try:
        want = layers[0](t["query"], k, v)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            out = layers[1](t["query"], k, v)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert torch.equal(out, want)
        weights = layers[1].key_weights.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layers[1](t["query"], k, v)
        for _ in range(3):
            layers[1].key_weights.fill_(3.0)
            out.zero_()
            graph.replay()
            layers[0](t["query"], k, v)  # eager work between the replays
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            at = ~weights.isnan()        # (a prompt of its own: every key of it is set)
            assert torch.equal(layers[1].key_weights[at], weights[at])
            assert (layers[1].key_weights[~at] == 3.0).all()
    finally:
        reset_context()
