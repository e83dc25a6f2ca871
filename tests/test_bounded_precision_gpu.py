"""The few-row operators' outputs are off by their weights' own fp32 error and
one final rounding."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import paged_attention_weights, paged_attention_window
from naivllm_amd.utils import synth
from oracle import bounded as ob
from tests.bounded_util import EPS32, HALF, weight_error
from tests.gpu_util import to_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hkv,D,rows", [(16, 8, 128, 1), (32, 8, 128, 9), (8, 1, 64, 5), (8, 8, 64, 40)])
@pytest.mark.parametrize("weighed", [False, True])
def test_outputs_are_rounded_once(H, Hkv, D, rows, weighed):
    print(f"case: precision {H}/{Hkv} {D} {rows} rows, weights {weighed}", flush=True)
    vb = synth.verify_batch(111, [900, 333], [rows] * 2, num_heads=H, num_kv_heads=Hkv, head_dim=D, block_size=64)
    t = to_device(vb)
    meta = (t["block_tables"], t["context_lens"], t["cu_seqlens_q"], t["positions"], 1 / np.sqrt(D), H, Hkv, D, 64, 64)
    if weighed:
        w = torch.zeros((vb.k_cache.shape[0], Hkv, 64), device="cuda")
        out = paged_attention_weights(t["query"], t["k_cache"], t["v_cache"], w, *meta, max_q_len=rows)
    else:
        out = paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *meta, window=2000, max_q_len=rows)
    want, want_abs, mag, _ = ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens,
                                          vb.cu_seqlens_q, vb.positions, 1 / np.sqrt(D), Hkv)
    got = out.float().cpu().numpy().astype(np.float64)
    # a weight held as two bf16 numbers is off by half a step of half a step; the product adds up to `keys` terms
    inner = (weight_error(mag, 900, D)[..., None] + HALF["bf16"] ** 2 + 900 * EPS32) * want_abs
    bound = inner * (1 + HALF["bf16"]) + HALF["bf16"] * np.abs(want) + 1e-30
    err = np.abs(got - want)
    assert (err <= bound).all(), f"{(err > bound).sum()} of {err.size} outside, worst by {(err / bound).max():.2f}"

