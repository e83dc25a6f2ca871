"""The few-row operators where a sequence's keys go to many workgroups, or one
workgroup turns over several runs of table entries."""

import pytest

from naivllm_amd.utils import synth
from tests.test_bounded_attention_gpu import _check_weights, _check_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens", [[8200], [7001, 60]])
@pytest.mark.parametrize("H,Hkv,D,rows", [(4, 1, 64, 9), (8, 1, 128, 1),   # scores stored
                                          (40, 1, 64, 2), (36, 1, 128, 5)])  # keys read again
def test_many_splits(dtype, lens, H, Hkv, D, rows):
    print(f"case: weights of {lens} keys, {H}/{Hkv} {D} {rows} rows {dtype}", flush=True)
    _check_weights(synth.verify_batch(141, lens, [rows] * len(lens), num_heads=H, num_kv_heads=Hkv, head_dim=D, dtype=dtype,
                                      block_size=64))


def test_many_splits_with_unmapped_pages():
    print("case: weights of 8200 keys, holes", flush=True)
    for H, rows in ((4, 9), (40, 2)):
        vb = synth.verify_batch(142, [8200], [rows], num_heads=H, num_kv_heads=1, head_dim=64, block_size=16,
                                pad_rows=[1])
        vb.block_tables[0, [0, 3, 77] + list(range(200, 260))] = -1  # (whole splits among them)
        _check_weights(vb)


# 500 pairs on 512 places: a sequence's keys are not split, nor in more than two where they are read again
def _one_token_pages(dtype, rows):
    vb = synth.verify_batch(143, [6000] + [rows] * 249, [rows] * 250, num_heads=2, num_kv_heads=2, head_dim=64, dtype=dtype,
                            block_size=1)
    vb.block_tables[0, [5, 2100, 5900]] = -1
    return vb


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 6])  # scores stored; too many of them: keys read again
def test_more_pages_than_a_workgroup_stages(dtype, rows):
    print(f"case: weights, one-token pages, {rows} rows {dtype}", flush=True)
    _check_weights(_one_token_pages(dtype, rows))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(5000, 64), (5900, 0), (3000, 2500)])
def test_a_window_of_more_pages_than_a_workgroup_stages(dtype, window, sinks):
    print(f"case: window {window} sinks {sinks}, one-token pages {dtype}", flush=True)
    _check_window(_one_token_pages(dtype, 3), window, sinks)
