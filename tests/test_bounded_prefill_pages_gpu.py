"""Prompts over tables of more pages than a workgroup holds at a time."""

import pytest
import torch

from naivllm_amd.layers.attention import _prefill_work
from tests.test_bounded_prefill_gpu import _batch, _check, _check_key_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,prefix,H,Hkv,windows,waves", [
    ([70] * 40, [4000] + [5] * 39, 8, 8, [(3700, 200), (2500, 0)], 4),
    ([1100] * 4, [2200] * 4, 16, 8, [(2600, 300)], 8)])
def test_windows_over_one_token_pages(new, prefix, H, Hkv, windows, waves):
    vb = _batch(151, new, prefix, H, Hkv, 64, 1)
    vb.block_tables[0, [0, 199, 400, 1900, 2300, 3100]] = -1
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for window, sinks in windows:
        print(f"case: {len(new)} prompts, one-token pages, window {window} sinks {sinks}", flush=True)
        work, (n, merges, rows, _) = _prefill_work(new, vb.context_lens.tolist(), H, Hkv, 1, cus, window, sinks, False)
        tiles = work[:8 * n].view(n, 8)
        assert merges == 0 and rows * (2 if H // Hkv % 2 == 0 else 1) == 32 * waves
        assert int((tiles[:, 6] - tiles[:, 5]).max()) > 2048
        _check(vb, window, sinks)


def test_key_weights_over_one_token_pages():
    print("case: prompt weights, one-token pages", flush=True)
    vb = _batch(152, [70] * 40, [4000] + [5] * 39, 8, 8, 64, 1)
    vb.block_tables[0, [3, 2500, 4010]] = -1
    _check_key_weights(vb)
