"""paged_attention_window and paged_attention_weights against the oracle."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import paged_attention_weights, paged_attention_window
from naivllm_amd.utils import synth
from oracle import bounded as ob
from tests.bounded_util import EPS32, as_device, check_attention, weight_error
from tests.gpu_util import to_device

pytestmark = pytest.mark.gpu


def _args(vb, t):
    return (t["block_tables"], t["context_lens"], t["cu_seqlens_q"], t["positions"], 1.0 / np.sqrt(vb.head_dim),
            vb.num_heads, vb.num_kv_heads, vb.head_dim, vb.block_size, 64)


def _oracle(vb, window=None, sinks=0):
    return ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q, vb.positions,
                        1.0 / np.sqrt(vb.head_dim), vb.num_kv_heads, window, sinks)


def _window(vb, window, sinks, **kw):
    t = to_device(vb)
    out = paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *_args(vb, t), window=window, sinks=sinks,
                                 max_q_len=vb.max_q_len, **kw)
    torch.cuda.synchronize()
    return out


def _check_window(vb, window, sinks):
    want, want_abs, mag, _ = _oracle(vb, window, sinks)
    out = _window(vb, window, sinks)
    check_attention(out, want, want_abs, mag, vb.dtype, window + sinks + 1, f"window {window} sinks {sinks}")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 100, 129, 600, 5000])
@pytest.mark.parametrize("sinks", [0, 1, 4, 40])
def test_window_sizes(dtype, window, sinks):
    print(f"case: window {window} sinks {sinks} {dtype}", flush=True)
    _check_window(synth.verify_batch(31, [700, 33, 1, 257], [5, 1, 1, 9], dtype=dtype, block_size=64), window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D", [(16, 8, 128), (32, 8, 128), (8, 8, 64), (8, 1, 64), (12, 4, 128), (40, 1, 128)])
@pytest.mark.parametrize("rows", [1, 3, 9])
def test_window_head_layouts(dtype, H, Hkv, D, rows):
    print(f"case: heads {H}/{Hkv} dim {D} rows {rows} {dtype}", flush=True)
    vb = synth.verify_batch(32, [500, 77], [rows, rows], num_heads=H, num_kv_heads=Hkv, head_dim=D, dtype=dtype,
                            block_size=16)
    _check_window(vb, 100, 3)


@pytest.mark.parametrize("block_size", [1, 2, 16, 256, 1024])
def test_window_page_sizes(block_size):
    print(f"case: page {block_size}", flush=True)
    vb = synth.verify_batch(33, [2300, 40], [4, 4], dtype="bf16", block_size=block_size, num_kv_heads=2, num_heads=4)
    _check_window(vb, 777, 5)
    _check_window(vb, 4000, 5)


def test_window_one_token_pages_beyond_the_staged_table():
    # one pair in one-token pages: more table entries per workgroup than its LDS holds
    print("case: 3000 one-token pages, 300 pairs", flush=True)
    vb = synth.verify_batch(34, [3000] + [5] * 299, [1] * 300, dtype="f32", block_size=1, num_heads=2, num_kv_heads=2,
                            head_dim=64)
    _check_window(vb, 2900, 64)


def test_window_long_context_reads_only_what_is_seen():
    """Pages between the sinks and the windows hold NaN, or are unmapped:
    nothing of them reaches a result."""
    print("case: NaN between sinks and window", flush=True)
    vb = synth.verify_batch(35, [1500, 900], [4, 2], dtype="bf16", block_size=32)
    want, want_abs, mag, _ = _oracle(vb, 200, 7)
    t = to_device(vb)
    for b, (n, rows) in enumerate(((1500, 4), (900, 2))):
        for j in range(7, n - rows - 200 + 1):  # no row sees these
            page = int(vb.block_tables[b, j // 32])
            t["k_cache"][page, j % 32] = float("nan")
            t["v_cache"][page, j % 32] = float("nan")
        for j in range(n, -(-n // 32) * 32):    # nor those past the context
            page = int(vb.block_tables[b, j // 32])
            t["k_cache"][page, j % 32] = float("nan")
            t["v_cache"][page, j % 32] = float("inf")
    t["block_tables"][0, 10:30] = -1
    out = paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *_args(vb, t), window=200, sinks=7,
                                 max_q_len=4)
    check_attention(out, want, want_abs, mag, "bf16", 208, "NaN outside")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_window_unmapped_pages_and_rows_that_see_nothing(dtype):
    print(f"case: holes {dtype}", flush=True)
    vb = synth.verify_batch(36, [600, 300, 64, 10], [5, 9, 3, 2], dtype=dtype, block_size=16, pad_rows=[1, 0, 3, 0])
    vb.block_tables[0, [0, 35, 36]] = -1
    vb.block_tables[1, :] = -1          # no page at all
    vb.block_tables[3, 0] = -1
    for window, sinks in ((40, 4), (1, 0), (1000, 0)):
        _check_window(vb, window, sinks)
    out = _window(vb, 40, 4)
    assert not out[5:14].any() and not out[14:17].any() and not out[4].any()


def test_window_positions_apart_and_contexts_short_of_them():
    """Rows in any order of positions, and a context that ends before them."""
    print("case: scattered positions", flush=True)
    vb = synth.verify_batch(37, [900, 500], [4, 3], dtype="f32", block_size=32)
    vb.positions[:4] = [20, 890, 3, 400]
    vb.context_lens[1] = 450  # the rows' own keys are not there
    _check_window(vb, 64, 2)
    vb.context_lens[1] = 0
    _check_window(vb, 64, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_sequences_without_rows(dtype):
    print(f"case: sequences without rows {dtype}", flush=True)
    vb = synth.verify_batch(40, [300, 50, 77, 10], [3, 0, 2, 0], dtype=dtype, block_size=16)
    _check_window(vb, 40, 4)
    _check_weights(vb)


def test_scales_of_every_sign():
    print("case: scales", flush=True)
    vb = synth.verify_batch(44, [300], [3], dtype="f32", block_size=16)
    t = to_device(vb)
    for scale in (0.0, -0.09, 2.0):
        want, want_abs, mag, _ = ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens,
                                              vb.cu_seqlens_q, vb.positions, scale, vb.num_kv_heads, 50, 2)
        meta = _args(vb, t)
        out = paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *meta[:4], scale, *meta[5:], window=50,
                                     sinks=2, max_q_len=3)
        check_attention(out, want, want_abs, np.abs(mag), "f32", 60, f"scale {scale}")


def test_window_rows_behind_the_last_sequence_stay():
    vb = synth.verify_batch(38, [100], [3], dtype="bf16", block_size=16)
    t = to_device(vb)
    query = torch.cat([t["query"], t["query"]])
    out = torch.full_like(query, 7.0)
    positions = torch.cat([t["positions"], t["positions"]])
    paged_attention_window(query, t["k_cache"], t["v_cache"], t["block_tables"], t["context_lens"], t["cu_seqlens_q"],
                           positions, 0.1, 16, 8, 128, 16, 16, window=30, max_q_len=3, out=out)
    assert (out[3:] == 7.0).all() and not (out[:3] == 7.0).all()


def test_window_takes_strided_and_unaligned_queries():
    vb = synth.verify_batch(39, [300], [4], dtype="bf16", block_size=16)
    t = to_device(vb)
    want = _window(vb, 50, 2)
    wide = torch.zeros((4, 16, 256), dtype=torch.bfloat16, device="cuda")
    wide[..., :128] = t["query"]
    odd = torch.zeros(4 * 16 * 128 + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = t["query"].flatten()
    for q in (wide[..., :128], odd[1:].view(4, 16, 128)):
        out = paged_attention_window(q, t["k_cache"], t["v_cache"], *_args(vb, t), window=50, sinks=2, max_q_len=4)
        assert torch.equal(out, want)


# ---------------------------------------------------------------------------
# key weights
# ---------------------------------------------------------------------------


def _check_weights(vb, seed=5):
    want, want_abs, mag, sums = _oracle(vb)
    t = to_device(vb)
    nb, bs = vb.k_cache.shape[:2]
    old = synth.normal(seed, 3, nb * vb.num_kv_heads * bs).reshape(nb, vb.num_kv_heads, bs).astype(np.float32) ** 2
    weights = as_device(old)
    out = paged_attention_weights(t["query"], t["k_cache"], t["v_cache"], weights, *_args(vb, t),
                                  max_q_len=vb.max_q_len)
    torch.cuda.synchronize()
    keys = int(max(vb.context_lens))
    check_attention(out, want, want_abs, mag, vb.dtype, keys, "out")
    first, spans = [], {}
    for b in range(len(vb.context_lens)):
        pos = vb.positions[vb.cu_seqlens_q[b]:vb.cu_seqlens_q[b + 1]]
        live = pos[pos >= 0]
        first.append(int(live.min()) if live.size else 0)
        # (only the keys up to the last row get a weight)
        spans[b] = sums[b][:, :int(live.max()) + 1] if live.size else sums[b][:, :0]
    new = ob.add_weights(old, spans, vb.block_tables, first)
    rel = weight_error(mag.max(), keys, vb.head_dim)
    rows = vb.max_q_len * vb.num_heads // vb.num_kv_heads
    got = weights.cpu().numpy().astype(np.float64)
    # a sum of rows weights, each rel off, with as many additions; then the addition to the old value
    bound = (rel + (rows + 1) * EPS32) * np.abs(new) + EPS32 * np.abs(new) + 1e-30
    assert (np.abs(got - new) <= bound).all(), f"weights: worst by {(np.abs(got - new) / bound).max():.2f}"
    touched = new != old
    assert (got[~touched] == old[~touched]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D", [(16, 8, 128), (32, 8, 128), (8, 8, 64), (8, 1, 64), (12, 4, 128), (40, 1, 64)])
@pytest.mark.parametrize("rows", [1, 2, 9])
def test_weights_head_layouts(dtype, H, Hkv, D, rows):
    print(f"case: weights heads {H}/{Hkv} dim {D} rows {rows} {dtype}", flush=True)
    _check_weights(synth.verify_batch(41, [300, 77, rows], [rows] * 3, num_heads=H, num_kv_heads=Hkv, head_dim=D,
                                      dtype=dtype, block_size=16))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("block_size", [1, 32, 256])
def test_weights_lengths_holes_and_padding(dtype, block_size):
    print(f"case: weights page {block_size} {dtype}", flush=True)
    vb = synth.verify_batch(42, [1, 33, 1100, 64, 5], [1, 3, 3, 2, 3], dtype=dtype, block_size=block_size,
                            pad_rows=[0, 1, 0, 2, 0])
    vb.block_tables[2, 1] = -1
    _check_weights(vb)
    vb.block_tables[1, :] = -1
    vb.context_lens[4] = 0
    _check_weights(vb)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,rows,H,Hkv,D", [([60, 41, 9], 9, 40, 1, 64), ([64, 30], 33, 4, 2, 64),
                                              ([1100] * 30 + [900, 33], 9, 32, 8, 128)])
def test_weights_of_whole_sequences_and_keys_read_again(dtype, lens, rows, H, Hkv, D):
    """No split to join and too many scores to store: by the rows of a kv
    head, or by the call's."""
    print(f"case: weights unsplit, {len(lens)} sequences {rows} rows {H}/{Hkv} {dtype}", flush=True)
    _check_weights(synth.verify_batch(43, lens, [rows] * len(lens) if rows <= 9 else [rows, 30], num_heads=H,
                                      num_kv_heads=Hkv, head_dim=D, dtype=dtype, block_size=16))


def test_weights_rows_behind_the_last_sequence_and_other_places_stay():
    vb = synth.verify_batch(43, [100], [3], dtype="bf16", block_size=16)
    vb.context_lens[0] = 500  # a table wider than the rows reach: keys past the last row keep their place's value
    _check_weights(vb)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,H", [(2, 16), (9, 32)])
def test_a_row_of_nan_stays_alone(dtype, rows, H):
    """A NaN query row: NaN for itself and for the weights of the keys it
    sees, nothing for other rows, heads and keys; in a padding row, nothing."""
    print(f"case: a NaN row {dtype} {rows} {H}", flush=True)
    vb = synth.verify_batch(45, [700, 300], [rows, rows], num_heads=H, dtype=dtype, block_size=16, pad_rows=[1, 0])
    t = to_device(vb)
    want = paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *_args(vb, t), window=200, sinks=4, max_q_len=rows)
    w_want = torch.rand((vb.k_cache.shape[0], 8, 16), device="cuda")
    w = w_want.clone()
    every = paged_attention_weights(t["query"], t["k_cache"], t["v_cache"], w_want, *_args(vb, t), max_q_len=rows)
    t["query"][rows - 1] = float("nan")        # padding
    t["query"][rows, 5 * H // 16] = float("nan")    # the second sequence's first row, one head
    out = paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *_args(vb, t), window=200, sinks=4, max_q_len=rows)
    out_w = paged_attention_weights(t["query"], t["k_cache"], t["v_cache"], w, *_args(vb, t), max_q_len=rows)
    for got, good in ((out, want), (out_w, every)):
        assert got[rows, 5 * H // 16].isnan().all()
        good[rows, 5 * H // 16] = 0
        got[rows, 5 * H // 16] = 0
        assert torch.equal(got, good)
    head = 5 * H // 16 // (H // 8)
    seen = 300 - rows + 1                      # keys that the row sees
    for b, n in enumerate((700 - (1 if rows > 1 else 0), 300)):
        j = np.arange(n)
        at = (torch.from_numpy(vb.block_tables[b, j // 16]).long().cuda(), slice(None), torch.from_numpy(j % 16).cuda())
        got, good = w[at], w_want[at]
        if b == 1:
            assert got[:seen, head].isnan().all()
            got[:seen, head] = good[:seen, head] = 0
        assert torch.equal(got, good)
