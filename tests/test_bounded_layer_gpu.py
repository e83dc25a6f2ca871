"""The Attention layer over a bounded cache, driven step by step as a runner
drives it (set_context, then the layer): with a window, and with key weights
and an eviction between steps, against 64-bit attention over the very keys
that each step may see."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import Attention, evict_kvcache
from naivllm_amd.utils import synth
from naivllm_amd.utils.context import reset_context, set_context
from oracle import bounded as ob
from tests.bounded_util import check_attention, weight_error

pytestmark = pytest.mark.gpu


class Sequences:
    """Sequences over one pool of pages, and the layer that serves them."""

    def __init__(self, seed, dtype, H=4, Hkv=2, D=64, block_size=16, pages=(30, 30), weights=False, **kw):
        self.dtype, self.H, self.Hkv, self.D, self.bs, self.seed = dtype, H, Hkv, D, block_size, seed
        torch_dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
        perm = synth.randperm(seed, 1, sum(pages) + 2).astype(np.int32)
        self.tables = np.full((len(pages), max(pages)), -1, dtype=np.int32)
        at = 0
        for b, p in enumerate(pages):
            self.tables[b, :p] = perm[at:at + p]
            at += p
        self.lens = [0] * len(pages)  # keys in the cache
        self.layer = Attention(H, D, 1.0, Hkv, block_size, **kw)
        nan = float("nan")  # (what no step has written)
        self.layer.k_cache, self.layer.v_cache = (
            torch.full((sum(pages) + 2, block_size, Hkv, D), nan, dtype=torch_dtype, device="cuda") for _ in range(2))
        if weights:
            self.layer.key_weights = torch.full((sum(pages) + 2, Hkv, block_size), nan, device="cuda")
        self.k, self.v = (np.zeros((sum(pages) + 2, block_size, Hkv, D)) for _ in range(2))
        self.w = np.zeros((sum(pages) + 2, Hkv, block_size))
        self.turn = 0

    def step(self, counts, kind, window=None, sinks=0, paged=True):
        """counts[b] new rows of each sequence; checks the layer's result."""
        self.turn += 1
        T = sum(counts)
        draw = lambda i, h: synth.round_to(synth.normal(self.seed, 100 * self.turn + i, T * h * self.D), self.dtype).reshape(T, h, self.D)  # noqa: E731
        q, k, v = draw(1, self.H), draw(2, self.Hkv), draw(3, self.Hkv)
        first = list(self.lens)
        ends = [n + c for n, c in zip(self.lens, counts)]
        pos = np.concatenate([np.arange(n, e) for n, e in zip(first, ends)]).astype(np.int64)
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        seq = np.repeat(np.arange(len(counts)), counts)
        slots = self.tables[seq, pos // self.bs].astype(np.int64) * self.bs + pos % self.bs
        self.k.reshape(-1, self.Hkv, self.D)[slots], self.v.reshape(-1, self.Hkv, self.D)[slots] = k, v
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        f = lambda x: dev(x.astype(np.float32)).to(self.layer.k_cache.dtype)  # noqa: E731
        kw = dict(cu_seqlens_q=dev(cu), slot_mapping=dev(slots), context_lens=dev(np.array(ends)),
                  block_tables=dev(self.tables) if paged else None, seqlens_q=list(counts), seqlens_k=ends)
        set_context(kind == "prefill", is_verify=kind == "verify", positions=dev(pos), **kw)
        try:
            out = self.layer(f(q), f(k), f(v)).view(T, self.H, self.D)
        finally:
            reset_context()
        torch.cuda.synchronize()
        want, want_abs, mag, sums = ob.attention(q, self.k, self.v, self.tables, np.array(ends), cu, pos,
                                                 1.0 / np.sqrt(self.D), self.Hkv, window, sinks)
        check_attention(out, want, want_abs, mag, self.dtype, max(ends), f"{kind} step {self.turn}")
        self.lens = ends
        if self.layer.key_weights is not None:
            self.w = ob.add_weights(self.w, sums, self.tables, first)
            got = self.layer.key_weights.cpu().numpy()
            for b, n in enumerate(ends):
                at = self.tables[b, np.arange(n) // self.bs], slice(None), np.arange(n) % self.bs
                # (one call's weights are off by at most this share, as are sums of several calls')
                share = weight_error(mag.max(), max(ends), self.D) + (2 * T * self.H + self.turn) * 2.0 ** -24
                assert (np.abs(got[at] - self.w[at]) <= share * self.w[at] + 1e-30).all(), f"weights, step {self.turn}"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (4, 1, 128)])
def test_a_request_under_a_window(dtype, H, Hkv, D):
    print(f"case: layer with a window {dtype} {H}/{Hkv}", flush=True)
    s = Sequences(81, dtype, H, Hkv, D, window=50, sinks=4)
    w = dict(window=50, sinks=4)
    s.step([130, 40], "prefill", paged=False, **w)  # the step's own keys
    s.step([1, 1], "decode", **w)
    s.step([100, 3], "prefill", **w)                # a chunk behind cached keys
    s.step([5, 2], "verify", **w)
    s.step([7, 9], "prefill", **w)                  # a few rows behind cached keys
    for _ in range(3):
        s.step([1, 1], "decode", **w)


def test_pages_behind_the_window_may_go():
    print("case: layer with a window, pages given back", flush=True)
    s = Sequences(82, "bf16", window=40, sinks=16)
    s.step([200, 180], "prefill", window=40, sinks=16)
    for b, n in enumerate(s.lens):
        gone = slice(1, (n + 1 - 40) // 16)         # (the next row's window starts at n + 1 - 40)
        for page in s.tables[b, gone]:
            s.layer.k_cache[int(page)] = s.layer.v_cache[int(page)] = float("nan")
        s.tables[b, gone] = -1
    s.step([1, 1], "decode", window=40, sinks=16)
    s.step([4, 3], "verify", window=40, sinks=16)
    s.step([60, 55], "prefill", window=40, sinks=16)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("apart", [False, True])
def test_a_request_with_evictions(dtype, apart):
    """Prefill, decode and verify steps keep score, evictions cut the caches,
    and later steps attend to what stayed."""
    print(f"case: layer with key weights {dtype} apart {apart}", flush=True)
    s = Sequences(83, dtype, pages=(30, 30, 30), weights=True)
    s.step([210, 50, 3], "prefill")
    for _ in range(2):
        s.step([1, 1, 1], "decode")
    s.step([3, 5, 2], "verify")
    for budget, sinks, recent in ((64, 4, 16), (40, 0, 8)):
        tables = torch.from_numpy(s.tables).cuda()
        out, to = None, s.tables
        if apart:
            # each sequence's last pages, which it does not use
            to = np.full((3, 8), -1, dtype=np.int32)
            to[:, :5] = s.tables[:, 25:30] if budget == 64 else s.tables[:, 20:25]
            out = torch.from_numpy(to).cuda()
        layer = s.layer
        # (the table's own values, which differ from the oracle's by roundings: an eviction goes by them)
        before = layer.key_weights.cpu().numpy().copy()
        lens, kept = evict_kvcache(layer.k_cache, layer.v_cache, layer.key_weights, tables,
                                   torch.tensor(s.lens, device="cuda"), budget, sinks=sinks, recent=recent,
                                   out_block_tables=out)
        s.k, s.v, _, want_lens, want_kept = ob.evict(s.k, s.v, before, s.tables, np.array(s.lens), budget, sinks, recent,
                                                     to if apart else None)
        assert (kept.cpu().numpy() == want_kept).all() and (lens.cpu().numpy() == want_lens).all()
        # the oracle's weights move with the rows
        w = s.w.copy()
        for b, n in enumerate(want_lens):
            for h in range(s.Hkv):
                j, i = want_kept[b, h, :n], np.arange(n)
                w[to[b, i // s.bs], h, i % s.bs] = s.w[s.tables[b, j // s.bs], h, j % s.bs]
        s.w, s.lens = w, [int(n) for n in want_lens]
        if apart:
            rest = [[p for p in row if p not in to[b]] for b, row in enumerate(s.tables.tolist())]
            s.tables = np.array([[p for p in to[b].tolist() if p >= 0] + rest[b] for b in range(3)], dtype=np.int32)
        s.step([1, 1, 1], "decode")
        s.step([2, 4, 3], "verify")
        s.step([30, 1, 8], "prefill")


def test_refusals_of_the_layer():
    s = Sequences(84, "bf16", weights=True)
    with pytest.raises(ValueError, match="block_tables"):
        s.step([20, 20], "prefill", paged=False)
    s = Sequences(84, "bf16", weights=True, window=8)
    with pytest.raises(ValueError, match="not both"):
        s.step([20, 20], "prefill")
    with pytest.raises(ValueError, match="window"):
        Attention(4, 64, window=-1)
    with pytest.raises(ValueError, match="sinks"):
        Attention(4, 64, window=4, sinks=1.5)
