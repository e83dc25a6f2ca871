"""The bounded cache's operators captured, replayed, on several streams at
once, and over pages that sequences share."""

import threading
import time

import numpy as np
import pytest
import torch

from naivllm_amd import _lib
from naivllm_amd.layers.attention import (KeyWeightsPlan, PrefillPlan, evict_kvcache, paged_attention_weights,
                                          paged_attention_window, prefill_attention, prefill_key_weights)
from naivllm_amd.utils import synth
from oracle import bounded as ob
from tests.bounded_util import weight_error
from tests.gpu_util import to_device

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _few(seed, lens=(900, 333, 70), rows=5, dtype="bf16", **kw):
    vb = synth.verify_batch(seed, list(lens), [rows] * len(lens), dtype=dtype, block_size=16, **kw)
    t = to_device(vb)
    meta = (t["block_tables"], t["context_lens"], t["cu_seqlens_q"], t["positions"], 1.0 / np.sqrt(vb.head_dim),
            vb.num_heads, vb.num_kv_heads, vb.head_dim, vb.block_size, 64)
    weights = torch.rand((vb.k_cache.shape[0], vb.num_kv_heads, 16), device="cuda")
    return vb, t, meta, weights


def _calls(seed):
    """name -> a function of fresh state: (state tensors, a step that works on them and returns its results)."""
    vb, t, meta, weights = _few(seed, rows=9)
    _, tp, mp, wp = _few(seed + 1, (900, 333, 400), 200)
    new, ends = [200] * 3, [900, 333, 400]
    plan = PrefillPlan(new, ends, 16, 8, 16, DEV, window=150, sinks=4)
    whole, adder = PrefillPlan(new, ends, 16, 8, 16, DEV), KeyWeightsPlan(new, ends, 16, 8, 16, DEV)

    def window():
        return [], lambda: [paged_attention_window(t["query"], t["k_cache"], t["v_cache"], *meta, window=100, sinks=4,
                                                   max_q_len=9)]

    def key_weights():
        w = weights.clone()
        return [w], lambda: [paged_attention_weights(t["query"], t["k_cache"], t["v_cache"], w, *meta, max_q_len=9)]

    def prompt():
        return [], lambda: [prefill_attention(tp["query"], tp["k_cache"], tp["v_cache"], plan, 0.09, 128, mp[0])]

    def prompt_weights():
        w, stats = wp.clone(), torch.empty((600, 16, 2), device="cuda")

        def step():
            out = prefill_attention(tp["query"], tp["k_cache"], tp["v_cache"], whole, 0.09, 128, mp[0], stats=stats)
            prefill_key_weights(tp["query"], tp["k_cache"], w, adder, stats, 0.09, 128, mp[0])
            return [out]
        return [w, stats], step

    def evict():
        k, v, w = t["k_cache"].clone(), t["v_cache"].clone(), weights.clone()
        return [k, v, w], lambda: list(evict_kvcache(k, v, w, meta[0], meta[1], 128, sinks=4, recent=30))

    return dict(window=window, key_weights=key_weights, prompt=prompt, prompt_weights=prompt_weights, evict=evict)


@pytest.mark.parametrize("name", ["window", "key_weights", "prompt", "prompt_weights", "evict"])
def test_captured_and_replayed(name):
    print(f"case: captured {name}", flush=True)
    make = _calls(91)[name]
    want_state, want_step = make()
    state, step = make()
    step()                                   # (a first call outside the capture)
    start = [x.clone() for x in make()[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for x, y in zip(state, start):
        x.copy_(y)
    for turn in range(4):
        graph.replay()
        want = want_step()                   # eager work between the replays
        torch.cuda.synchronize()
        for got, w in zip(results + state, want + want_state):
            assert torch.equal(got, w), (name, turn)


@pytest.mark.parametrize("name", ["window", "key_weights", "prompt_weights", "evict"])
def test_two_graphs_at_once(name):
    print(f"case: two graphs {name}", flush=True)
    makes = [_calls(92)[name], _calls(95)[name]]
    runs = []
    for make in makes:
        want_state, want_step = make()
        want = want_step()
        state, step = make()
        step()
        start = [x.clone() for x in make()[0]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step()
        runs.append((graph, state, start, results, want + want_state, torch.cuda.Stream()))
    for _ in range(3):
        for graph, state, start, _, _, stream in runs:
            for x, y in zip(state, start):
                x.copy_(y)
        torch.cuda.synchronize()
        for graph, *_, stream in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, state, _, results, want, _ in runs:
            for got, w in zip(results + state, want):
                assert torch.equal(got, w), name


def test_two_streams_at_once():
    print("case: two streams", flush=True)
    calls = [_calls(93), _calls(94)]
    for name in ("window", "key_weights", "prompt", "prompt_weights", "evict"):
        wants = []
        for c in calls:
            state, step = c[name]()
            wants.append(step() + state)
        torch.cuda.synchronize()
        made = [c[name]() for c in calls]
        streams = [torch.cuda.Stream() for _ in calls]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        results = []
        for (state, step), s in zip(made, streams):
            with torch.cuda.stream(s):
                results.append(step() + state)
        torch.cuda.synchronize()
        for got, want in zip(results, wants):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), name


@pytest.mark.parametrize("name,native", [("window", "nsv_window_attention"), ("key_weights", "nsv_weights_attention")])
def test_two_threads_on_one_stream(name, native, monkeypatch):
    """A call's launches, which share the stream's scratch, stay together: the
    second thread's begin when the first's are all enqueued."""
    print(f"case: two threads {name}", flush=True)
    calls = [_calls(101)[name], _calls(104)[name]]
    wants = []
    for make in calls:
        state, step = make()
        wants.append(step() + state)
    torch.cuda.synchronize()
    real, inside, most = _lib.lib(), [], []

    class Watched:
        def __getattr__(self, attr):
            call = getattr(real, attr)
            if attr != native:
                return call

            def watched(*args):
                inside.append(1)
                most.append(len(inside))
                time.sleep(0.02)
                rc = call(*args)
                inside.pop()
                return rc
            return watched

    monkeypatch.setattr(_lib, "lib", lambda: Watched())
    made, results, start = [make() for make in calls], [None, None], threading.Barrier(2)
    torch.cuda.synchronize()

    def work(i):
        start.wait()
        for _ in range(3):
            got = made[i][1]()
            if results[i] is None:
                results[i] = [x.clone() for x in got + made[i][0]]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join(60)
    torch.cuda.synchronize()
    assert len(most) == 6 and max(most) == 1
    for got, want in zip(results, wants):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_shared_page_gets_the_weights_of_every_sequence():
    """Two sequences behind one cached prefix: its keys' places take both
    sums, from the few-row operator (stored scores and, with many rows, keys
    read again) and from the prompts' one."""
    for rows, H in ((1, 16), (9, 32), (60, 16)):
        print(f"case: shared pages, {rows} rows", flush=True)
        vb = synth.verify_batch(96, [700, 650], [rows] * 2, num_heads=H, block_size=16)
        vb.block_tables[1, :30] = vb.block_tables[0, :30]
        t = to_device(vb)
        scale = 1.0 / np.sqrt(128)
        _, _, mag, sums = ob.attention(vb.q, vb.k_cache, vb.v_cache, vb.block_tables, vb.context_lens, vb.cu_seqlens_q,
                                       vb.positions, scale, 8)
        old = np.abs(synth.normal(9, 3, vb.k_cache.shape[0] * 8 * 16)).reshape(-1, 8, 16).astype(np.float32)
        w = torch.from_numpy(old).cuda()
        if rows <= 9:
            paged_attention_weights(t["query"], t["k_cache"], t["v_cache"], w, t["block_tables"], t["context_lens"],
                                    t["cu_seqlens_q"], t["positions"], scale, H, 8, 128, 16, 16, max_q_len=rows)
        else:
            plan = PrefillPlan([rows] * 2, [700, 650], H, 8, 16, DEV)
            stats = torch.empty((2 * rows, H, 2), device="cuda")
            prefill_attention(t["query"], t["k_cache"], t["v_cache"], plan, scale, 128, t["block_tables"], stats=stats)
            prefill_key_weights(t["query"], t["k_cache"], w, KeyWeightsPlan([rows] * 2, [700, 650], H, 8, 16, DEV), stats,
                                scale, 128, t["block_tables"])
        want = ob.add_weights(old, sums, vb.block_tables, [700 - rows, 650 - rows])  # (one after the other)
        share = weight_error(mag.max(), 700, 128) + (rows * H // 8 + 4) * 2.0 ** -24
        got = w.cpu().numpy()
        assert (np.abs(got - want) <= share * want + 1e-30).all(), rows


def test_a_plan_made_on_another_stream():
    print("case: plans of another stream", flush=True)
    _, t, meta, w = _few(97, (900, 333, 400), 200)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        plan, adder = (PrefillPlan([200] * 3, [900, 333, 400], 16, 8, 16, DEV),
                       KeyWeightsPlan([200] * 3, [900, 333, 400], 16, 8, 16, DEV))
    stats = torch.empty((600, 16, 2), device="cuda")
    a, b = w.clone(), w.clone()
    prefill_attention(t["query"], t["k_cache"], t["v_cache"], plan, 0.09, 128, meta[0], stats=stats)
    prefill_key_weights(t["query"], t["k_cache"], a, adder, stats, 0.09, 128, meta[0])
    torch.cuda.synchronize()
    prefill_key_weights(t["query"], t["k_cache"], b, adder, stats, 0.09, 128, meta[0])
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    """Arguments that are refused before anything is launched."""
    vb, t, meta, w = _few(98)
    q, k, v = t["query"], t["k_cache"], t["v_cache"]

    def window(*m, query=q, kc=k, vc=v, **kw):
        kw.setdefault("window", 10)
        return paged_attention_window(query, kc, vc, *(m or meta), **kw)

    def refused(match, f, *a, **kw):
        with pytest.raises(ValueError, match=match):
            f(*a, **kw)

    refused("query must be", window, query=q[:, :4])
    refused("share one dtype", window, query=q.float())
    refused("same contiguous shape", window, vc=v[:-1])
    refused("contiguous", window, kc=k.transpose(0, 1))
    refused("entries", window, *meta[:3], meta[3][:-1], *meta[4:])
    refused("entries", window, meta[0], meta[1][:-1], *meta[2:])
    refused("on cpu", window, meta[0].cpu(), *meta[1:])
    refused("out must be", window, out=torch.empty_like(q, dtype=torch.float32))
    refused("overlap", window, out=q)
    refused("overlap", paged_attention_weights, q, k, v, w, *meta, out=q)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    refused("16 bytes", window, out=odd)
    refused("unsupported", window, max_q_len=65)
    refused("unsupported dtype", window, query=q.half(), kc=k.half(), vc=v.half())
    refused("key_weights must be", paged_attention_weights, q, k, v, w.double(), *meta)
    refused("key_weights must be", paged_attention_weights, q, k, v, w[:, :4], *meta)
    tables, lens = meta[0], meta[1]
    refused("exceed the budget", evict_kvcache, k, v, w, tables, lens, 8, sinks=5, recent=4)
    refused("budget", evict_kvcache, k, v, w, tables, lens, 0)
    refused("do not hold", evict_kvcache, k, v, w, tables, lens, 40, out_block_tables=tables[:, :2])
    refused("entries", evict_kvcache, k, v, w, tables, lens[:1], 8)
    refused("key_weights", evict_kvcache, k, v, w[:-1], tables, lens, 8)
    plan = PrefillPlan([5] * 3, [900, 333, 70], 16, 8, 16, DEV, window=4)
    stats = torch.empty((15, 16, 2), device="cuda")
    refused("without a window", prefill_attention, q, k, v, plan, 0.1, 128, tables, stats=stats)
    whole = PrefillPlan([5] * 3, [900, 333, 70], 16, 8, 16, DEV)
    refused("stats must be", prefill_attention, q, k, v, whole, 0.1, 128, tables, stats=stats[:-1])
    adder = KeyWeightsPlan([5] * 3, [900, 333, 70], 16, 8, 16, DEV)
    refused("stats must be", prefill_key_weights, q, k, w, adder, stats.double(), 0.1, 128, tables)
    refused("pages for sequences", prefill_key_weights, q, k, w, adder, stats, 0.1, 128, tables[:, :4].contiguous())
    refused("bfloat16", prefill_key_weights, q.float(), k, w, adder, stats, 0.1, 128, tables)
    refused("at least", prefill_key_weights, q[:3], k, w, adder, stats, 0.1, 128, tables)
    refused("window", PrefillPlan, [5], [5], 16, 8, 16, DEV, window=-1)


def test_batches_of_nothing():
    _, t, _, w = _few(99)
    empty = dict(dtype=torch.int32, device="cuda")
    meta = (torch.empty((0, 3), **empty), torch.empty(0, dtype=torch.int64, device="cuda"), torch.zeros(1, **empty),
            torch.empty(0, dtype=torch.int64, device="cuda"), 0.1, 16, 8, 128, 16, 16)
    q, before = t["query"][:0], w.clone()
    assert paged_attention_window(q, t["k_cache"], t["v_cache"], *meta, window=4).shape == (0, 16, 128)
    assert paged_attention_weights(q, t["k_cache"], t["v_cache"], w, *meta).shape == (0, 16, 128)
    lens, kept = evict_kvcache(t["k_cache"], t["v_cache"], w, meta[0], meta[1], 8)
    assert lens.shape == (0,) and kept.shape == (0, 8, 8) and torch.equal(w, before)
