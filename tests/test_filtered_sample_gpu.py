"""sample_filtered against the oracle."""

import threading

import numpy as np
import pytest
import torch

from naivllm_amd.spec_engine.rejection_sampler import sample_filtered
from oracle.filtered import Row
from tests.filtered_util import logits, on_gpu, settings, sum_error

pytestmark = pytest.mark.gpu


def _check(x, f, u, got=None, kept=None, **call):
    """x [B, V] (CPU), f numpy settings, u numpy."""
    B, V = x.shape
    if got is None:
        kept = torch.full((B,), -7, dtype=torch.int32, device="cuda")
        got = sample_filtered(x.cuda(), uniforms=torch.from_numpy(u).cuda(), kept=kept, **on_gpu(f), **call)
    torch.cuda.synchronize()
    got, kept, x = got.tolist(), kept.tolist(), x.double().numpy()
    same = 0
    for b in range(B):
        row = Row(x[b], *(f[k][b] if k in f else d for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0),
                                                              ("min_p", 0.0))))
        why = row.admits(kept[b], got[b], min(max(float(u[b]), 0.0), 1.0) if u[b] == u[b] else 0.0, sum_error(V))
        assert why is None, f"row {b}: {why}"
        same += kept[b] == row.n and got[b] == row.sample(u[b] if u[b] == u[b] else 0.0)
    return same


def _uniforms(seed, B):
    return np.random.default_rng(seed).random(B, dtype=np.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 100, 1000, 2049, 8191, 8192, 8193, 50001, 151936])
def test_vocabularies(V, dtype):
    print(f"case: sample_filtered V {V} {dtype}", flush=True)
    for n, shape in enumerate(("flat", "peaked", "levels")):
        same = _check(logits(V + n, 7, V, dtype, shape), settings(V + n, 7), _uniforms(V + n, 7))
        assert same == 7, f"{shape}: {same} of 7"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [163841, 262144, 1 << 20])
def test_large_vocabularies(V, dtype):
    print(f"case: sample_filtered large V {V} {dtype}", flush=True)
    _check(logits(V, 7, V, dtype), settings(V, 7), _uniforms(V, 7))
    x = logits(V + 1, 2, V, dtype, "equal")
    _check(x, dict(temperature=np.ones(2, np.float32), top_p=np.array([0.5, 1.0], np.float32)), _uniforms(5, 2))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("setting", [dict(), dict(top_k=7), dict(top_p=0.7), dict(min_p=0.3), dict(top_k=90, top_p=0.5),
                                     dict(top_k=50, top_p=0.9, min_p=0.01)])
def test_many_draws_of_a_row(dtype, setting):
    """Uniform numbers over the whole range: every kept token is drawn, in order."""
    print(f"case: sample_filtered draws {setting} {dtype}", flush=True)
    B, V = 512, 600
    for shape in ("flat", "levels", "equal"):
        x = logits(17, 1, V, dtype, shape).expand(B, V).contiguous()
        u = np.append(np.linspace(0, 1, B - 1, endpoint=False), 1 - 2.0 ** -24).astype(np.float32)
        f = {k: np.full(B, v, np.int32 if k == "top_k" else np.float32) for k, v in setting.items()}
        assert _check(x, dict(f, temperature=np.full(B, 0.9, np.float32)), u) == B


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cuts_between_close_values(dtype):
    """A lone maximum whose next tokens lie in a range that might have passed;
    more equal and close tokens than are looked at one by one; temperatures at
    which one range of values spans many orders of weight."""
    print(f"case: sample_filtered close values {dtype}", flush=True)
    V = 30000
    x = logits(3, 8, V, dtype)
    x[0] = x[0].clamp_max(8.0)
    x[0, 77] = 8.9
    x[1] = x[1].clamp_max(8.0)
    x[1, [99, 700]] = 8.9
    x[2, ::3] = 5.0                                              # 10,000 equal ones
    x[3] = 5.0 + logits(4, 1, V, "f32")[0].to(x.dtype) * 1e-3    # all within a few of the type's steps, or fp32's
    x[4] = -5.0 - logits(5, 1, V, "f32")[0].abs().to(x.dtype) * 1e-4
    x[5] = logits(6, 1, V, dtype)[0] * 1e-6
    x[6, 5:] = -np.inf
    x[7] = x[7] * 1000
    for n, f in enumerate((dict(), dict(min_p=np.full(8, 0.5)), dict(top_p=np.full(8, 0.4)), dict(top_k=np.full(8, 1000)),
                           dict(top_k=np.full(8, 5000), top_p=np.full(8, 0.9), min_p=np.full(8, 0.02)), dict(top_p=np.full(8, 1e-6)))):
        f = {k: v.astype(np.int32 if k == "top_k" else np.float32) for k, v in f.items()}
        for T in (1.0, 0.02, 30.0):
            _check(x, dict(f, temperature=np.full(8, T, np.float32)), _uniforms(n, 8))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_extreme_settings(dtype):
    print(f"case: sample_filtered extremes {dtype}", flush=True)
    V, nan, inf = 3001, np.nan, np.inf
    rows = []
    for t in (0.0, -1.0, nan, 1e-6, 2e-6, 1e-3, 1.0, 1e4, 1e30, inf):
        rows += [(t, 0, 1.0, 0.0), (t, 5, 0.5, 0.1)]
    for k in (-2 ** 31, -1, 0, 1, 2, V - 1, V, V + 1, 2 ** 31 - 1):
        rows.append((1.0, k, 1.0, 0.0))
    for p in (-1.0, 0.0, 1e-38, 1e-9, 1 - 2.0 ** -24, 1.0, 2.0, inf, nan):
        rows.append((1.0, 0, p, 0.0))
    for m in (-1.0, 0.0, 1e-38, 1e-9, 1 - 2.0 ** -24, 1.0, 2.0, inf, nan):
        rows.append((1.0, 0, 1.0, m))
    f = {k: np.array([r[i] for r in rows], np.int32 if k == "top_k" else np.float32)
         for i, k in enumerate(("temperature", "top_k", "top_p", "min_p"))}
    for shape in ("flat", "equal"):
        for u in (0.0, 0.5, 1 - 2.0 ** -24):
            _check(logits(23, len(rows), V, dtype, shape), f, np.full(len(rows), u, np.float32))
    _check(logits(24, 4, V, dtype), dict(temperature=np.ones(4, np.float32)), np.array([1.0, 7.0, -3.0, nan], np.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [900, 20011, 151936])
def test_masks(V, dtype):
    """Masked tokens of -inf, of the type's lowest value and of a constant, from
    a few of them to all; infinities and NaN."""
    print(f"case: sample_filtered masks V {V} {dtype}", flush=True)
    low = torch.finfo(logits(0, 1, 1, dtype).dtype).min
    rng = np.random.default_rng(V)
    rows = []
    for fill in (-np.inf, low, -1e4, -1.0):
        for share in (0.02, 0.5, 0.99, 1 - 1.5 / V, 1.0):
            x = logits(int(1e3 * share), 1, V, dtype)
            if share == 1.0:
                x.fill_(fill)
            else:
                x[torch.from_numpy(rng.random((1, V)) < share)] = fill
            rows.append(x)
    for value, count in ((np.inf, 1), (np.inf, 5), (-np.inf, 5), (np.nan, 1), (np.nan, 3), (-0.0, V // 2)):
        x = logits(len(rows), 1, V, dtype)
        x[0, torch.from_numpy(rng.choice(V, count, replace=False))] = value
        rows.append(x)
    rows.append(rows[-1].clamp_max(0.0))  # both zeros on top
    half = logits(99, 1, V, dtype)
    half[0, V // 3:] = -np.inf  # a whole stretch
    rows.append(half)
    x = torch.cat(rows)
    for n, f in enumerate((dict(), dict(top_k=np.full(len(x), 40, np.int32)), dict(top_p=np.full(len(x), 0.8, np.float32)),
                           dict(min_p=np.full(len(x), 0.05, np.float32)))):
        _check(x, dict(f, temperature=np.full(len(x), 0.8, np.float32)), _uniforms(n, len(x)))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_values_of_most_tokens(dtype):
    """More than 65,535 tokens of one value: all over the row, in stretches one
    after another, and where no wave's first lane holds it."""
    print(f"case: sample_filtered crowded values {dtype}", flush=True)
    V = 300001
    x = logits(1, 6, V, dtype)
    x[0, :90000] = -1.0
    x[0, 100000:190000] = 1.0
    x[0, 200000:] = -1.0
    x[1, torch.arange(V) % 512 != 0] = 0.5
    x[2, torch.arange(V) % 8 != 0] = 3.0
    x[3, ::2] = -0.0
    x[3, 1::2] = 0.0
    x[4, torch.arange(V) % 3 > 0] = 20.0
    x[5, torch.arange(V) % 512 != 0] = -0.0
    f = dict(temperature=np.full(6, 0.8, np.float32))
    for n, more in enumerate((dict(), dict(top_p=np.full(6, 0.7, np.float32)), dict(top_k=np.full(6, 150000, np.int32)),
                              dict(min_p=np.full(6, 0.01, np.float32)))):
        assert _check(x, dict(f, **more), _uniforms(n, 6)) == 6
        # so many rows that one workgroup does a whole one
        f15 = on_gpu({k: np.tile(v, 15) for k, v in dict(f, **more).items()})
        kept = torch.zeros(90, dtype=torch.int32, device="cuda")
        got = sample_filtered(x.cuda().repeat(15, 1), uniforms=torch.from_numpy(np.tile(_uniforms(n, 6), 15)).cuda(), kept=kept, **f15)
        assert (got.view(15, 6) == got[:6]).all() and (kept.view(15, 6) == kept[:6]).all()
        assert _check(x, dict(f, **more), _uniforms(n, 6), got[:6], kept[:6]) == 6


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 30, 9001])
def test_values_next_to_zero(V, dtype):
    """Maxima among the type's smallest numbers, below zero too, beside either
    zero and beside nothing."""
    print(f"case: sample_filtered next to zero V {V} {dtype}", flush=True)
    least = 2.0 ** -133 if dtype == "bf16" else 2.0 ** -149  # the type's smallest
    few = (-least, -3 * least, -100 * least, least, 5 * least, 0.0, -0.0, -2.0 ** -126, 2.0 ** -126, -1.0)
    rng = np.random.default_rng(V)
    rows = [np.full(V, v) for v in few] + [rng.choice(few[:n], V) for n in range(2, len(few) + 1)]
    rows += [np.where(rng.random(V) < 0.5, -np.inf, r) for r in rows[:8]]
    rows += [np.where(rng.random(V) < 0.9, -5.0, r) for r in rows[:8]]
    x = torch.tensor(np.stack(rows)).float().to(logits(0, 1, 1, dtype).dtype)
    for n, f in enumerate((dict(), dict(top_k=np.full(len(x), 3, np.int32)), dict(top_p=np.full(len(x), 0.6, np.float32)))):
        for T in (0.0, 0.9):
            assert _check(x, dict(f, temperature=np.full(len(x), T, np.float32)), _uniforms(n, len(x))) == len(x)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,V", [(33, 16384), (65, 20011), (129, 20011), (1100, 1201), (300, 70001)])
def test_many_rows(B, V, dtype):
    """Rows in one part and in several, of one launch and of several."""
    print(f"case: sample_filtered {B} rows of {V} {dtype}", flush=True)
    for shape in ("peaked", "levels"):
        assert _check(logits(B, B, V, dtype, shape), settings(B, B), _uniforms(B, B)) == B


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V,pitch,offset", [(1000, 1001, 0), (1000, 1003, 3), (4096, 4096, 1), (8190, 8197, 5), (24593, 30000, 7)])
def test_pitches_and_outputs(V, pitch, offset, dtype):
    """Rows off 16-byte boundaries; a strided column of drafts; neighbours untouched."""
    print(f"case: sample_filtered pitch {V} {pitch} {offset} {dtype}", flush=True)
    B = 5
    x, f, u = logits(V, B, V, dtype, "peaked"), settings(V, B), _uniforms(V, B)
    buf = torch.full((offset + B * pitch,), 1e4, dtype=x.dtype, device="cuda")
    view = buf[offset:].as_strided((B, V), (pitch, 1))
    view.copy_(x)
    out = torch.full((B, 3), -5, dtype=torch.int32, device="cuda")
    kept = torch.zeros(B, dtype=torch.int32, device="cuda")
    got = sample_filtered(view, uniforms=torch.from_numpy(u).cuda(), out=out[:, 1], kept=kept, **on_gpu(f))
    assert got.data_ptr() == out[:, 1].data_ptr()
    assert _check(x, f, u, got, kept) == B
    assert (out[:, 0] == -5).all() and (out[:, 2] == -5).all()


def test_numbers_for_every_row_and_empty_batch():
    print("case: sample_filtered numbers", flush=True)
    x, u = logits(3, 4, 500, "f32"), _uniforms(3, 4)
    kept = torch.zeros(4, dtype=torch.int32, device="cuda")
    got = sample_filtered(x.cuda(), 0.7, torch.from_numpy(u).cuda(), top_k=20, top_p=0.9, min_p=0.01, kept=kept)
    f = dict(temperature=np.full(4, 0.7, np.float32), top_k=np.full(4, 20), top_p=np.full(4, 0.9, np.float32),
             min_p=np.full(4, 0.01, np.float32))
    assert _check(x, f, u, got, kept) == 4
    assert sample_filtered(x[:0].cuda(), 1.0, torch.zeros(0, device="cuda")).shape == (0,)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_and_on_another_stream(dtype):
    """A captured call reads the buffers as they are at each replay, beside
    eager calls of the same buffers' kind on another stream."""
    print(f"case: sample_filtered captured {dtype}", flush=True)
    B, V = 6, 20001
    x = logits(0, B, V, dtype).cuda()
    f, u = on_gpu(settings(0, B)), torch.zeros(B, device="cuda")
    out, kept = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    sample_filtered(x, uniforms=u, out=out, kept=kept, **f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_filtered(x, uniforms=u, out=out, kept=kept, **f)
    side = torch.cuda.Stream()
    for n in range(4):
        new, nf, nu = logits(30 + n, B, V, dtype, "peaked"), settings(30 + n, B), _uniforms(30 + n, B)
        x.copy_(new)
        u.copy_(torch.from_numpy(nu))
        for name, t in on_gpu(nf).items():
            f[name].copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            k2 = torch.zeros(B, dtype=torch.int32, device="cuda")
            o2 = sample_filtered(x, uniforms=u, kept=k2, **f)
        torch.cuda.synchronize()
        assert _check(new, nf, nu, out, kept) == B
        assert torch.equal(o2, out) and torch.equal(k2, kept)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_behind_32_bits(dtype):
    """Rows whose first element is the 2^31-th and later of their storage."""
    print(f"case: sample_filtered rows behind 32 bits {dtype}", flush=True)
    B, V, pitch = 3, 5003, 2 ** 30 + 2 ** 28 + 7
    x, f, u = logits(7, B, V, dtype), settings(7, B), _uniforms(7, B)
    view = torch.empty((B - 1) * pitch + V, dtype=x.dtype, device="cuda").as_strided((B, V), (pitch, 1))
    view.copy_(x)
    kept = torch.zeros(B, dtype=torch.int32, device="cuda")
    got = sample_filtered(view, uniforms=torch.from_numpy(u).cuda(), kept=kept, **on_gpu(f))
    assert _check(x, f, u, got, kept) == B


def test_two_threads_on_a_stream():
    """Calls of two threads on one stream, which share its scratch."""
    print("case: sample_filtered from two threads", flush=True)
    jobs = []
    for n, (B, V, dtype) in enumerate(((9, 20001, "bf16"), (5, 30001, "f32"))):
        x, f, u = logits(n, B, V, dtype), settings(n, B), _uniforms(n, B)
        kept = [torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(40)]
        jobs.append((x, f, u, x.cuda(), torch.from_numpy(u).cuda(), on_gpu(f), kept, []))
    torch.cuda.synchronize()

    def run(job):
        for kept in job[6]:
            job[7].append(sample_filtered(job[3], uniforms=job[4], kept=kept, **job[5]))

    threads = [threading.Thread(target=run, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for x, f, u, _, _, _, kept, got in jobs:
        assert len(got) == 40
        for k, g in zip(kept, got):
            assert torch.equal(g, got[0]) and torch.equal(k, kept[0])
        assert _check(x, f, u, got[0], kept[0]) == len(x)
