"""CachePages against the oracle, bit for bit."""

import numpy as np
import pytest
import torch

from naivllm_amd import _lib
from naivllm_amd.layers.pages import CachePages
from oracle import pages as op

pytestmark = pytest.mark.gpu


def _pools(nb, bs, heads=2, dim=64, dtype=torch.bfloat16, layers=2, weights=True, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kv = [torch.randn((nb, bs, heads, dim), device="cuda", generator=gen).to(dtype) for _ in range(2 * layers)]
    kw = [torch.rand((nb, heads, bs), device="cuda", generator=gen) for _ in range(layers if weights else 0)]
    return kv, kw


def _moved(kv, kw, moves, bs):
    """The pools after the moves (src, dst, keys)."""
    kv, kw = [t.clone() for t in kv], [t.clone() for t in kw]
    for src, dst, *keys in moves:
        n = max(0, min(bs, keys[0])) if keys else bs
        for t in kv:
            t[dst, :n] = t[src, :n]
        for t in kw:
            t[dst, :, :n] = t[src, :, :n]
    return kv + kw


def _same(got, want):
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _held(nb, ids):
    h = torch.zeros(nb, dtype=torch.bool, device="cuda")
    h[list(ids)] = True
    return h


def _check_fork(tables, lens, parents, nb, bs, held=(), pools=None, **kw):
    kv, weights = pools or _pools(nb, bs, **kw)
    want = op.fork(tables, lens, parents, nb, bs, held)
    after = _moved(kv, weights, want[3], bs)
    before = _i32(tables)
    new, new_lens, lacking = CachePages(kv, weights).fork(before, torch.tensor(lens, device="cuda"), _i32(parents),
                                                          held=_held(nb, held) if held else None)
    torch.cuda.synchronize()
    assert new.tolist() == want[0] and new_lens.tolist() == want[1] and lacking.item() == want[2]
    assert before.tolist() == tables
    _same(kv + weights, after)


def _check_compact(tables, nb, bs, held=(), in_place=False, **kw):
    kv, weights = _pools(nb, bs, **kw)
    want = op.compact(tables, nb, held)
    after = _moved(kv, weights, want[3], bs)
    t = _i32(tables)
    new, ids, top = CachePages(kv, weights).compact(t, held=_held(nb, held) if held else None,
                                                    out_tables=t if in_place else None)
    torch.cuda.synchronize()
    assert new.tolist() == want[0] and ids.tolist() == want[1] and top.item() == want[2]
    _same(kv + weights, after)


def _beams(rng, B, W, bs, nb, holes=False):
    """Tables whose rows share some leading pages, as a fork leaves them."""
    ids = rng.permutation(nb).tolist()
    lens = [int(rng.integers(0, W * bs + 1)) for _ in range(B)]
    tables = []
    for b in range(B):
        row = [ids.pop() for _ in range(min(W, lens[b] // bs + int(rng.integers(0, 3))))] if len(ids) > W else []
        if b and rng.random() < 0.5:
            n = min(lens[b] // bs, lens[b - 1] // bs, len(row))
            row[:n] = tables[b - 1][:n]
        tables.append(row + [-1] * (W - len(row)))
    if holes:  # pages behind a window, and ids outside the pool
        for row in tables:
            for j in range(W):
                if rng.random() < 0.1:
                    row[j] = int(rng.choice([-1, nb, -7, 2 ** 31 - 1]))
    return tables, lens


@pytest.mark.parametrize("bs", [1, 2, 16, 256])
@pytest.mark.parametrize("B", [1, 2, 5, 17, 70])
def test_fork(B, bs):
    print(f"case: fork {B} rows page {bs}", flush=True)
    for n in range(4):
        rng = np.random.default_rng(100 * B + n)
        W = [1, 3, 65, 130][n] if bs < 256 and B < 70 else 1 + n
        nb = B * W + 3 * B + 7
        tables, lens = _beams(rng, B, W, bs, nb - 2 * B, holes=n == 3)
        parents = [int(rng.integers(-1, B)) for _ in range(B)] if n else [0] * B
        used = {e for row in tables for e in row}
        held = [i for i in range(nb) if i not in used][:2 + n]
        _check_fork(tables, lens, parents, nb, bs, held, layers=1, dim=32 if bs == 256 else 64)


@pytest.mark.parametrize("dtype,heads,dim,bs", [(torch.float32, 1, 64, 16), (torch.bfloat16, 3, 40, 4), (torch.bfloat16, 1, 1, 3),
                                                (torch.bfloat16, 1, 2, 16), (torch.float32, 5, 7, 8), (torch.bfloat16, 8, 128, 64)])
def test_layouts(dtype, heads, dim, bs):
    """Rows and pages off 16 bytes, down to 2 bytes per key."""
    print(f"case: pages {dtype} {heads} {dim} {bs}", flush=True)
    rng = np.random.default_rng(bs)
    tables, lens = _beams(rng, 6, 9, bs, 60)
    _check_fork(tables, lens, [0, 0, 0, 3, 3, 1], 90, bs, heads=heads, dim=dim, dtype=dtype)
    _check_compact(tables, 90, bs, [3, 80], heads=heads, dim=dim, dtype=dtype)


def test_fork_without_enough_pages():
    print("case: fork short of pages", flush=True)
    tables = [[0, 1, 2, -1], [3, 4, 5, -1], [-1] * 4, [-1] * 4]
    lens = [17, 20, 0, 0]
    for nb in (6, 7, 8, 9, 12):
        for parents in ([0, 1, 0, 1], [0, 0, 0, 0], [1, 1, 0, -1], [1, 0, 1, 0]):
            _check_fork(tables, lens, parents, nb, 8)
            _check_fork(tables, lens, parents, nb, 8, held=[1, nb - 1])


def test_fork_odd_rows():
    """Parents out of range, lengths below zero and past the table, an empty batch."""
    print("case: fork odd rows", flush=True)
    tables = [[4, 9, 2], [7, -1, 1], [-1, -1, -1], [5, 6, 8]]
    _check_fork(tables, [-5, 24, 3, 10 ** 12], [3, 0, 0, 3], 30, 8)
    _check_fork(tables, [24, 5, 0, 23], [9, -3, 2 ** 31 - 1, -2 ** 31], 30, 8)
    kv, kw = _pools(4, 4)
    new, lens, lacking = CachePages(kv, kw).fork(_i32([]).reshape(0, 3), torch.zeros(0, dtype=torch.int64, device="cuda"), _i32([]))
    assert new.shape == (0, 3) and lens.shape == (0,) and lacking.item() == 0


def test_many_rows_and_pages():
    print("case: fork 4096 rows", flush=True)
    B, nb = 4096, 20000
    tables = [[3 * b, 3 * b + 1] for b in range(B)]
    lens = [5 + b % 4 for b in range(B)]
    parents = [b // 2 for b in range(B)]
    pools = _pools(nb, 4, heads=1, dim=8, layers=1)
    _check_fork(tables, lens, parents, nb, 4, held=range(15000, 15007), pools=pools)
    print("case: compact 262144 pages", flush=True)
    nb = 1 << 18
    rng = np.random.default_rng(3)
    ids = rng.choice(nb, 30000, replace=False).tolist()
    _check_compact([ids[i:i + 100] for i in range(0, 30000, 100)], nb, 1, held=ids[:50] + [nb - 1], heads=1, dim=8, layers=1)


@pytest.mark.parametrize("bs", [1, 16, 64])
@pytest.mark.parametrize("full", [0.0, 0.1, 0.5, 0.9, 1.0])
def test_compact(full, bs):
    print(f"case: compact {full} page {bs}", flush=True)
    for n, nb in enumerate((1, 2, 31, 32, 33, 64, 200, 2100 if bs == 1 else 300)):
        rng = np.random.default_rng(nb)
        ids = rng.permutation(nb)[:int(full * nb)].tolist()
        held = rng.choice(nb, nb // 10, replace=False).tolist()
        rows = [ids[i:i + 7] + [-1] * (7 - len(ids[i:i + 7])) for i in range(0, max(1, len(ids)), 7)]
        rows.append(rows[0][::-1])  # a page of two rows
        rows.append([nb, -5, 2 ** 31 - 1, -1, nb + 3, -2, -1])
        _check_compact(rows, nb, bs, held, in_place=n % 2 == 0, layers=1)


def test_more_pools_than_one_launch_takes():
    print("case: pages of 150 pools", flush=True)
    tables, lens = [[9, 3, 7], [1, -1, -1]], [5, 2]
    _check_fork(tables, lens, [0, 0], 20, 2, layers=50)
    _check_compact(tables, 20, 2, layers=50)


def test_copy():
    print("case: copy pages", flush=True)
    kv, kw = _pools(40, 16)
    pairs = [(1, 2, 16), (1, 3, 5), (4, 5, 0), (6, 7, -3), (8, 9, 99), (10, 10, 16), (-1, 11, 16), (12, 40, 16), (39, 0, 1)]
    src, dst, keys = map(_i32, zip(*pairs))
    after = _moved(kv, kw, [p for p in pairs if 0 <= p[0] < 40 and 0 <= p[1] < 40], 16)
    pages = CachePages(kv, kw)
    pages.copy(src, dst, keys)
    torch.cuda.synchronize()
    _same(kv + kw, after)
    after = _moved(kv, kw, [(20, 21), (20, 22), (23, 24)], 16)
    pages.copy(_i32([20, 20, 23]), _i32([21, 22, 24]))
    pages.copy(_i32([]), _i32([]))
    torch.cuda.synchronize()
    _same(kv + kw, after)


def test_a_beam_search_by_replays():
    """Two buffers of tables in turn, captured; each replay forks the last one's
    rows and writes a key of its own; in the end every row holds its history."""
    print("case: fork replayed", flush=True)
    B, W, bs, nb, steps = 6, 8, 4, 60, 9
    cache = torch.zeros((nb, bs, 1, 8), device="cuda")
    pages = CachePages([cache])
    tables = [torch.full((B, W), -1, dtype=torch.int32, device="cuda") for _ in range(2)]
    lens = [torch.zeros(B, dtype=torch.int64, device="cuda") for _ in range(2)]
    tables[0].copy_(torch.arange(B * W, device="cuda").reshape(B, W))
    parents, step = _i32([0] * B), torch.zeros((), device="cuda")
    rows = torch.arange(B, device="cuda")
    short = torch.zeros((), dtype=torch.int32, device="cuda")

    def body(i):
        _, _, lacking = pages.fork(tables[i], lens[i], parents, out_tables=tables[1 - i], out_lens=lens[1 - i])
        short.add_(lacking)
        at = lens[1 - i]
        page = tables[1 - i].gather(1, (at // bs)[:, None])[:, 0].long()
        cache[page, at % bs, 0] = (100 * step + rows)[:, None].expand(B, 8)
        at.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        keep = [t.clone() for t in tables + lens + [cache]]
        body(0)
        body(1)
        for t, k in zip(tables + lens + [cache], keep):
            t.copy_(k)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            body(i)
        graphs.append(g)
    rng = np.random.default_rng(8)
    history = [[] for _ in range(B)]
    for n in range(steps):
        choice = rng.integers(0, B, B).tolist() if n else list(range(B))
        parents.copy_(_i32(choice))
        step.fill_(n)
        graphs[n % 2].replay()
        history = [history[p] + [100.0 * n + b] for b, p in enumerate(choice)]
        torch.cuda.synchronize()
        t, m = tables[1 - n % 2], lens[1 - n % 2].tolist()
        assert m == [n + 1] * B
        for b in range(B):
            assert [cache[int(t[b, j // bs]), j % bs, 0, 0].item() for j in range(m[b])] == history[b], (n, b)
    assert short.item() == 0


@pytest.mark.parametrize("bad", [
    lambda p, t, n, r: p.fork(t.long(), n, r), lambda p, t, n, r: p.fork(t[0], n, r), lambda p, t, n, r: p.fork(t[:, :0], n, r),
    lambda p, t, n, r: p.fork(t, n.int(), r), lambda p, t, n, r: p.fork(t, n[:1], r), lambda p, t, n, r: p.fork(t, n, r.long()),
    lambda p, t, n, r: p.fork(t, n, r[:1]), lambda p, t, n, r: p.fork(t, n, r, held=torch.zeros(9, device="cuda").bool()),
    lambda p, t, n, r: p.fork(t, n, r, held=_i32([0] * 10)), lambda p, t, n, r: p.fork(t, n, r, out_tables=t),
    lambda p, t, n, r: p.fork(t, n, r, out_lens=n), lambda p, t, n, r: p.fork(t, n, r, out_tables=t[:, :2]),
    lambda p, t, n, r: p.fork(t.cpu(), n, r), lambda p, t, n, r: p.fork(_i32([[0]] * 4097), torch.zeros(4097, device="cuda").long(), _i32([0] * 4097)),
    lambda p, t, n, r: p.compact(t.float()), lambda p, t, n, r: p.compact(t, out_tables=_i32([[0] * 3] * 4).t()),
    lambda p, t, n, r: p.compact(t, held=torch.zeros(10)), lambda p, t, n, r: p.copy(r, r[:1]), lambda p, t, n, r: p.copy(n, n),
    lambda p, t, n, r: p.copy(r, r, n), lambda p, t, n, r: p.copy(t, t)])
def test_refusals(bad):
    p = CachePages(*_pools(10, 4))
    with pytest.raises(ValueError):
        bad(p, _i32([[0, 1, 2], [3, 4, 5]]), torch.tensor([3, 4], device="cuda"), _i32([0, 0]))


def test_refused_pools():
    kv, kw = _pools(10, 4)
    for bad in (lambda: CachePages([]), lambda: CachePages([kv[0], kv[0]]), lambda: CachePages([kv[0], kv[1][:9]]),
                lambda: CachePages([kv[0][:, :, :, ::2]]), lambda: CachePages([kv[0].half()]), lambda: CachePages([kv[0].flatten(2)]),
                lambda: CachePages(kv, [kw[0][:5]]), lambda: CachePages(kv, [kw[0].double()]), lambda: CachePages(kv, [kw[0].transpose(1, 2)]),
                lambda: CachePages([kv[0].cpu()]), lambda: CachePages([kv[0][:0]])):
        with pytest.raises(ValueError):
            bad()


def test_pages_behind_32_bits():
    print("case: pages past 4 GiB of a pool", flush=True)
    nb, bs = 70000, 16
    kv = [torch.empty((nb, bs, 8, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2)]  # 64 KiB a page
    pages = CachePages(kv)
    marks = [69999, 69000, 66000]
    for n, t in enumerate(kv):
        for page in marks:
            t[page] = torch.randn(t.shape[1:], device="cuda").bfloat16() + n
    was = [[t[page].clone() for page in marks] for t in kv]
    tables, lens, lacking = pages.fork(_i32([[69999, 69000], [-1, -1]]), torch.tensor([20, 0], device="cuda"), _i32([0, 0]),
                                       held=_held(nb, range(68000)))
    assert tables.tolist() == [[69999, 69000], [69999, 68000]] and lens.tolist() == [20, 20] and lacking.item() == 0
    for t, w in zip(kv, was):
        assert torch.equal(t[68000, :4], w[1][:4])
    pages.copy(_i32([66000]), _i32([67000]))
    tables, _, top = pages.compact(_i32([[69999, 69000, 67000]]), held=_held(nb, range(65999)))
    assert tables.tolist() == [[65999, 66000, 66001]] and top.item() == 66002
    for t, w in zip(kv, was):
        for page, content in zip((65999, 66000, 66001), w):
            assert torch.equal(t[page], content)


def test_empty_batches_of_the_library():
    """The entries themselves, by the workspace sizes that they name: nothing is
    short, nothing but held pages is in use."""
    print("case: pages of empty batches, library entries", flush=True)
    kv, kw = _pools(6, 4)
    before = [t.clone() for t in kv + kw]
    pages = CachePages(kv, kw)  # (holds the array of pools)
    h, shape, stream = _lib.lib(), pages._shape, torch.cuda.current_stream().cuda_stream
    lacking, top, ids, held = _i32(7), _i32(7), _i32([7] * 6), _held(6, [1, 4])
    need = h.nsv_fork_pages_workspace_size(0, 3, 6)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    assert h.nsv_fork_pages(*shape, None, None, None, held.data_ptr(), 0, 3, None, None, lacking.data_ptr(), ws.data_ptr(), need,
                            stream) == 0
    need = h.nsv_compact_pages_workspace_size(6)
    ws2 = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert h.nsv_compact_pages(*shape, None, held.data_ptr(), 0, 3, None, ids.data_ptr(), top.data_ptr(), ws2.data_ptr(), need,
                               stream) == 0
    torch.cuda.synchronize()
    assert lacking.item() == 0 and top.item() == 5 and ids.tolist() == [-1, 1, -1, -1, 4, -1]
    _same(kv + kw, before)


def test_pools_that_overlap_are_refused():
    """Views of one allocation are pools of their own only where they are apart."""
    print("case: pools that overlap", flush=True)
    kv = torch.zeros((2, 12, 4, 1, 8), device="cuda")
    kw = torch.zeros((13, 2, 4), device="cuda")
    CachePages([kv[0], kv[1]], [kw[:12]])
    CachePages([kv[1, 6:], kv[0, :6], kv[0, 6:], kv[1, :6]], [kw[:6], kw[7:]])
    for caches, weights in (([kv[0, :8], kv[0, 4:]], []), ([kv[0, 1:9], kv[1, :8], kv[0, :8]], []), ([kv[0, :6]], [kw[:6], kw[5:11]]),
                            ([kv[0]], [kv[0, :6].view(12, 4, 4)])):
        with pytest.raises(ValueError):
            CachePages(caches, weights)
