"""evict_kvcache where the table that rows go to is the sequence's own, a copy
of it, or one that keeps some of its pages at their places."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import evict_kvcache
from oracle import bounded as ob
from tests.test_evict_gpu import _case

pytestmark = pytest.mark.gpu


def _bits(x):
    return x.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32).numpy()


def _check(case, lens, budget, out_of, want_out=None, sinks=4, recent=20, index=torch.int32):
    """out_of: the device's table -> the output table that the call gets;
    want_out: the oracle's (its own tables: in place)."""
    k, v, w, tables = case[:4]
    lens = np.array(lens, dtype=np.int64)
    want = ob.evict(_bits(k), _bits(v), w.numpy(), tables, lens, budget, sinks, recent, want_out)
    gk, gv, gw = (x.cuda() for x in (k, v, w))
    on_device = torch.from_numpy(tables).cuda().to(index)
    new_lens, kept = evict_kvcache(gk, gv, gw, on_device, torch.from_numpy(lens).cuda(), budget, sinks=sinks, recent=recent,
                                   out_block_tables=out_of(on_device))
    torch.cuda.synchronize()
    assert (kept.cpu().numpy() == want[4]).all(), "kept"
    assert (new_lens.cpu().numpy() == want[3]).all(), "lens"
    for name, got, x in (("k", gk, want[0]), ("v", gv, want[1])):
        assert (_bits(got.cpu()) == x).all(), name
    assert (gw.cpu().numpy().view(np.int32) == want[2].view(np.int32)).all(), "weights"


# few rows; many, which go by way of staging rows in place; beyond what a workgroup holds of the weights
SHAPES = [dict(lens=[700, 150, 20], budget=300, Hkv=2, D=64, block_size=16),
          dict(lens=[9600, 8300], budget=8192, Hkv=2, D=64, block_size=16),
          dict(lens=[40000], budget=9001, Hkv=1, D=32, block_size=64)]


@pytest.mark.parametrize("shape", SHAPES, ids=["short", "staged", "long"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_the_table_itself_is_in_place(shape, index):
    print(f"case: evict to the same table {shape} {index}", flush=True)
    case = _case(121, shape["lens"], shape["Hkv"], shape["D"], shape["block_size"])
    _check(case, shape["lens"], shape["budget"], lambda t: t, index=index)


@pytest.mark.parametrize("shape", SHAPES, ids=["short", "staged", "long"])
@pytest.mark.parametrize("how", ["clone", "narrow"])
def test_copies_of_the_table(shape, how):
    print(f"case: evict to a {how} of the table {shape}", flush=True)
    case = _case(122, shape["lens"], shape["Hkv"], shape["D"], shape["block_size"])
    pages = -(-shape["budget"] // shape["block_size"])
    out = case[3] if how == "clone" else np.ascontiguousarray(case[3][:, :pages])
    _check(case, shape["lens"], shape["budget"], lambda t: t.clone() if how == "clone" else t[:, :pages].clone(), out)


def test_a_narrower_view_of_one_sequence():
    print("case: evict to a view at the table's own address", flush=True)
    case = _case(123, [700], 2, 64, 16)
    _check(case, [700], 300, lambda t: t[:, :19], np.ascontiguousarray(case[3][:, :19]))


@pytest.mark.parametrize("block_size", [1, 16])
def test_some_pages_kept_and_some_new(block_size):
    """Each sequence keeps other pages of its old table at their places: the
    first, the last, every second, none."""
    print(f"case: evict to tables of old and new pages, {block_size}", flush=True)
    lens, budget = [900, 901, 1200, 700], 333
    pages = -(-budget // block_size)
    case = _case(124, lens, 2, 64, block_size, spare=4 * pages)
    out = case[4][:4 * pages].reshape(4, pages).copy()
    out[0, 0] = case[3][0, 0]
    out[1, pages - 1] = case[3][1, pages - 1]
    out[2, ::2] = case[3][2, :pages:2]
    _check(case, lens, budget, lambda t: torch.from_numpy(out).cuda(), out)
