"""Refused arguments of the page operators (CPU: nothing is launched)."""

import ctypes

import pytest
import torch

from naivllm_amd import _lib
from naivllm_amd.layers.pages import CachePages, _Pool

ARG, UNSUPPORTED, WORKSPACE = -1, -2, -3


def _pools(base=0x1000, segments=1, key_bytes=256):
    return (_Pool * 1)(_Pool(base, segments, key_bytes))


def _fork(pools=None, n=1, nb=10, bs=16, tables=0x1000, lens=0x2000, parents=0x3000, B=2, W=3, out=0x4000, out_lens=0x5000,
          lacking=0x6000, ws=0x7000, size=1 << 20):
    pools = _pools() if pools is None else pools
    return _lib.lib().nsv_fork_pages(ctypes.addressof(pools), n, nb, bs, tables, lens, parents, None, B, W, out, out_lens,
                                     lacking, ws, size, None)


def _compact(pools=None, n=1, nb=10, bs=16, tables=0x1000, B=2, W=3, out=0x4000, ids=0x5000, top=0x6000, ws=0x7000,
             size=1 << 20):
    pools = _pools() if pools is None else pools
    return _lib.lib().nsv_compact_pages(ctypes.addressof(pools), n, nb, bs, tables, None, B, W, out, ids, top, ws, size, None)


def _copy(pools=None, n=1, nb=10, bs=16, src=0x1000, dst=0x2000, moves=3):
    pools = _pools() if pools is None else pools
    return _lib.lib().nsv_copy_pages(ctypes.addressof(pools), n, nb, bs, src, dst, None, moves, None)


@pytest.mark.parametrize("call", [_fork, _compact, _copy])
def test_pools(call):
    for bad in (dict(base=0), dict(base=0x1001), dict(segments=0), dict(key_bytes=0), dict(key_bytes=3), dict(key_bytes=-2)):
        assert call(pools=_pools(**bad)) == ARG, bad
    assert call(n=-1) == call(nb=0) == call(bs=0) == ARG
    assert call(nb=(1 << 18) + 1) == call(pools=_pools(key_bytes=1 << 28)) == UNSUPPORTED


def test_fork():
    for bad in (dict(tables=None), dict(lens=None), dict(parents=None), dict(out=None), dict(out_lens=None), dict(lacking=None),
                dict(B=-1), dict(W=0), dict(out=0x1000), dict(out=0x1014), dict(out_lens=0x2008)):
        assert _fork(**bad) == ARG, bad
    assert _fork(B=4097) == _fork(B=2048, W=1 << 20, out=1 << 40) == UNSUPPORTED
    need = _lib.lib().nsv_fork_pages_workspace_size(2, 3, 10)
    assert need > 0 and _fork(size=need - 1) == _fork(ws=None) == _fork(ws=0x7008) == WORKSPACE
    assert _lib.lib().nsv_fork_pages_workspace_size(4097, 3, 10) == 0


def test_compact():
    for bad in (dict(tables=None), dict(out=None), dict(ids=None), dict(top=None), dict(B=-1), dict(W=0), dict(out=0x1004)):
        assert _compact(**bad) == ARG, bad
    need = _lib.lib().nsv_compact_pages_workspace_size(10)
    assert need > 0 and _compact(size=need - 1) == _compact(ws=None) == _compact(ws=0x7008) == WORKSPACE
    assert _lib.lib().nsv_compact_pages_workspace_size(1 << 20) == 0


def test_copy():
    assert _copy(src=None) == _copy(dst=None) == _copy(moves=-1) == ARG
    assert _copy(moves=0) == 0


def test_pools_on_the_cpu_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        CachePages([torch.zeros(4, 2, 1, 8)])


def test_fork_of_an_empty_batch_says_what_it_needs():
    size = _lib.lib().nsv_fork_pages_workspace_size
    need = size(0, 3, 10)
    assert need > 0 and size(-1, 3, 10) == size(0, 0, 10) == size(0, 3, 0) == 0
    assert _fork(B=0, size=need - 1) == _fork(B=0, ws=None) == WORKSPACE
