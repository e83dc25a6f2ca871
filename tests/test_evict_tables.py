"""Which tables of an eviction are one and the same: nothing here launches a
kernel."""

import pytest
import torch

from naivllm_amd import _lib
from naivllm_amd.layers.attention import _evict_tables


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_the_table_itself_is_in_place(index):
    tables = torch.arange(12, dtype=index).view(2, 6)
    assert _evict_tables(tables, None)[1] is None
    got, out = _evict_tables(tables, tables)
    assert out is None and got.dtype == torch.int32 and torch.equal(got.long(), tables.long())
    strided = torch.arange(24, dtype=index).view(2, 12)[:, ::2]
    assert _evict_tables(strided, strided)[1] is None


def test_another_view_of_the_table():
    tables = torch.arange(12, dtype=torch.int32).view(2, 6)
    assert _evict_tables(tables, tables[:])[1] is None           # the same memory, the same shape
    assert _evict_tables(tables, tables.clone())[1] is not None
    one = tables[:1]
    got, out = _evict_tables(one, one[:, :4])                    # the same address, fewer pages
    assert out is not None and out.shape == (1, 4) and out.data_ptr() == got.data_ptr()


def test_the_library_takes_the_same_address_as_in_place():
    h = _lib.lib()

    def evict(out, ws=None, size=0):
        return h.nsv_evict_kv(16, 16, 16, 16, 16, out, 16, 16, 1, 2, 64, 16, 600, 600, 1, 8192, 0, 0, ws, size, None)

    need = h.nsv_evict_workspace_size(1, 2, 64, 16, 600, 0, 1, 8192)
    assert need > 0
    for out in (None, 16):  # (16: block_tables' own address)
        assert evict(out) == evict(out, 16, need - 1) == -3
