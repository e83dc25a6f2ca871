"""Refused arguments of filtered sampling and acceptance (CPU: nothing is launched)."""

import ctypes

import pytest
import torch

from naivllm_amd import _lib
from naivllm_amd.spec_engine.rejection_sampler import accept_filtered, sample_filtered

P = ctypes.c_void_p(0x1000)  # any address: refused calls touch nothing
ARG, UNSUPPORTED, WORKSPACE = -1, -2, -3


def _sample(logits=P, pitch=100, temperature=P, uniforms=P, B=2, V=100, dtype=1, out=P, stride=1,
            ws=P, ws_bytes=1 << 30):
    return _lib.lib().nsv_sample_filtered(logits, pitch, temperature, None, None, None, uniforms, B, V, dtype, out, stride,
                                          None, ws, ws_bytes, None)


def _accept(target=P, t_stride=4, draft=P, d_seq=3, d_row=1, mode=None, drafts=P, live=P, temperature=P, uniforms=P, B=2,
            K=3, V=100, dtype=1, out=P, out_len=P, ws=P, ws_bytes=1 << 30):
    return _lib.lib().nsv_accept_filtered(target, t_stride, draft, d_seq, d_row, mode, drafts, live, temperature, None, None,
                                          None, uniforms, B, K, V, dtype, out, out_len, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(temperature=None), dict(uniforms=None), dict(out=None), dict(B=-1),
                                 dict(V=0), dict(V=-5), dict(dtype=2), dict(pitch=99), dict(stride=0)])
def test_sample_arguments(bad):
    assert _sample(**bad) == ARG


def test_sample_shapes():
    assert _sample(V=(1 << 20) + 1, pitch=1 << 21) == UNSUPPORTED
    assert _sample(B=65536) == UNSUPPORTED
    assert _sample(B=0) == 0
    size = _lib.lib().nsv_sample_filtered_workspace_size
    need = size(2, 151936, 1)
    assert need > 0 and size(2, (1 << 20) + 1, 1) == size(-1, 100, 1) == 0
    assert _sample(V=151936, pitch=151936, ws=None) == _sample(V=151936, pitch=151936, ws_bytes=need - 1) == WORKSPACE


@pytest.mark.parametrize("bad", [dict(target=None), dict(drafts=None), dict(live=None), dict(temperature=None),
                                 dict(uniforms=None), dict(out=None), dict(out_len=None), dict(B=-1), dict(K=-1), dict(K=64),
                                 dict(V=0), dict(dtype=3), dict(t_stride=3), dict(d_row=0), dict(d_seq=-1),
                                 dict(draft=None, mode=P)])
def test_accept_arguments(bad):
    assert _accept(**bad) == ARG


def test_accept_shapes_and_workspace():
    h = _lib.lib()
    assert _accept(V=(1 << 20) + 1) == UNSUPPORTED and _accept(B=65536) == UNSUPPORTED
    assert _accept(B=0) == 0
    need = h.nsv_accept_filtered_workspace_size(2, 3, 100, 1)
    assert need > 0 and _accept(ws_bytes=need - 1) == WORKSPACE and _accept(ws=None) == WORKSPACE
    assert h.nsv_accept_filtered_workspace_size(2, 64, 100, 1) == 0 and h.nsv_accept_filtered_workspace_size(-1, 3, 100, 1) == 0


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(2, 10)
    with pytest.raises(ValueError, match="GPU"):
        sample_filtered(x, 1.0, torch.zeros(2))
    with pytest.raises(ValueError, match="GPU"):
        accept_filtered(x, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), 1.0, torch.zeros(1, 2))


def test_alignment():
    odd, two, eight = (ctypes.c_void_p(0x1000 + n) for n in (1, 2, 8))
    assert _sample(logits=odd) == _sample(logits=two, dtype=0) == _accept(target=odd) == _accept(draft=two, dtype=0) == ARG
    assert _sample(ws=eight) == _accept(ws=eight) == WORKSPACE
