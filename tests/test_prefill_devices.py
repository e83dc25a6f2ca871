"""The prompts' operators refuse tensors and plans of another device than the
query's: nothing here launches a kernel."""

from types import SimpleNamespace

import pytest
import torch

from naivllm_amd.layers.attention import prefill_attention, prefill_key_weights


class Somewhere:
    """A tensor of another device than the one it was made on, as far as
    checks see it."""

    def __init__(self, t, index):
        self._t, self._index = t, index

    is_cuda = property(lambda self: self._index >= 0)
    device = property(lambda self: torch.device("cuda", self._index) if self._index >= 0 else torch.device("cpu"))

    def get_device(self):
        return self._index

    def __getattr__(self, name):
        return getattr(self._t, name)


def _call(op, **index):
    at = lambda name, t: Somewhere(t, index.get(name, 0))  # noqa: E731
    query = at("query", torch.zeros((2, 4, 64), dtype=torch.bfloat16))
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    plan = SimpleNamespace(num_heads=4, num_kv_heads=2, rows=2, keys=2, sequences=1, block_size=16, longest=2, window=0,
                           work=at("plan", torch.zeros(8, dtype=torch.int32)))
    tables = at("block_tables", torch.zeros((1, 2), dtype=torch.int32))
    if op == "attention":
        return prefill_attention(query, at("k", cache), at("v", cache), plan, 0.1, 64, tables)
    if op == "contiguous":
        kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
        return prefill_attention(query, at("k", kv), at("v", kv), plan, 0.1, 64)
    return prefill_key_weights(query, at("k_cache", cache), torch.zeros((4, 2, 16)), plan, None, 0.1, 64, tables)


@pytest.mark.parametrize("op,name", [("attention", "k"), ("attention", "v"), ("attention", "block_tables"),
                                     ("attention", "plan"), ("contiguous", "k"), ("contiguous", "v"),
                                     ("contiguous", "plan"), ("weights", "k_cache"), ("weights", "block_tables"),
                                     ("weights", "plan")])
@pytest.mark.parametrize("index", [-1, 1])
def test_refused(op, name, index):
    with pytest.raises(ValueError, match=f"{name} is on {'cpu' if index < 0 else 'cuda:1'}, query on cuda:0"):
        _call(op, **{name: index})
