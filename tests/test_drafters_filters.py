"""Drafters that apply a temperature alone, and sequences with filters (CPU)."""

import pytest

from naivllm_amd.engine.sequence import Sequence
from naivllm_amd.sampling_parameters import SamplingParams
from naivllm_amd.spec_engine import HybridDrafter, ModelDrafter


class Lookup:
    """An n-gram drafter that has a match for sequences beginning with 1."""

    def draft(self, seqs):
        for s in seqs:
            s.draft_tokens = [7, 8] if s.token_ids[0] == 1 else []
            for t in s.draft_tokens:
                s.append_token(t)
        return [list(s.draft_tokens) for s in seqs], [None] * len(seqs)


class Pages:
    def can_ensure_capacity(self, *a):
        return True

    def ensure_capacity(self, *a):
        raise AssertionError("reserved pages for a refused call")


def _drafter():
    model = ModelDrafter.__new__(ModelDrafter)
    model.num_speculative_tokens, model.block_manager = 4, Pages()
    return HybridDrafter(Lookup(), model)


@pytest.mark.parametrize("first", [1, 2])  # with a match and without
@pytest.mark.parametrize("filters", [dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1)])
def test_hybrid_refuses_filters_before_it_drafts(first, filters):
    seqs = [Sequence([1, 2, 3], SamplingParams(temperature=1.0)), Sequence([first, 4], SamplingParams(temperature=1.0, **filters))]
    drafter = _drafter()
    with pytest.raises(ValueError, match="top_k"):
        drafter.draft(seqs)
    assert [s.token_ids for s in seqs] == [[1, 2, 3], [first, 4]] and not any(s.draft_tokens for s in seqs)
    assert drafter.model_rounds == drafter.model_seqs == 0


def test_hybrid_takes_greedy_sequences_with_filters():
    seqs = [Sequence([1, 2], SamplingParams(temperature=0.0, top_k=5))]
    assert _drafter().draft(seqs) == ([[7, 8]], [None])
