"""SamplingParams' filters: their checks, and what a sequence takes from them."""

import pytest

from naivllm_amd.engine.sequence import Sequence
from naivllm_amd.sampling_parameters import SamplingParams


@pytest.mark.parametrize("bad", [dict(top_k=-1), dict(top_k=2.0), dict(top_k=True), dict(top_k=None), dict(top_p=0.0),
                                 dict(top_p=1.01), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.5),
                                 dict(min_p=float("nan"))])
def test_refuses(bad):
    with pytest.raises(ValueError, match=next(iter(bad))):
        SamplingParams(temperature=1.0, **bad)


@pytest.mark.parametrize("settings,filtered", [
    (dict(temperature=1.0), False), (dict(temperature=1.0, top_k=5), True), (dict(temperature=0.5, top_p=0.9), True),
    (dict(temperature=2.0, min_p=0.1), True), (dict(temperature=0.0, top_k=5, top_p=0.5, min_p=0.5), False)])
def test_a_sequence_knows_whether_it_is_filtered(settings, filtered):
    seq = Sequence([1, 2, 3], SamplingParams(**settings))
    assert seq.filtered is filtered
    assert (seq.top_k, seq.top_p, seq.min_p) == (settings.get("top_k", 0), settings.get("top_p", 1.0), settings.get("min_p", 0.0))


def test_the_defaults_filter_nothing():
    assert not Sequence([1]).filtered


def test_settings_of_the_references_fields():
    class Plain:
        temperature, max_tokens, ignore_eos, max_model_length = 0.8, 5, False, None

    seq = Sequence([1, 2], Plain())
    assert not seq.filtered and (seq.top_k, seq.top_p, seq.min_p) == (0, 1.0, 0.0)


def test_a_top_k_beyond_32_bits_keeps_everything():
    seq = Sequence([1], SamplingParams(temperature=1.0, top_k=1 << 40))
    assert seq.top_k == 0x7fffffff


@pytest.mark.parametrize("top_k", [-1, -2 ** 31 - 1, -2 ** 40])
def test_a_callers_own_settings_below_zero_keep_everything(top_k):
    class Own:
        temperature, max_tokens, ignore_eos, max_model_length = 0.8, 5, False, None

    Own.top_k = top_k
    seq = Sequence([1], Own())
    assert seq.top_k == 0 and not seq.filtered
