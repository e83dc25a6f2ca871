"""Calls that sample_filtered and accept_filtered refuse before a launch."""

import pytest
import torch

from naivllm_amd.spec_engine.rejection_sampler import accept_filtered, sample_filtered

pytestmark = pytest.mark.gpu


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32, device="cuda")


def _sample(**kw):
    a = dict(logits=torch.zeros(3, 64, device="cuda"), temperature=1.0, uniforms=torch.zeros(3, device="cuda")) | kw
    return sample_filtered(a.pop("logits"), a.pop("temperature"), a.pop("uniforms"), **a)


@pytest.mark.parametrize("bad", [
    lambda: dict(logits=torch.zeros(64, device="cuda")), lambda: dict(logits=torch.zeros(3, 64, device="cuda").half()),
    lambda: dict(logits=torch.zeros(64, 3, device="cuda").t()), lambda: dict(logits=torch.zeros(1, 64, device="cuda").expand(3, 64)),
    lambda: dict(logits=torch.zeros(200, device="cuda").as_strided((3, 64), (40, 1))),
    lambda: dict(logits=torch.zeros(3, (1 << 20) + 1, device="cuda", dtype=torch.bfloat16)),
    lambda: dict(temperature=None), lambda: dict(temperature=torch.ones(2, device="cuda")), lambda: dict(temperature="1"),
    lambda: dict(uniforms=None), lambda: dict(uniforms=torch.zeros(4, device="cuda")),
    lambda: dict(uniforms=torch.zeros(3, 1, device="cuda")),
    lambda: dict(top_k=2.5), lambda: dict(top_k=True), lambda: dict(top_k=torch.ones(3, device="cuda")),
    lambda: dict(top_p=_i32(2)), lambda: dict(min_p=torch.zeros(3, dtype=torch.bool, device="cuda")),
    lambda: dict(out=_i32(4)), lambda: dict(out=_i32(3).long()), lambda: dict(out=torch.zeros(3, dtype=torch.int32)),
    lambda: dict(out=_i32(1).expand(3)), lambda: dict(kept=_i32(3, 2)[:, 0]), lambda: dict(kept=_i32(2))])
def test_sample(bad):
    with pytest.raises(ValueError):
        _sample(**bad())


def _accept(**kw):
    a = dict(target=torch.zeros(6, 64, device="cuda"), drafts=_i32(2, 2), live=_i32(2), temperature=1.0,
             uniforms=torch.zeros(2, 3, device="cuda"), draft_logits=torch.zeros(4, 64, device="cuda"), draft_seq_stride=2) | kw
    return accept_filtered(a.pop("target"), a.pop("drafts"), a.pop("live"), a.pop("temperature"), a.pop("uniforms"), **a)


@pytest.mark.parametrize("bad", [
    lambda: dict(target=torch.zeros(5, 64, device="cuda")), lambda: dict(target=torch.zeros(6, 128, device="cuda")[:, :64]),
    lambda: dict(drafts=_i32(4)), lambda: dict(live=_i32(3)), lambda: dict(uniforms=torch.zeros(2, 2, device="cuda")),
    lambda: dict(draft_logits=torch.zeros(3, 64, device="cuda")), lambda: dict(draft_logits=torch.zeros(4, 63, device="cuda")),
    lambda: dict(draft_logits=torch.zeros(4, 64, device="cuda").bfloat16()), lambda: dict(draft_row_stride=0),
    lambda: dict(draft_seq_stride=-1), lambda: dict(draft_seq_stride=3), lambda: dict(target_seq_stride=2),
    lambda: dict(draft_mode=_i32(3)), lambda: dict(draft_logits=None, draft_mode=_i32(2)), lambda: dict(temperature=None),
    lambda: dict(drafts=_i32(1, 64), live=_i32(1), uniforms=torch.zeros(1, 65, device="cuda"),
                 target=torch.zeros(65, 64, device="cuda"), draft_logits=None),
    lambda: dict(out_tokens=_i32(2, 2)), lambda: dict(out_tokens=_i32(2, 6)[:, ::2]), lambda: dict(out_len=_i32(3))])
def test_accept(bad):
    with pytest.raises(ValueError):
        _accept(**bad())


def test_what_is_allowed_runs():
    assert _sample(top_k=torch.full((3,), 2 ** 40, device="cuda"), out=_i32(3, 2)[:, 1]).shape == (3,)
    tokens, lens = _accept()
    assert tokens.shape == (2, 3) and lens.tolist() == [1, 1]


@pytest.mark.parametrize("draft", [lambda: torch.zeros(4, 128, device="cuda")[:, :64], lambda: torch.zeros(8, 64, device="cuda")[::2],
                                   lambda: torch.zeros(2, 3, 64, device="cuda")[:, :2],
                                   lambda: torch.zeros(1, 64, device="cuda").expand(4, 64)])
def test_draft_rows_apart(draft):
    """Rows of draft logits that do not lie one behind another: whatever lies
    between them would be taken for rows."""
    with pytest.raises(ValueError, match="draft_logits must be contiguous"):
        _accept(draft_logits=draft())


def test_draft_rows_of_a_larger_buffer():
    """Contiguous ones of it are taken, whatever lies before and behind."""
    buf = torch.full((7, 64), 9.0, device="cuda")
    buf[2:6] = 0.0
    buf[2, 5] = 3.0
    got, want = _accept(draft_logits=buf[2:6], top_k=4), _accept(draft_logits=buf[2:6].clone(), top_k=4)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0][:, 0], want[0][:, 0])


@pytest.mark.parametrize("top_k", [-2 ** 31 - 1, -2 ** 40, -10 ** 30, 10 ** 30])
def test_whole_numbers_past_32_bits(top_k):
    """As top_k: all stay."""
    kept = _i32(3)
    _sample(top_k=top_k, kept=kept)
    assert kept.tolist() == [64] * 3
