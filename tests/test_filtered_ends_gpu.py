"""Filtered sampling and acceptance by uniform numbers at and next to the end
of their range, against the oracle."""

import numpy as np
import pytest
import torch

from naivllm_amd.spec_engine.rejection_sampler import accept_filtered, sample_filtered
from tests.filtered_util import logits, on_gpu
from tests.test_filtered_accept_gpu import _case, _run, _want
from tests.test_filtered_sample_gpu import _check

pytestmark = pytest.mark.gpu


def _settings(B, **kw):
    f = dict(temperature=np.ones(B, np.float32))
    return f | {k: np.full(B, v, np.int32 if k == "top_k" else np.float32) for k, v in kw.items()}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_behind_two_kept(dtype):
    """1 takes the last token kept, not the first behind it."""
    print(f"case: sample_filtered of 1, three tokens {dtype}", flush=True)
    x = logits(0, 1, 3, dtype).copy_(torch.tensor([[2.0, 1.0, 0.0]]))
    for kw in (dict(top_k=2), dict(top_p=0.8), dict(min_p=0.2)):
        for u in (1.0, 7.0):
            assert _check(x, _settings(1, **kw), np.full(1, u, np.float32)) == 1, (kw, u)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [0.0, 200.0])
@pytest.mark.parametrize("setting", [dict(top_k=2), dict(top_k=300), dict(top_p=0.5), dict(top_p=0.9), dict(min_p=0.3),
                                     dict(min_p=2e-3), dict(top_k=400, top_p=0.8, min_p=0.01)])
def test_one_under_filters(dtype, shift, setting):
    """The same of long rows, whose cuts lie between distinct and between equal
    values; rows around 200 have more fp32 tokens next to a cut than are listed."""
    print(f"case: sample_filtered of 1, {setting} around {shift} {dtype}", flush=True)
    B, V = 4, 20011
    for n, shape in enumerate(("flat", "peaked", "levels", "equal")):
        x = (logits(50 + n, B, V, "f32", shape) + shift).to(logits(0, 1, 1, dtype).dtype)
        assert _check(x, _settings(B, **setting), np.ones(B, np.float32)) == B, shape


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("mode", ["model", "ngram", "hybrid"])
def test_one_in_rounds(mode, dtype):
    """Nearly all numbers are 1: samples, refused drafts, residuals, bonus rows."""
    print(f"case: accept_filtered of 1, {mode} {dtype}", flush=True)
    target, draft, f, drafts, live, u = _case(61, 9, 4, 2049, dtype, near=0.02)
    f = dict(temperature=np.full(9, 0.9, np.float32), top_k=np.where(np.arange(9) % 3 == 0, 40, 0).astype(np.int32),
             top_p=np.where(np.arange(9) % 3 == 1, 0.8, 1.0).astype(np.float32),
             min_p=np.where(np.arange(9) % 3 == 2, 0.02, 0.0).astype(np.float32))
    u[:] = 1.0
    u[::2, 0] = 0.0  # (1 refuses a draft more likely in the draft row)
    draft = None if mode == "ngram" else draft
    modes = (np.arange(9) % 2).astype(np.int32) if mode == "hybrid" else None
    assert _run(target, draft, f, drafts, live, u, modes) == _want(target, draft, f, drafts, live, u, modes)


@pytest.mark.parametrize("setting", [dict(), dict(top_k=900), dict(top_p=1 - 2.0 ** -24, top_k=4000)])
@pytest.mark.parametrize("count", [1, 3, 700])
def test_one_behind_a_far_maximum(count, setting):
    """At a low temperature tokens of 3 weigh e^-150 beside a maximum of 3.3 in
    another stretch of the row, and e^-62 of the largest value next to them: the
    sample of 1 is the maximum or one of them, never a masked token."""
    print(f"case: sample_filtered of 1 behind a far maximum, {count} tokens, {setting}", flush=True)
    B, V = 2, 20000
    x = torch.full((B, V), -np.inf)
    x[:, 5000] = 3.3
    x[0, 10000:10000 + count] = 3.0
    x[1, 10000:10000 + count] = 3.0 + 2.0 ** -20 * torch.arange(count)
    f = _settings(B, **setting) | dict(temperature=np.full(B, 0.002, np.float32))
    kept = torch.zeros(B, dtype=torch.int32, device="cuda")
    got = sample_filtered(x.cuda(), uniforms=torch.ones(B, device="cuda"), kept=kept, **on_gpu(f))
    assert torch.isfinite(x.gather(1, got.cpu().long()[:, None])).all()
    assert _check(x, f, np.ones(B, np.float32), got, kept) is not None


def test_wide_numbers_below_one():
    """64-bit numbers below 1 that round to 1 in 32 bits, and such a number for
    every row: a draft as likely in both rows stays, a sample is a kept token."""
    print("case: filtered draws of 64-bit numbers next to 1", flush=True)
    B, K, V = 3, 2, 64
    near = torch.tensor([1 - 2.0 ** -26, 1 - 2.0 ** -40, 1 - 2.0 ** -53], dtype=torch.float64, device="cuda")
    rows = logits(5, B * (K + 1), V, "f32").cuda()
    draft = rows.view(B, K + 1, V)[:, :K].reshape(-1, V).contiguous()
    drafts = draft.argmax(1).view(B, K).int()
    tokens, lens = accept_filtered(rows, drafts, torch.full((B,), K, dtype=torch.int32), 1.0, near[:, None].expand(B, K + 1),
                                   draft_logits=draft, draft_seq_stride=K, top_k=5)
    assert lens.tolist() == [K + 1] * B and torch.equal(tokens[:, :K], drafts)
    x = torch.tensor([[2.0, 1.0, 0.0]], device="cuda").expand(B, 3).contiguous()
    for u in (near, 1 - 2.0 ** -30):
        assert sample_filtered(x, 1.0, u, top_k=2).tolist() == [1] * B
