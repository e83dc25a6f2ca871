"""accept_filtered against the oracle, and together with sample_filtered."""

import numpy as np
import pytest
import torch

from naivllm_amd.spec_engine.rejection_sampler import accept_filtered, sample_filtered
from oracle.filtered import Row, accept
from tests.filtered_util import logits, on_gpu, settings

pytestmark = pytest.mark.gpu
NAMES = ("temperature", "top_k", "top_p", "min_p")


def _case(seed, B, K, V, dtype, shape="peaked", near=0.5):
    """Target rows, draft rows near them, drafts of which most are likely."""
    target = logits(seed, B * (K + 1), V, dtype, shape).view(B, K + 1, V)
    gen = torch.Generator().manual_seed(seed)
    draft = (target[:, :K].float() + near * torch.randn((B, K, V), generator=gen)).to(target.dtype)
    f, rng = settings(seed, B), np.random.default_rng(seed)
    drafts = np.zeros((B, K), np.int32)
    for b in range(B):
        for i in range(K):
            r = Row(draft[b, i].double().numpy(), *(f[n][b] for n in NAMES))
            drafts[b, i] = r.sample(rng.random()) if rng.random() < 0.85 else rng.integers(0, V)
    live = np.array([K - (b % 4 == 3) - (b % 6 == 5) * K // 2 for b in range(B)], np.int32).clip(0)
    return target, draft, f, drafts, live, rng.random((B, K + 1), dtype=np.float32)


def _want(target, draft, f, drafts, live, u, mode=None):
    out = []
    K = drafts.shape[1]
    for b in range(len(drafts)):
        n = int(min(max(live[b], 0), K))
        rows = draft is not None and (mode is None or mode[b] != 0)
        out.append(accept(target[b, :n + 1].double().numpy(), draft[b, :n].double().numpy() if rows else None,
                          drafts[b, :n].tolist(), np.append(u[b, :n], u[b, K if rows and f["temperature"][b] > 1e-6 else n]),
                          *(f[name][b] for name in NAMES)))
    return out


def _run(target, draft, f, drafts, live, u, mode=None, **kw):
    B, K = drafts.shape
    V = target.shape[-1]
    tokens = torch.full((B, K + 1), -9, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    if draft is not None and "draft_logits" not in kw:
        kw |= dict(draft_logits=draft.reshape(-1, V).cuda(), draft_seq_stride=K)
    if mode is not None:
        kw["draft_mode"] = torch.from_numpy(mode).cuda()
    accept_filtered(target.reshape(-1, V).cuda(), torch.from_numpy(drafts).cuda(), torch.from_numpy(live).cuda(),
                    uniforms=torch.from_numpy(u).cuda(), out_tokens=tokens, out_len=lens, **on_gpu(f), **kw)
    torch.cuda.synchronize()
    return _lists(tokens, lens)


def _lists(tokens, lens):
    tokens, lens = tokens.tolist(), lens.tolist()
    assert all(x == -9 for t, n in zip(tokens, lens) for x in t[n:]), "written past a sequence's tokens"
    return [t[:n] for t, n in zip(tokens, lens)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("mode", ["model", "ngram", "hybrid"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 11), (2, 3, 100), (7, 4, 2048), (14, 5, 2049), (3, 2, 40009)])
def test_rounds(B, K, V, mode, dtype):
    print(f"case: accept_filtered {mode} {B} {K} {V} {dtype}", flush=True)
    for n, shape in enumerate(("peaked", "flat", "levels")):
        target, draft, f, drafts, live, u = _case(V + K + n, B, K, V, dtype, shape)
        draft = None if mode == "ngram" else draft
        modes = (np.arange(B) % 2).astype(np.int32) if mode == "hybrid" else None
        got = _run(target, draft, f, drafts, live, u, modes)
        assert got == _want(target, draft, f, drafts, live, u, modes), shape


def test_full_vocabulary():
    print("case: accept_filtered 151936", flush=True)
    target, draft, f, drafts, live, u = _case(5, 3, 4, 151936, "bf16", "flat", 0.2)
    f["temperature"][:] = [0.7, 1.0, 1.3]
    assert _run(target, draft, f, drafts, live, u) == _want(target, draft, f, drafts, live, u)


@pytest.mark.parametrize("K", [0, 63])
def test_draft_counts(K):
    print(f"case: accept_filtered K {K}", flush=True)
    target, draft, f, drafts, live, u = _case(K, 7, K, 37, "bf16", "flat", 0.05)
    live = np.array([K, 0, K + 5, -3, K // 2, K, K], np.int32)
    for d in (draft, None):
        assert _run(target, d, f, drafts, live, u) == _want(target, d, f, drafts, live, u)


def test_drafts_outside_the_vocabulary_and_no_residual():
    """Equal rows leave no residual: a refused draft's token comes from the
    target itself, an accepted one never fails."""
    print("case: accept_filtered equal rows", flush=True)
    target, _, f, drafts, live, u = _case(9, 14, 3, 300, "f32")
    draft = target[:, :3]
    drafts[::2, 1] = [300, -1, 2 ** 30, -2 ** 31, 300, 301, 5000]
    got = _run(target, draft, f, drafts, live, u)
    assert got == _want(target, draft, f, drafts, live, u)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_masked_rows_and_nan(dtype):
    print(f"case: accept_filtered masks {dtype}", flush=True)
    target, draft, f, drafts, live, u = _case(21, 14, 3, 999, dtype, "flat")
    gen = torch.Generator().manual_seed(5)
    hide = torch.rand(target.shape, generator=gen) < 0.9
    target = target.masked_fill(hide, -np.inf)
    draft = draft.masked_fill(hide[:, :3], -np.inf)
    target[3, 0] = -np.inf   # a target row with nothing left
    draft[4, 1] = -np.inf
    target[5, 1, 77] = np.nan
    draft[6, 0, 5] = np.nan
    target[7, 0, [3, 8]] = np.inf
    assert _run(target, draft, f, drafts, live, u) == _want(target, draft, f, drafts, live, u)


def test_step_major_draft_rows_and_padded_sequences():
    """The round's layouts: draft rows [K, batch, V], sequences of more rows than K + 1."""
    print("case: accept_filtered layouts", flush=True)
    B, K, V = 5, 3, 1501
    target, draft, f, drafts, live, u = _case(31, B, K, V, "bf16")
    wide = torch.full((B, K + 3, V), 7.0, dtype=target.dtype)
    wide[:, :K + 1] = target
    steps = torch.full((K, B + 2, V), 7.0, dtype=target.dtype)
    steps[:, :B] = draft.transpose(0, 1)
    got = _run(wide, draft, f, drafts, live, u, target_seq_stride=K + 3, draft_logits=steps.cuda(), draft_seq_stride=1,
               draft_row_stride=B + 2)
    assert got == _want(target, draft, f, drafts, live, u)


def test_captured_graphs_beside_each_other():
    """Two captured rounds and an eager one, at once on three streams."""
    print("case: accept_filtered captured", flush=True)
    B, K, V = 8, 4, 30011
    cases = [_case(40 + n, B, K, V, "bf16") for n in range(3)]
    args, outs, graphs = [], [], []
    for target, draft, f, drafts, live, u in cases:
        args.append(((target.reshape(-1, V).cuda(), torch.from_numpy(drafts).cuda(), torch.from_numpy(live).cuda()),
                     dict(uniforms=torch.from_numpy(u).cuda(), draft_logits=draft.reshape(-1, V).cuda(),
                          draft_seq_stride=K, **on_gpu(f))))
        outs.append(dict(out_tokens=torch.full((B, K + 1), -9, dtype=torch.int32, device="cuda"),
                         out_len=torch.zeros(B, dtype=torch.int32, device="cuda")))
    accept_filtered(*args[2][0], **args[2][1], **outs[2])
    torch.cuda.synchronize()
    for n in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            accept_filtered(*args[n][0], **args[n][1], **outs[n])
        graphs.append(g)
    want = [_want(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for o in outs:
            o["out_tokens"].fill_(-9)
            o["out_len"].zero_()
        torch.cuda.synchronize()
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                if n < 2:
                    graphs[n].replay()
                else:
                    accept_filtered(*args[n][0], **args[n][1], **outs[n])
        torch.cuda.synchronize()
        assert [_lists(o["out_tokens"], o["out_len"]) for o in outs] == want


def test_drafted_and_accepted_tokens_follow_the_filtered_target():
    """A round as it is used: drafts sampled under the filters from the draft
    row, accepted under them; the first tokens' frequencies over many
    sequences are the filtered target's."""
    print("case: accept_filtered distribution", flush=True)
    B, V = 20000, 24
    target, draft = logits(1, 2, V, "f32"), logits(2, 1, V, "f32")
    f = dict(temperature=0.9, top_k=12, top_p=0.93, min_p=0.004)
    gen = torch.Generator(device="cuda").manual_seed(7)
    u = torch.rand((B, 3), device="cuda", generator=gen)
    rows = draft.cuda().expand(B, V).contiguous()
    drafts = sample_filtered(rows, uniforms=u[:, 2].contiguous(), **f)
    tokens, lens = accept_filtered(target.cuda().expand(B, 2, V).reshape(-1, V).contiguous(), drafts[:, None],
                                   torch.ones(B, dtype=torch.int32, device="cuda"), uniforms=u[:, :2].contiguous(),
                                   draft_logits=rows, draft_seq_stride=1, **f)
    for n, row in ((0, target[0]), (1, target[1])):
        p = Row(row.double().numpy(), *f.values()).probabilities()
        some = tokens[:, n][lens > n].cpu().numpy()
        share = np.bincount(some, minlength=V) / len(some)
        assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / len(some)) + 1e-12).all(), n
