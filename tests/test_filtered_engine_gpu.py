"""The filters inside the engine's rounds, and the operators together: sampled
continuations of one prompt that share its pages."""

import numpy as np
import pytest
import torch

from naivllm_amd.engine.sequence import Sequence
from naivllm_amd.layers.qwen3 import Qwen3Verify
from naivllm_amd.sampling_parameters import SamplingParams
from naivllm_amd.spec_engine import ModelDrafter, SpecLLMEngine
from naivllm_amd.spec_engine.rejection_sampler import accept_filtered, sample_filtered
from naivllm_amd.utils import synth
from oracle import ngram as on
from oracle import round as orr
from oracle.filtered import Row, accept
from tests.test_fused_gpu import dense_forward
from tests.test_model_draft_gpu import DRAFT, TARGET, _load, prompts_with_spans

pytestmark = pytest.mark.gpu
BASE = dict(model_config=TARGET, draft_model_config=DRAFT, num_speculative_tokens=4, ngram_min_size=2, ngram_max_size=4,
            max_num_sequences=4, max_model_length=512, block_size=16, seed=9)
# These untrained models share the embedding with the output, so the last token's own logit is some 190 and the others'
# at most 60: below a temperature of 10 its weight is all there is (e^-13 for the next), at 100 the next has e^-1.3.
HOT = 100.0


@pytest.mark.parametrize("method", ["ngram", "model", "hybrid", "none"])
def test_a_filtered_round_matches_a_host_restatement(method):
    # every draft and every accepted token is the oracle's on the round's own logits and numbers
    print(f"case: filtered {method} round vs host restatement", flush=True)
    eng = SpecLLMEngine({**BASE, "spec_method": method, "enforce_eager": True})
    r = eng._round(True, filtered=True)
    K, V = r.K, TARGET.vocab_size
    prompts = prompts_with_spans(8, 4)
    hists = [prompts[0][:45], prompts[1][:37], [int(x) for x in synth.randint(5, 92, 33, 0, V)], prompts[3][:52]]
    filters = [(90.0, 0, 0.9, 0.0), (70.0, 40, 1.0, 0.0), (HOT, 200, 0.8, 0.02), (0.0, 0, 1.0, 0.0)]
    _load(eng, r, hists, temps=[f[0] for f in filters])
    for b, (_, k, p, m) in enumerate(filters):
        r.top_k[b], r.top_p[b], r.min_p[b] = k, p, m
    B = len(hists)
    r.body(B)
    torch.cuda.synchronize()
    wide = lambda t: t.double().cpu().numpy()  # noqa: E731
    drafts = [r.drafts[b, :int(r.num_drafts[b])].tolist() for b in range(B)]
    ng = on.draft(hists, K, 2, 4) if K else [[]] * B
    mode = [0] * B
    if method in ("model", "hybrid"):
        DL, DU, MD = wide(r.draft_logits), r.draft_uniforms.cpu().numpy(), r.model_drafts[:B].tolist()
        flat = DU.reshape(-1)
        assert len(np.unique(flat)) == len(flat)  # a number of its own for every draw
        for b in range(B):
            assert MD[b] == [Row(DL[i, b], *filters[b]).sample(DU[i, b]) for i in range(K)], b
        mode = [int(method == "model" or not ng[b]) for b in range(B)]
        assert r.draft_mode[:B].tolist() == mode
        assert drafts == [MD[b] if mode[b] else ng[b] for b in range(B)]
        if method == "hybrid":
            assert 0 < sum(mode) < B  # the case mixes both kinds
    else:
        assert drafts == ng
    T, U = wide(r.logits[:B * (K + 1)]), r.uniforms.cpu().numpy()
    got = [r.out_tokens[b, :int(r.out_len[b])].tolist() for b in range(B)]
    for b in range(B):
        n = len(drafts[b])
        rows = mode[b] and filters[b][0] > 0
        want = accept(T[b * (K + 1):b * (K + 1) + n + 1], DL[:n, b] if rows else None, drafts[b],
                      np.append(U[b, :n], U[b, K if rows else n]), *filters[b])
        assert got[b] == want, b
        history, _ = orr.commit(hists[b], len(hists[b]) - 2, want, 100, -1, True, None)
        assert r.history[b, :int(r.hist_len[b])].tolist() == history


@pytest.mark.parametrize("method", ["ngram", "model", "hybrid", "none"])
@pytest.mark.parametrize("eager", [False, True])
def test_one_token_left_is_greedy_decoding(method, eager):
    # top-k 1 and a tiny top-p leave the first of the largest logits at any temperature
    print(f"case: filters that leave one token, {method}, eager {eager}", flush=True)
    prompts = prompts_with_spans(7, 4)
    common = dict(max_tokens=24, ignore_eos=True)
    with SpecLLMEngine({**BASE, "spec_method": "none"}) as plain:
        want = [o["token_ids"] for o in plain.generate(prompts, SamplingParams(temperature=0.0, **common))["outputs"]]
    params = [SamplingParams(temperature=HOT, top_k=1, **common), SamplingParams(temperature=2 * HOT, top_k=1, min_p=1.0, **common),
              SamplingParams(temperature=HOT, top_p=1e-6, **common), SamplingParams(temperature=0.0, top_k=9, **common)]
    with SpecLLMEngine({**BASE, "spec_method": method, "enforce_eager": eager}) as eng:
        for again in range(2):  # and once more through the same round
            got = eng.generate(prompts, params)
            assert list(eng.rounds) == ["filtered"]
            assert [o["token_ids"] for o in got["outputs"]] == want, again
        greedy = eng.generate(prompts, SamplingParams(temperature=0.0, **common))
        assert [o["token_ids"] for o in greedy["outputs"]] == want and set(eng.rounds) == {"filtered", False}


def test_generated_tokens_are_among_the_kept():
    # top-k 3 in captured rounds: each token within the 3 largest of a dense float32 forward, up to its error
    print("case: tokens of a filtered generation", flush=True)
    prompts = prompts_with_spans(12, 3)
    with SpecLLMEngine({**BASE, "spec_method": "hybrid"}) as eng:
        out = eng.generate(prompts, SamplingParams(temperature=HOT, top_k=3, max_tokens=30, ignore_eos=True))["outputs"]
        ranks = []
        for prompt, o in zip(prompts, out):
            ids = torch.tensor(prompt + o["token_ids"], device="cuda")
            rows = dense_forward(eng.model, ids)[len(prompt) - 1:-1]
            drawn = rows.gather(1, ids[len(prompt):, None])
            # the forward is within 2e-2 of the dense one in norm: a logit by 5 times that in its row's root mean square
            error = 5 * 2e-2 * rows.pow(2).mean(1, keepdim=True).sqrt()
            assert (drawn >= rows.topk(3).values[:, 2:] - 2 * error).all()
            ranks += (rows > drawn).sum(1).tolist()
        assert len(set(ranks)) > 1  # and not the argmax alone


def test_a_drafter_outside_the_rounds_refuses_filters():
    class Pages:
        def ensure_capacity(self, *a):
            raise AssertionError("reserved pages for a refused call")

    drafter = ModelDrafter.__new__(ModelDrafter)
    drafter.num_speculative_tokens, drafter.block_manager = 4, Pages()
    with pytest.raises(ValueError, match="top_k"):
        drafter.draft([Sequence([1, 2, 3], SamplingParams(temperature=1.0, top_k=5))])


class Rows:
    """Sequences of one model, decoded together a token at a time."""

    def __init__(self, model, B, width):
        self.model, self.B = model, B
        self.tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(B, dtype=torch.int64, device="cuda")
        self.cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")

    def step(self, tokens, rows=1):
        """The logits behind ``tokens`` [B * rows], which the cache takes in."""
        bs, dev = self.model.block_size, "cuda"
        at = (self.lens[:, None] + torch.arange(rows, device=dev)).view(-1)
        seq = torch.arange(self.B, device=dev).repeat_interleave(rows)
        slots = self.tables[seq, at // bs].long() * bs + at % bs
        self.lens += rows
        return self.model.forward(tokens.long(), at, slots, self.tables, self.lens, self.cu * rows, rows)


@pytest.mark.parametrize("prompt_len", [41, 48])  # a partly filled page, and none
def test_continuations_of_one_prompt(prompt_len):
    # The prompt prefilled once and forked; filtered samples; survivors forked again, one row ended; the pages
    # compacted; a round of drafts accepted.  Beside it, rows with pages of their own, moved by plain indexing:
    # the same tokens and the same logits, bit for bit (a page's number enters no arithmetic).
    print(f"case: continuations of a {prompt_len}-token prompt", flush=True)
    B, bs, width, steps, K = 5, 16, 6, 9, 2
    model = Qwen3Verify(TARGET, "cuda", seed=5)
    model.allocate_kv_cache(B * width + 3, bs)
    pages = model.cache_pages()
    held = torch.zeros(pages.num_blocks, dtype=torch.bool, device="cuda")
    held[[0, 7]] = True
    for cache in model.k_caches + model.v_caches:
        cache[held] = 3.0  # another's
    rng = np.random.default_rng(prompt_len)
    prompt = [int(x) for x in rng.integers(0, TARGET.vocab_size, prompt_len)]
    first = [30, 4, 19, 8, 2, 25]
    start = model.prefill([prompt], [0], [first])

    other = Qwen3Verify(TARGET, "cuda", seed=5)
    other.allocate_kv_cache(B * width, bs)
    own = Rows(other, B, width)
    own.tables.copy_(torch.arange(B * width, device="cuda").view(B, width))
    own.lens.fill_(prompt_len)
    for mine, theirs in zip(model.k_caches + model.v_caches, other.k_caches + other.v_caches):
        theirs.copy_(mine[first].repeat(B, 1, 1, 1))

    run = Rows(model, B, width)
    run.tables[0] = torch.tensor(first, device="cuda")
    run.lens[0] = prompt_len
    parents = torch.zeros(B, dtype=torch.int32, device="cuda")
    run.tables, run.lens, lacking = pages.fork(run.tables, run.lens, parents, held=held)
    assert int(lacking) == 0
    filters = dict(temperature=HOT, top_k=60, top_p=0.95, min_p=0.01)
    history = [list(prompt) for _ in range(B)]
    logits = own_logits = start.expand(B, -1).contiguous()
    gen = torch.Generator(device="cuda").manual_seed(3)

    def fork(order):
        nonlocal logits, own_logits, history
        parents = torch.tensor(order, dtype=torch.int32, device="cuda")
        run.tables, run.lens, lacking = pages.fork(run.tables, run.lens, parents, held=held)
        assert int(lacking) == 0
        at = parents.long()
        logits, own_logits, history = logits[at], own_logits[at], [list(history[p]) for p in order]
        own.lens = own.lens[at]
        for cache in other.k_caches + other.v_caches:
            cache.copy_(cache.view(B, width, *cache.shape[1:])[at].reshape(cache.shape))

    for i in range(steps):
        u = torch.rand(B, device="cuda", generator=gen)
        tokens = sample_filtered(logits, uniforms=u, **filters)
        assert torch.equal(tokens, sample_filtered(own_logits, uniforms=u, **filters))
        for h, t in zip(history, tokens.tolist()):
            h.append(t)
        logits, own_logits = run.step(tokens), own.step(tokens)
        assert torch.equal(logits, own_logits), i
        if i in (2, 6):
            fork([3, 3, 0, 4, 3])
        if i == 4:
            before = run.tables.clone()
            run.tables, new_ids, top = pages.compact(run.tables, held=held)
            used = before.unique()
            assert int(top) == len(used[used >= 0]) + 2 and int(run.tables.max()) < int(top)
            assert new_ids[[0, 7]].tolist() == [0, 7]
    assert len({tuple(h) for h in history}) > 1
    # a round: K drafts a row from the rows' own filters on the same logits, then the rows they verify
    drafts = torch.stack([sample_filtered(logits, uniforms=torch.rand(B, device="cuda", generator=gen), **filters)
                          for _ in range(K)], 1)
    pending = sample_filtered(logits, uniforms=torch.rand(B, device="cuda", generator=gen), **filters)
    verify = torch.cat([pending[:, None], drafts], 1).view(-1)
    rows, own_rows = run.step(verify, K + 1), own.step(verify, K + 1)
    assert torch.equal(rows, own_rows)
    u = torch.rand(B, K + 1, device="cuda", generator=gen)
    live = torch.tensor([2, 2, 0, 1, 2], dtype=torch.int32, device="cuda")
    tokens, n = accept_filtered(rows, drafts, live, uniforms=u, **filters)
    for b in range(B):
        k = int(live[b])
        want = accept(rows.view(B, K + 1, -1)[b, :k + 1].double().cpu().numpy(), None, drafts[b, :k].tolist(),
                      u[b, :k + 1].cpu().numpy(), *filters.values())
        assert tokens[b, :int(n[b])].tolist() == want
    # the histories' dense forward, with the verify rows behind them
    for b in range(B):
        ids = torch.tensor(history[b] + verify.view(B, -1)[b].tolist(), device="cuda")
        want = dense_forward(model, ids)[-(K + 1):]
        got = rows.view(B, K + 1, -1)[b].float()
        assert ((got - want).norm(dim=1) / want.norm(dim=1)).max() < 2e-2
    for cache in model.k_caches + model.v_caches:
        assert (cache[held] == 3.0).all()
