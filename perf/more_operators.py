"""Operators of several sampled continuations, as measurable cases.

Kinds of cases and what each stands for:
  sample   the next token of every row, from its logits and one uniform number,
           under a temperature, top-k, top-p and min-p of the row's own
  accept   a round's drafts kept or refused under the same filters: by
           min(1, p_target / p_draft) with a draw from the residual where the
           drafts come with logits, else while each equals the target's sample
  fork     rows of a paged cache that go on from other rows (one prompt's
           continuations, a beam step): whole pages become shared, pages still
           written to become each row's own, their live keys copied
  compact  the pages in use move to the front of their pools

Of a row x with maximum M, a temperature T <= 1e-6 leaves the first maximum.
Else w = exp((x - M) / T), and the tokens are ordered by falling x, equal ones by
rising index.  top-k leaves the first k (0: all), top-p the fewest of them whose
sum reaches p times theirs, min-p those with w >= min_p; what all three leave is a
beginning of the order, W its sum.  The sample of u is its first token whose
running sum exceeds u W; p(token) = w / W inside, 0 outside.

A draft d with logits stays if u p_draft(d) < p_target(d); at the first that does
not, the token is the first index whose running sum of max(p_target - p_draft, 0)
exceeds u' times their sum; behind kept drafts it is the last row's sample of u'.

A forked row has its parent's pages: whole ones shared, the others the parent's own
for its first child; the later children get free pages for them, the lowest first,
row by row.  Compacting moves the highest page that may move to the lowest free one
until they meet.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GREEDY = 1e-6


def listed() -> list[dict]:
    return [
        # the smallest call: one request's next token, nucleus sampling
        dict(name="sample_b1_top_p", kind="sample", dtype="bf16", rows=1, vocab=151936, shape="peaked", masked=0.0,
             filters="top_p"),
        # eight requests that each brought their own settings, one of them none, one greedy
        dict(name="sample_b8_mixed", kind="sample", dtype="bf16", rows=8, vocab=151936, shape="peaked", masked=0.0,
             filters="mixed"),
        # a large batch whose distributions are flat: the nucleus holds most of the vocabulary
        dict(name="sample_b256_flat", kind="sample", dtype="bf16", rows=256, vocab=151936, shape="flat", masked=0.0,
             filters="top_p"),
        # fp32 logits of an odd vocabulary, most tokens masked by a grammar
        dict(name="sample_b21_f32_masked", kind="sample", dtype="f32", rows=21, vocab=50001, shape="peaked",
             masked=0.9, filters="mixed"),
        # a verify round of eight requests with a draft model's five tokens each
        dict(name="accept_b8_model", kind="accept", dtype="bf16", batch=8, drafts=5, vocab=151936, shape="peaked",
             mode="model", filters="top_p"),
        # prompt-lookup drafts of one request: every row is sampled
        dict(name="accept_b1_ngram", kind="accept", dtype="bf16", batch=1, drafts=8, vocab=151936, shape="peaked",
             mode="ngram", filters="mixed"),
        # fp32, flat distributions, both kinds of drafts in one round
        dict(name="accept_b3_f32_hybrid", kind="accept", dtype="f32", batch=3, drafts=7, vocab=50001, shape="flat",
             mode="hybrid", filters="mixed"),
        # one prompt goes on as four continuations (four layers of caches)
        dict(name="fork_b4", kind="fork", dtype="bf16", batch=4, prompts=1, layers=4, kv_heads=8, dim=128, page=256,
             context=1250, reserve=2, weights=False),
        # a beam step: sixty-four rows of four prompts, small pages
        dict(name="fork_b64_beams", kind="fork", dtype="bf16", batch=64, prompts=4, layers=2, kv_heads=8, dim=128,
             page=16, context=2003, reserve=2, weights=True),
        # a few short fp32 sequences left in a pool that others have gone from
        dict(name="compact_b3_f32", kind="compact", dtype="f32", batch=3, layers=1, kv_heads=2, dim=64, page=16,
             context=700, spread=0.4, full=0.5, weights=True),
        # eight long sequences in a pool that is a third full
        dict(name="compact_b8_long", kind="compact", dtype="bf16", batch=8, layers=1, kv_heads=8, dim=128, page=64,
             context=2500, spread=0.5, full=0.35, weights=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    """One more case of the listed cases' ranges."""
    kind = rng.choice(["sample", "sample", "sample", "accept", "accept", "accept", "fork", "fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("sample", "accept"):
        vocab = rng.choice([151936, _log_int(rng, 1000, 151936), _log_int(rng, 1000, 151936)])
        case = dict(kind=kind, dtype=dtype, vocab=vocab, shape=rng.choice(["peaked", "peaked", "flat"]),
                    filters=rng.choice(["none", "top_k", "top_p", "top_p", "min_p", "mixed", "mixed"]))
        if kind == "sample":
            most = 256 if dtype == "bf16" else 128
            return dict(case, rows=_log_int(rng, 1, most), masked=rng.choice([0.0, 0.0, 0.5, 0.99]))
        return dict(case, batch=_log_int(rng, 1, 8 if dtype == "bf16" else 4), drafts=rng.choice([1, 2, 3, 5, 8]),
                    mode=rng.choice(["model", "model", "ngram", "hybrid"]))
    kv_heads, dim, page = rng.choice([(8, 128), (8, 128), (1, 64), (3, 64)]) + (rng.choice([16, 16, 64, 256]),)
    base = dict(kind=kind, dtype=dtype, layers=rng.choice([1, 2, 3]) if page < 256 else 1, kv_heads=kv_heads, dim=dim,
                page=page, weights=rng.choice([False, True]))
    if kind == "fork":
        batch = _log_int(rng, 2, 24)
        return dict(base, batch=batch, prompts=rng.randint(1, min(5, batch)), context=_log_int(rng, 1, 2000),
                    reserve=rng.randint(0, 2))
    return dict(base, batch=_log_int(rng, 1, 8), context=_log_int(rng, 16, 2000), spread=round(rng.uniform(0.2, 1.0), 2),
                full=round(rng.uniform(0.3, 0.95), 2))


# ---------------------------------------------------------------------------
# what follows from a case alone
# ---------------------------------------------------------------------------


def _lengths(case: dict, count: int, spread: float) -> list[int]:
    """Lengths of a case's sequences: the first is the longest."""
    rng = random.Random(f"{case['kind']} {case['batch']} {case['context']}")
    lo = max(1, int(spread * case["context"]))
    return [case["context"]] + [rng.randint(lo, case["context"]) for _ in range(count - 1)]


def _beams(case: dict) -> tuple[list[int], list[int], list[int]]:
    """A fork's rows before it: each one's prompt and length (rows of one prompt
    share its pages and have as many keys), and the row each goes on from."""
    batch, prompts = case["batch"], case["prompts"]
    rng = random.Random(f"beams {batch} {prompts} {case['context']}")
    lens = _lengths(case, prompts, 0.6)
    prompt = [b * prompts // batch for b in range(batch)]
    if prompts == 1:  # one prompt's prefill is over: every row goes on from row 0
        return prompt, [lens[0]] + [0] * (batch - 1), [0] * batch
    rows = {p: [b for b in range(batch) if prompt[b] == p] for p in range(prompts)}
    parents = [rng.choice(rows[p]) for p in prompt]
    if rng.random() < 0.3:
        parents[rng.randrange(batch)] = -1  # a row that has ended
    return prompt, [lens[p] for p in prompt], parents


def _compact_pages(case: dict) -> tuple[list[int], int, int]:
    """Pages of each sequence, pages that others hold, and the pool's pages."""
    need = [-(-n // case["page"]) for n in _lengths(case, case["batch"], case["spread"])]
    held = max(1, sum(need) // 20)
    return need, held, max(sum(need) + held + 1, round((sum(need) + held) / case["full"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _logits(rows: int, case: dict, gen) -> torch.Tensor:
    """fp32 logits: a broad normal bulk, and for a peaked shape some forty
    tokens of a row well above it."""
    x = torch.randn((rows, case["vocab"]), device=DEVICE, generator=gen).mul_(2.2)
    if case["shape"] == "peaked":
        at = torch.randint(0, case["vocab"], (rows, 40), device=DEVICE, generator=gen)
        up = torch.empty((rows, 40), device=DEVICE).exponential_(0.35, generator=gen)
        x.scatter_(1, at, 8.0 + up)
    return x


def _filters(rows: int, case: dict, gen) -> dict:
    """Each row's settings, on the GPU."""
    kind, mixed = case["filters"], case["filters"] == "mixed"
    u = torch.rand((4, rows), device=DEVICE, generator=gen)
    out = dict(temperature=0.5 + u[0])
    which = torch.arange(rows, device=DEVICE) % 6  # mixed: top-p; top-k; all three; min-p; greedy; none
    if kind in ("top_k", "mixed"):
        k = (1 + 99 * u[1]).to(torch.int32)
        out["top_k"] = torch.where((which == 1) | (which == 2), k, 0).to(torch.int32) if mixed else k
    if kind in ("top_p", "mixed"):
        p = 0.8 + 0.19 * u[2]
        out["top_p"] = torch.where((which == 0) | (which == 2), p, 1.0) if mixed else p
    if kind in ("min_p", "mixed"):
        m = 0.01 + 0.1 * u[3]
        out["min_p"] = torch.where((which == 2) | (which == 3), m, 0.0) if mixed else m
    if mixed:
        out["temperature"] = torch.where(which == 4, 0.0, out["temperature"])
    return out


def _random_caches(case: dict, pool: int, gen) -> tuple[list, list]:
    """K and V pools of the layers, and key weights where the case has them."""
    shape = (pool, case["page"], case["kv_heads"], case["dim"])
    kv = [torch.randn(shape, device=DEVICE, generator=gen).to(DTYPES[case["dtype"]]) for _ in range(2 * case["layers"])]
    weights = [torch.rand((pool, case["kv_heads"], case["page"]), device=DEVICE, generator=gen)
               for _ in range(case["layers"] if case["weights"] else 0)]
    return kv, weights


def _int32(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case=case)
    if case["kind"] == "sample":
        rows, x = case["rows"], _logits(case["rows"], case, gen)
        if case["masked"]:
            x.masked_fill_(torch.rand(x.shape, device=DEVICE, generator=gen) < case["masked"], -math.inf)
        return state | dict(x=x.to(DTYPES[case["dtype"]]), filters=_filters(rows, case, gen),
                            uniforms=torch.rand(rows, device=DEVICE, generator=gen),
                            kept=torch.empty(rows, dtype=torch.int32, device=DEVICE))
    if case["kind"] == "accept":
        batch, K, V, dtype = case["batch"], case["drafts"], case["vocab"], DTYPES[case["dtype"]]
        target = _logits(batch * (K + 1), case, gen).view(batch, K + 1, V)
        # the draft model's logits: the target's, seen through some noise
        noise = torch.randn((batch, K, V), device=DEVICE, generator=gen)
        draft = (target[:, :K] + 0.4 * noise).to(dtype).contiguous()
        target = target.to(dtype)
        filters = _filters(batch, case, gen)
        # drafts: samples of the draft rows, or of the target's where they were looked up; some of them anything
        per_row = {name: x.repeat_interleave(K) for name, x in filters.items()}
        mode = torch.arange(batch, device=DEVICE) % 2 if case["mode"] == "hybrid" else None
        drafts = _sample(draft.view(-1, V), torch.rand(batch * K, device=DEVICE, generator=gen), per_row)[0].view(batch, K)
        if case["mode"] != "model":
            looked = _sample(target[:, :K].reshape(-1, V), torch.rand(batch * K, device=DEVICE, generator=gen), per_row)[0]
            looked = looked.view(batch, K)
            drafts = looked if mode is None else torch.where(mode[:, None] == 1, drafts, looked)
        odd = torch.rand((batch, K), device=DEVICE, generator=gen) < 0.05
        anything = torch.randint(0, V, (batch, K), device=DEVICE, generator=gen)
        live = [max(0, K - (b % 4 == 3)) for b in range(batch)]  # a sequence with a draft fewer
        return state | dict(
            target=target.view(-1, V), draft=draft.view(-1, V) if case["mode"] != "ngram" else None, filters=filters,
            drafts=torch.where(odd, anything, drafts).to(torch.int32), num_drafts=_int32(live),
            mode=None if mode is None else mode.to(torch.int32),
            uniforms=torch.rand((batch, K + 1), device=DEVICE, generator=gen),
            # entries past a sequence's tokens are never written
            tokens=torch.full((batch, K + 1), -1, dtype=torch.int32, device=DEVICE),
            lens=torch.empty(batch, dtype=torch.int32, device=DEVICE))
    if case["kind"] == "fork":
        prompt, lens, parents = _beams(case)
        page, batch = case["page"], case["batch"]
        whole = [n // page for n in lens]
        more = [-(-n // page) + case["reserve"] - n // page if n else 0 for n in lens]
        shared = {}  # a prompt's whole pages
        at, rows = 0, []
        for b in range(batch):
            if lens[b] and prompt[b] not in shared:
                shared[prompt[b]] = list(range(at, at + whole[b]))
                at += whole[b]
            rows.append((shared[prompt[b]] if lens[b] else []) + list(range(at, at + more[b])))
            at += more[b]
        spare = batch * (case["reserve"] + 1)
        held = 3
        pool = at + spare + held
        perm = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
        width = max(map(len, rows)) + 1
        index = torch.tensor([r + [-1] * (width - len(r)) for r in rows], device=DEVICE)
        state["tables"] = torch.where(index >= 0, perm[index.clamp_min(0)], -1).to(torch.int32)
        state |= dict(lens=torch.tensor(lens, dtype=torch.int64, device=DEVICE), parents=_int32(parents))
    else:
        need, held, pool = _compact_pages(case)
        perm = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
        index = torch.full((len(need), max(need) + 1), -1)
        at = 0
        for b, n in enumerate(need):
            index[b, :n] = torch.arange(at, at + n)
            at += n
        index = index.to(DEVICE)
        state["tables"] = torch.where(index >= 0, perm[index.clamp_min(0)], -1).to(torch.int32)
    state["held"] = torch.zeros(pool, dtype=torch.bool, device=DEVICE)
    state["held"][perm[pool - held:].long()] = True  # pages of a prefix cache, say
    kv, weights = _random_caches(case, pool, gen)
    state |= dict(kv=kv, weights=weights)
    if own:
        from naivllm_amd.layers.pages import CachePages

        state["pages"] = CachePages(kv, weights)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _keep(x: torch.Tensor, filters: dict):
    """Rows x [R, V]: their order, the kept tokens' weights in it (0 behind
    them), how many stay, and all weights.  Running sums are 64-bit, as a token
    or a cut may lie next to a border."""
    vocab = x.shape[1]
    values, order = x.float().sort(dim=1, descending=True, stable=True)
    greedy = filters["temperature"] <= GREEDY
    scale = torch.where(greedy, 1.0, filters["temperature"]).double()[:, None]
    w = values.double()
    w = w.sub_(w[:, :1].clone()).div_(scale).exp_()
    n = torch.full((x.shape[0],), vocab, device=x.device)
    if "top_k" in filters:
        k = filters["top_k"].long()
        n = torch.where((k > 0) & (k < vocab), k, n)
    run = w.cumsum(1)
    if "top_p" in filters:
        p = filters["top_p"].double()
        reach = p * run.gather(1, n[:, None] - 1)[:, 0]
        n = torch.where(p < 1, torch.minimum(n, 1 + (run < reach[:, None]).sum(1)), n)
    if "min_p" in filters:
        n = torch.minimum(n, (w >= filters["min_p"].double()[:, None]).sum(1))
    n = torch.where(greedy, 1, n.clamp_min(1))
    w.mul_(torch.arange(vocab, device=x.device)[None] < n[:, None])
    return order, w, n


def _sample(x: torch.Tensor, uniforms: torch.Tensor, filters: dict):
    order, w, n = _keep(x, filters)
    run = w.cumsum(1)
    at = (run <= (uniforms.double() * run[:, -1])[:, None]).sum(1).minimum(n - 1)
    return order.gather(1, at[:, None])[:, 0].to(torch.int32), n.to(torch.int32)


def _probabilities(x: torch.Tensor, filters: dict) -> torch.Tensor:
    order, w, _ = _keep(x, filters)
    w.div_(w.sum(1, keepdim=True))
    return torch.zeros_like(w).scatter_(1, order, w)


def _accept(state: dict):
    case, filters = state["case"], state["filters"]
    batch, K, V = case["batch"], case["drafts"], case["vocab"]
    u, drafts, live = state["uniforms"], state["drafts"].long(), state["num_drafts"].long()
    rows = torch.arange(K + 1, device=DEVICE)
    target = state["target"].view(batch, K + 1, V)
    # by samples: every row's own, kept while equal
    of_row = {name: x.repeat_interleave(K + 1) for name, x in filters.items()}
    got = _sample(state["target"], u.flatten(), of_row)[0].view(batch, K + 1).long()
    same = (got[:, :K] == drafts) & (rows[:K] < live[:, None])
    count = same.long().cumprod(1).sum(1)
    tokens = got
    if state["draft"] is not None:
        of_draft = {name: x.repeat_interleave(K) for name, x in filters.items()}
        p = _probabilities(target[:, :K].reshape(-1, V), of_draft).view(batch, K, V)
        q = _probabilities(state["draft"], of_draft).view(batch, K, V)
        at = drafts[..., None]
        keep = (u[:, :K].double() * q.gather(2, at)[..., 0] < p.gather(2, at)[..., 0]) & (rows[:K] < live[:, None])
        n = keep.long().cumprod(1).sum(1)
        here = n.clamp_max(K - 1)[:, None, None].expand(-1, 1, V)
        pt = p.gather(1, here)[:, 0]
        left = (pt - q.gather(1, here)[:, 0]).clamp_min_(0)
        left = torch.where(left.sum(1, keepdim=True) > 0, left, pt)
        run = left.cumsum(1)
        goal = u[:, K].double() * run[:, -1]
        redrawn = (run <= goal[:, None]).sum(1)
        last = torch.arange(V, device=DEVICE).mul(left > 0).amax(1)  # (the last token with any weight)
        bonus = _sample(target.gather(1, live[:, None, None].expand(-1, 1, V))[:, 0], u[:, K], filters)[0].long()
        final = torch.where(n == live, bonus, torch.minimum(redrawn, last))
        drawn = torch.where(rows < n[:, None], torch.nn.functional.pad(drafts, (0, 1)), final[:, None])
        by_logits = filters["temperature"] > GREEDY
        if state["mode"] is not None:
            by_logits &= state["mode"] != 0
        tokens = torch.where(by_logits[:, None], drawn, tokens)
        count = torch.where(by_logits, n, count)
    state["tokens"].copy_(torch.where(rows <= count[:, None], tokens, -1))
    state["lens"].copy_(count + 1)
    return state["tokens"], state["lens"]


def _ascending(flags: torch.Tensor) -> torch.Tensor:
    """The indices of the true flags, rising; the list's rest is of no account."""
    n = flags.numel()
    out = torch.zeros(n + 1, dtype=torch.int64, device=flags.device)
    at = torch.where(flags, flags.cumsum(0) - 1, n)
    out[at] = torch.arange(n, device=flags.device)
    return out[:n]


def _fork(state: dict):
    page, tables, held = state["case"]["page"], state["tables"], state["held"]
    batch, width = tables.shape
    pool = held.numel()
    valid = state["parents"] >= 0
    parent = state["parents"].long().clamp_min(0)
    old = torch.where(valid[:, None], tables[parent].long(), -1)
    lens = torch.where(valid, state["lens"][parent], 0)
    rows = torch.arange(batch, device=DEVICE)
    first = torch.full((batch + 1,), batch, device=DEVICE)
    first = first.scatter_reduce(0, torch.where(valid, parent, batch), rows, "amin")
    column = torch.arange(width, device=DEVICE)
    need = (old >= 0) & ((column + 1) * page > lens[:, None]) & (first[parent] != rows)[:, None]
    stays = (old >= 0) & ~need
    used = torch.zeros(pool + 1, dtype=torch.bool, device=DEVICE)
    used[torch.where(stays, old, pool)] = True
    free = ~(used[:pool] | held)
    ends = need.sum(1).cumsum(0)
    fits = (ends <= free.sum()) | ~need.any(1)
    fresh = _ascending(free)[(need.flatten().cumsum(0) - 1).clamp(0, pool - 1).view(batch, width)]
    alive = (valid & fits)[:, None]
    new = torch.where(alive, torch.where(need, fresh, torch.where(stays, old, -1)), -1)
    new_lens = torch.where(alive[:, 0], lens, 0)
    short = (ends[-1] - free.sum()).clamp_min(0)
    # the page that is partly filled, of every row that got one of its own
    part = (lens // page).clamp_max(width - 1)[:, None]
    copies = (alive & need.gather(1, part) & (lens % page > 0)[:, None]).nonzero()[:, 0]
    src, dst = old.gather(1, part)[copies, 0], new.gather(1, part)[copies, 0]
    live = torch.arange(page, device=DEVICE)[None] < (lens % page)[copies][:, None]
    for cache in state["kv"]:
        cache[dst] = torch.where(live[..., None, None], cache[src], cache[dst])
    for cache in state["weights"]:
        cache[dst] = torch.where(live[:, None], cache[src], cache[dst])
    return new.to(torch.int32), new_lens, short.to(torch.int32), state["kv"], state["weights"]


def _compact(state: dict):
    tables, held = state["tables"].long(), state["held"]
    pool = held.numel()
    used = torch.zeros(pool + 1, dtype=torch.bool, device=DEVICE)
    used[torch.where(tables >= 0, tables, pool)] = True
    used = used[:pool]
    movable, hole = used & ~held, ~(used | held)
    below = hole.cumsum(0) - hole.long()
    above = movable.sum() - movable.cumsum(0)
    moves = movable & (below > above)
    ids = torch.arange(pool, device=DEVICE)
    new_ids = torch.where(used | held, torch.where(moves, _ascending(hole)[above.clamp_max(pool - 1)], ids), -1)
    src = moves.nonzero()[:, 0]
    dst = new_ids[src]
    for cache in state["kv"] + state["weights"]:
        cache[dst] = cache[src]
    out = torch.where(tables >= 0, new_ids[tables.clamp_min(0)], -1)
    return out.to(torch.int32), new_ids.to(torch.int32), (new_ids.amax() + 1).to(torch.int32), state["kv"], state["weights"]


def run(state: dict):
    kind = state["case"]["kind"]
    if not own:
        if kind == "sample":
            return _sample(state["x"], state["uniforms"], state["filters"])
        return {"accept": _accept, "fork": _fork, "compact": _compact}[kind](state)
    if kind == "sample":
        from naivllm_amd.spec_engine.rejection_sampler import sample_filtered

        return sample_filtered(state["x"], uniforms=state["uniforms"], kept=state["kept"], **state["filters"]), state["kept"]
    if kind == "accept":
        from naivllm_amd.spec_engine.rejection_sampler import accept_filtered

        rows = {}
        if state["draft"] is not None:
            rows = dict(draft_logits=state["draft"], draft_seq_stride=state["case"]["drafts"], draft_mode=state["mode"])
        return accept_filtered(state["target"], state["drafts"], state["num_drafts"], uniforms=state["uniforms"],
                               out_tokens=state["tokens"], out_len=state["lens"], **rows, **state["filters"])
    if kind == "fork":
        tables, lens, short = state["pages"].fork(state["tables"], state["lens"], state["parents"], held=state["held"])
        return tables, lens, short, state["kv"], state["weights"]
    tables, new_ids, top = state["pages"].compact(state["tables"], held=state["held"])
    return tables, new_ids, top, state["kv"], state["weights"]


def work(case: dict) -> dict:
    """Logits read once, whatever they leave; pages read and written once."""
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "sample":
        rows = case["rows"]
        return dict(bytes=rows * case["vocab"] * size + 32 * rows, flops=2 * rows * case["vocab"])
    if case["kind"] == "accept":
        batch, K = case["batch"], case["drafts"]
        rows = batch * (K + 1) + (batch * K if case["mode"] != "ngram" else 0)
        if case["mode"] == "hybrid":
            rows -= (batch + 1) // 2 * K
        return dict(bytes=rows * case["vocab"] * size + 16 * rows, flops=2 * rows * case["vocab"])
    key = case["kv_heads"] * case["dim"] * size * 2 * case["layers"]
    if case["weights"]:
        key += 4 * case["kv_heads"] * case["layers"]
    if case["kind"] == "fork":
        _, lens, parents = _beams(case)
        copied = sum(lens[p] % case["page"] for b, p in enumerate(parents) if p >= 0 and p in parents[:b])
        tables = 8 * case["batch"] * (-(-case["context"] // case["page"]) + case["reserve"])
        return dict(bytes=2 * copied * key + tables + 1, flops=0)
    need, held, pool = _compact_pages(case)
    moved = sum(need) * (1 - (sum(need) + held) / pool)  # (the mean over the orders of the pool's pages)
    return dict(bytes=round(2 * moved * case["page"] * key) + 8 * sum(need) + 5 * pool, flops=0)


# ---------------------------------------------------------------------------
# the definitions in 64 bits, row by row on the host
# ---------------------------------------------------------------------------


def _row(x: np.ndarray, temperature, top_k, top_p, min_p):
    """The kept tokens of one row, in order, and their weights."""
    order = np.argsort(-x, kind="stable")
    if temperature <= GREEDY:
        return order[:1], np.ones(1)
    w = np.exp((x[order] - x[order[0]]) / temperature)
    n = top_k if 0 < top_k < len(x) else len(x)
    if top_p < 1:
        sums = np.cumsum(w[:n])
        n = min(n, int(np.searchsorted(sums, top_p * sums[-1], side="left")) + 1)
    n = max(1, min(n, int(np.count_nonzero(w >= min_p))))
    return order[:n], w[:n]


def _pick(tokens: np.ndarray, w: np.ndarray, u: float) -> int:
    sums = np.cumsum(w)
    return int(tokens[min(int(np.searchsorted(sums, u * sums[-1], side="right")), int(np.flatnonzero(w)[-1]))])


def _host_filters(state: dict, rows: int) -> list[tuple]:
    f = {name: x.double().cpu().numpy() for name, x in state["filters"].items()}
    return [(f["temperature"][b], int(f["top_k"][b]) if "top_k" in f else 0, f["top_p"][b] if "top_p" in f else 1.0,
             f["min_p"][b] if "min_p" in f else 0.0) for b in range(rows)]


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "sample":
        x, u = state["x"].double().cpu().numpy(), state["uniforms"].double().cpu().numpy()
        kept = [_row(x[r], *f) for r, f in enumerate(_host_filters(state, case["rows"]))]
        return (_int32([_pick(*kept[r], u[r]) for r in range(len(kept))]), _int32([len(k[0]) for k in kept]))
    if case["kind"] == "accept":
        return _exact_accept(case, state)
    return _exact_pages(case, state)


def _exact_accept(case: dict, state: dict):
    batch, K, V = case["batch"], case["drafts"], case["vocab"]
    u, live = state["uniforms"].double().cpu().numpy(), state["num_drafts"].tolist()
    drafts = state["drafts"].tolist()
    out = np.full((batch, K + 1), -1)
    lens = []
    for b, f in enumerate(_host_filters(state, batch)):
        target = state["target"][b * (K + 1):(b + 1) * (K + 1)].double().cpu().numpy()
        draft = None if state["draft"] is None else state["draft"][b * K:(b + 1) * K].double().cpu().numpy()
        if draft is None or f[0] <= GREEDY or (state["mode"] is not None and b % 2 == 0):
            n, token = 0, _pick(*_row(target[0], *f), u[b, 0])
            while n < live[b] and token == drafts[b][n]:
                out[b, n] = token
                n += 1
                token = _pick(*_row(target[n], *f), u[b, n])
        else:
            n, token = 0, None
            while n < live[b]:
                p, q = np.zeros(V), np.zeros(V)
                for into, x in ((p, target[n]), (q, draft[n])):
                    tokens, w = _row(x, *f)
                    into[tokens] = w / w.sum()
                if not u[b, n] * q[drafts[b][n]] < p[drafts[b][n]]:
                    left = np.maximum(p - q, 0)
                    token = _pick(np.arange(V), left if left.sum() > 0 else p, u[b, K])
                    break
                out[b, n] = drafts[b][n]
                n += 1
            if token is None:
                token = _pick(*_row(target[n], *f), u[b, K])
        out[b, n] = token
        lens.append(n + 1)
    return _int32(out.tolist()), _int32(lens)


def _exact_pages(case: dict, state: dict):
    page, tables, held = case["page"], state["tables"].tolist(), state["held"].tolist()
    moved = []  # (from, to, keys)
    if case["kind"] == "fork":
        lens, parents = state["lens"].tolist(), state["parents"].tolist()
        new = [[-1] * len(tables[0]) for _ in parents]
        wants = []
        for b, p in enumerate(parents):
            for j, e in enumerate(tables[p] if p >= 0 else []):
                if e >= 0 and (j + 1) * page > lens[p] and p in parents[:b]:
                    wants.append((b, j, e))
                else:
                    new[b][j] = e
        taken = {e for row in new for e in row}
        free = [i for i in range(len(held)) if i not in taken and not held[i]]
        assert len(wants) <= len(free)  # (prepare leaves enough)
        for (b, j, e), f in zip(wants, free):
            new[b][j] = f
            keys = min(page, lens[parents[b]] - j * page)
            if keys > 0:
                moved.append((e, f, keys))
        first = (_int32(new), torch.tensor([lens[p] if p >= 0 else 0 for p in parents], dtype=torch.int64, device=DEVICE),
                 _int32(0))
    else:
        used = sorted({e for row in tables for e in row if e >= 0})
        ids = {e: e for e in used} | {i: i for i, h in enumerate(held) if h}
        low = [i for i in range(len(held)) if i not in ids]
        for e, hole in zip([e for e in reversed(used) if not held[e]], low):
            if hole < e:
                ids[e] = hole
                moved.append((e, hole, page))
        first = (_int32([[ids[e] if e >= 0 else -1 for e in row] for row in tables]),
                 _int32([ids.get(i, -1) for i in range(len(held))]), _int32(1 + max(ids.values())))
    for e, f, keys in moved:
        for cache in state["kv"]:
            cache[f, :keys] = cache[e, :keys]
        for cache in state["weights"]:
            cache[f, :, :keys] = cache[e, :, :keys]
    return first + (state["kv"], state["weights"])
