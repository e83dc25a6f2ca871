"""Operators of a bounded paged cache, as measurable cases.

Kinds of cases and what each stands for:
  window          paged attention of a few rows per sequence (a decode step or
                  a verify round) that sees the last `window` keys of each row
                  and the sequence's first `sinks` keys
  window_prompt   the same for the rows of a prefill step, from the paged cache
                  (behind a cached prefix) or from the step's own K/V
  weights         paged attention of a few rows per sequence that also adds
                  the attention weight of every key, summed over the rows and
                  over the query heads of a kv head, to a paged table
  weights_prompt  the same for the rows of a prefill step
  evict           the keys with the most weight of every (sequence, kv head)
                  stay, the first and the newest ones always; rows move to the
                  front of their own table, or to pages apart

A row at position p sees the keys j <= p of its sequence; with a window only
those with j > p - window or j < sinks.  A row at position -1 is padding: it
sees nothing, and its output is zero.  The weight of a key at or behind the
position of its sequence's first row is set by the call, an older key's is
added to.  Eviction keeps min(length, budget) keys in the order of their
positions; of equal weights the lower position stays.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # the smallest call: one request's decode step over a short window
        dict(name="window_decode_b1", kind="window", dtype="bf16", batch=1, heads=16, kv_heads=8, dim=128, page=256,
             context=1250, spread=1.0, rows=1, window=512, sinks=4),
        # verify rounds of eight requests far into long documents, a wide window
        dict(name="window_verify_b8_long", kind="window", dtype="bf16", batch=8, heads=32, kv_heads=8, dim=128,
             page=256, context=32768, spread=0.6, rows=9, window=4096, sinks=4),
        # the fp32 path: small pages, odd window and sinks, contexts on both sides of the window
        dict(name="window_verify_b3_f32", kind="window", dtype="f32", batch=3, heads=16, kv_heads=8, dim=64, page=16,
             context=5003, spread=0.1, rows=6, window=999, sinks=5),
        # eight uneven prompts prefilled together from their own K/V, a window shorter than the prompts
        dict(name="window_prompt_b8", kind="window_prompt", dtype="bf16", batch=8, heads=16, kv_heads=8, dim=128,
             page=0, new=1300, spread=0.5, prefix=0, window=512, sinks=4),
        # chunks of two long prompts behind cached keys
        dict(name="window_prompt_long", kind="window_prompt", dtype="bf16", batch=2, heads=32, kv_heads=8, dim=128,
             page=256, new=4050, spread=0.7, prefix=4096, window=2048, sinks=4),
        # a decode step of eight requests that keeps score of their keys
        dict(name="weights_decode_b8", kind="weights", dtype="bf16", batch=8, heads=16, kv_heads=8, dim=128, page=256,
             context=1300, spread=0.92, rows=1),
        # the same over three single-kv-head sequences in fp32, small pages
        dict(name="weights_verify_b3_f32", kind="weights", dtype="f32", batch=3, heads=8, kv_heads=1, dim=64, page=16,
             context=7001, spread=0.3, rows=3),
        # verify rounds of sixteen long requests: the largest read of the cache
        dict(name="weights_verify_b16_long", kind="weights", dtype="bf16", batch=16, heads=32, kv_heads=8, dim=128,
             page=256, context=32768, spread=0.5, rows=9),
        # one document prompt, its keys scored for a later eviction
        dict(name="weights_prompt_b1", kind="weights_prompt", dtype="bf16", batch=1, heads=16, kv_heads=8, dim=128,
             page=256, new=1206, spread=1.0, prefix=0),
        # a long prompt of the wider model
        dict(name="weights_prompt_long", kind="weights_prompt", dtype="bf16", batch=1, heads=32, kv_heads=8, dim=128,
             page=256, new=8192, spread=1.0, prefix=0),
        # one request's cache cut to under half, to pages of its own (the document's pages are shared)
        dict(name="evict_b1_apart", kind="evict", dtype="bf16", batch=1, kv_heads=8, dim=128, page=256, context=1250,
             spread=1.0, budget=512, sinks=4, recent=64, apart=True),
        # sixteen long requests cut to a fixed size where they are
        dict(name="evict_b16_long", kind="evict", dtype="bf16", batch=16, kv_heads=8, dim=128, page=256,
             context=32768, spread=0.5, budget=2048, sinks=4, recent=256, apart=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    """One more case of the listed cases' ranges."""
    kind = rng.choice(["window", "window", "window_prompt", "weights", "weights", "weights_prompt", "evict", "evict"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (32, 8), (8, 8), (8, 1), (12, 4)])
    dim, page, batch = rng.choice([128, 128, 64]), rng.choice([16, 64, 256]), rng.choice([1, 2, 3, 5, 8, 13, 16])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    spread = round(rng.uniform(0.3, 1.0), 2)
    base = dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page, spread=spread)
    if kind in ("window", "weights"):
        group = heads // kv_heads
        case = dict(base, context=_log_int(rng, 40, 32768 if dtype == "bf16" else 8192),
                    rows=min(rng.choice([1, 1, 2, 5, 9, 12]), 64 // group))
        if kind == "window":
            case |= dict(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 17, 64]))
        return case
    if kind in ("window_prompt", "weights_prompt"):
        batch = rng.choice([1, 2, 3, 5, 8])
        new = _log_int(rng, 40, 8192 // batch)
        prefix = page * rng.choice([0, 0, 1, _log_int(rng, 1, 4096 // page)])
        case = dict(base, dtype="bf16", batch=batch, new=new, prefix=prefix)
        if kind == "window_prompt":
            case |= dict(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 17, 64]),
                         page=rng.choice([page, 0]) if prefix == 0 else page)
        return case
    context = _log_int(rng, 200, 32768 if dtype == "bf16" else 16384)
    budget = _log_int(rng, 64, max(64, context // 2))
    sinks = rng.choice([0, 4, 17])
    del base["heads"]
    return dict(base, context=context, budget=budget, sinks=sinks, recent=rng.randint(0, budget - sinks),
                apart=rng.choice([False, True]))


def _lengths(case: dict, longest: int) -> list[int]:
    """Lengths of the case's sequences: the first is the longest, the others
    lie between spread * longest and it."""
    rng = random.Random(f"{case['kind']} {case['batch']} {longest}")
    lo = max(1, int(case["spread"] * longest))
    return [longest] + [rng.randint(lo, longest) for _ in range(case["batch"] - 1)]


def _row_counts(case: dict, lens: list[int]) -> list[int]:
    """Live rows of each sequence in a step of case["rows"] rows: all of them,
    in every third sequence one less (a draft fewer)."""
    return [max(1, min(case["rows"] - (b % 3 == 1), n)) for b, n in enumerate(lens)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _pattern(dim: int) -> torch.Tensor:
    """The direction that queries and much-attended keys share."""
    return torch.tensor([1.0 if i % 3 else -1.0 for i in range(dim)], device=DEVICE)


def _queries(shape, dtype, gen) -> torch.Tensor:
    return (torch.randn(shape, device=DEVICE, generator=gen) + _pattern(shape[-1])).to(dtype)


def _keys(shape, dtype, gen) -> torch.Tensor:
    """Keys of which a few draw much attention (a heavy-tailed share of the
    common direction)."""
    strength = 0.05 * torch.randn((*shape[:-1], 1), device=DEVICE, generator=gen).square()
    return (torch.randn(shape, device=DEVICE, generator=gen) + strength * _pattern(shape[-1])).to(dtype)


def _tables(lens: list[int], page: int, more: int, gen) -> tuple[torch.Tensor, int]:
    """Block tables with room for `more` keys per sequence, pages in no order,
    and the pool's size."""
    need = [-(-(n + more) // page) for n in lens]
    pool = sum(need) + 3
    perm = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
    tables = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = perm[at:at + n]
        at += n
    return tables, pool


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, dim, kv_heads, kind = DTYPES[case["dtype"]], case["dim"], case["kv_heads"], case["kind"]
    state = dict(case=case, scale=1.0 / math.sqrt(dim))
    if kind in ("window", "weights"):
        lens = _lengths(case, case["context"])
        counts, rows = _row_counts(case, lens), case["rows"]
        tables, pool = _tables(lens, case["page"], 0, gen)
        positions = torch.full((case["batch"], rows), -1, dtype=torch.int64)
        for b, (n, live) in enumerate(zip(lens, counts)):
            positions[b, :live] = torch.arange(n - live, n)
        state |= dict(query=_queries((case["batch"] * rows, case["heads"], dim), dtype, gen), tables=tables,
                      lens=torch.tensor(lens, dtype=torch.int64, device=DEVICE),
                      cu=torch.arange(0, case["batch"] * rows + 1, rows, dtype=torch.int32, device=DEVICE),
                      positions=positions.reshape(-1).to(DEVICE))
    elif kind in ("window_prompt", "weights_prompt"):
        new = _lengths(case, case["new"])
        ends = [n + case["prefix"] for n in new]
        state |= dict(query=_queries((sum(new), case["heads"], dim), dtype, gen), new=new, ends=ends)
        if case["page"]:
            tables, pool = _tables(ends, case["page"], 0, gen)
            state["tables"] = tables
        else:  # the step's own keys, back to back
            state |= dict(k=_keys((sum(ends), kv_heads, dim), dtype, gen),
                          v=torch.randn((sum(ends), kv_heads, dim), device=DEVICE, generator=gen).to(dtype))
            pool = 0
        row0 = np.cumsum([0] + new)
        widest = max(new)
        state |= dict(
            # where the step's rows lie in a batch padded to its longest prompt, and back
            pad=torch.tensor([[row0[b] + min(r, n - 1) for r in range(widest)] for b, n in enumerate(new)], device=DEVICE),
            unpad=torch.tensor(np.concatenate([b * widest + np.arange(n) for b, n in enumerate(new)]), device=DEVICE))
        if own:
            from naivllm_amd.layers.attention import KeyWeightsPlan, PrefillPlan

            window = dict(window=case["window"], sinks=case["sinks"]) if kind == "window_prompt" else {}
            state["plan"] = PrefillPlan(new, ends, case["heads"], kv_heads, case["page"] or None,
                                        torch.device(DEVICE, torch.cuda.current_device()), **window)
            if kind == "weights_prompt":
                state["weights_plan"] = KeyWeightsPlan(new, ends, case["heads"], kv_heads, case["page"],
                                                       torch.device(DEVICE, torch.cuda.current_device()))
                state["stats"] = torch.empty((sum(new), case["heads"], 2), device=DEVICE)
    else:
        lens = _lengths(case, case["context"])
        tables, pool = _tables(lens, case["page"], 0, gen)
        state |= dict(tables=tables, lens=torch.tensor(lens, dtype=torch.int64, device=DEVICE))
        if case["apart"]:
            out, extra = _tables([min(n, case["budget"]) for n in lens], case["page"], 0, gen)
            state["out_tables"] = torch.where(out >= 0, out + pool, -1).to(torch.int32)
            pool += extra
    if pool:
        shape = (pool, case["page"], kv_heads, dim)
        state |= dict(k=_keys(shape, dtype, gen), v=torch.randn(shape, device=DEVICE, generator=gen).to(dtype))
        if kind in ("weights", "weights_prompt", "evict"):
            # what earlier steps left: a heavy-tailed share for each key; on a grid before an eviction, so that some are equal
            w = torch.randn((pool, kv_heads, case["page"]), device=DEVICE, generator=gen).square()
            state["weights"] = (w.square() * 64).floor() / 64 if kind == "evict" else w / 64
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _gather(cache: torch.Tensor, tables: torch.Tensor, keys: torch.Tensor) -> torch.Tensor:
    """Rows [B, n, Hkv, D] of the keys [B, n] of each sequence."""
    page = cache.shape[1]
    return cache[tables.long().gather(1, keys // page), keys % page]


def _attend(q, k, v, visible, scale):
    """q [B, R, H, D], k and v [B, n, Hkv, D], visible [B, R, n] -> (out
    [B, R, H, D], weights [B, Hkv, n] summed over rows and group heads)."""
    batch, rows, heads, dim = q.shape
    kv_heads, n = k.shape[2], k.shape[1]
    q = q.float().view(batch, rows, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
    s = torch.matmul(q, k.float().permute(0, 2, 3, 1).contiguous()).mul_(scale)
    s = s.view(batch, kv_heads, -1, rows, n).masked_fill_(~visible[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-30))
    out = torch.matmul(p.view(batch, kv_heads, -1, n), v.float().permute(0, 2, 1, 3).contiguous())
    out = out.view(batch, kv_heads, -1, rows, dim).permute(0, 3, 1, 2, 4).reshape(batch, rows, heads, dim)
    return out, p.sum((2, 3))


def _sees(positions: torch.Tensor, keys: torch.Tensor, case: dict) -> torch.Tensor:
    """[B, R, n]: whether the row at a position sees the key at an index."""
    p, j = positions[:, :, None], keys[:, None, :]
    seen = j <= p
    if "window" in case:
        seen &= (j > p - case["window"]) | (j < case["sinks"])
    return seen


def _add_weights(weights, tables, lens, first, sums):
    """sums [B, Hkv, n] into the paged weights: set from key first[b] on,
    added before."""
    kv_heads, page = weights.shape[1:]
    j = torch.arange(sums.shape[2], device=sums.device)[None]
    j = j.minimum(lens[:, None] - 1)  # (keys past a sequence's last are its last again)
    sums = sums.gather(2, j[:, None].expand(-1, kv_heads, -1)).transpose(1, 2)
    at = tables.long().gather(1, j // page), j % page
    old = weights[at[0], :, at[1]]
    weights[at[0], :, at[1]] = torch.where((j < first[:, None])[..., None], old, 0.0) + sums


def _few_rows(state: dict):
    case, lens = state["case"], state["lens"]
    batch, rows = case["batch"], case["rows"]
    q = state["query"].view(batch, rows, case["heads"], case["dim"])
    positions = state["positions"].view(batch, rows)
    if case["kind"] == "window":
        # each sequence's sinks and the union of its rows' windows
        sinks, span = case["sinks"], case["window"] + rows - 1
        keys = torch.cat([torch.arange(sinks, device=DEVICE).expand(batch, -1),
                          lens[:, None] - span + torch.arange(span, device=DEVICE)[None]], 1)
        fits = (keys >= 0) & (keys < lens[:, None])
        fits[:, sinks:] &= keys[:, sinks:] >= sinks
    else:
        keys = torch.arange(case["context"], device=DEVICE).expand(batch, -1)
        fits = keys < lens[:, None]
    at = keys.clamp_min(0).minimum(lens[:, None] - 1)
    visible = _sees(positions, keys, case) & fits[:, None]
    out, sums = _attend(q, _gather(state["k"], state["tables"], at), _gather(state["v"], state["tables"], at), visible,
                        state["scale"])
    out = out.to(state["query"].dtype).reshape(state["query"].shape)
    if case["kind"] == "window":
        return out
    _add_weights(state["weights"], state["tables"], lens, positions[:, 0], sums)
    return out, state["weights"]


def _prompt(state: dict):
    case = state["case"]
    new, ends = (torch.tensor(state[x], device=DEVICE) for x in ("new", "ends"))
    row = torch.arange(state["pad"].shape[1], device=DEVICE)[None]
    keys = torch.arange(max(state["ends"]), device=DEVICE).expand(case["batch"], -1)
    at = keys.minimum(ends[:, None] - 1)
    if case["page"]:
        k, v = (_gather(state[x], state["tables"], at) for x in "kv")
    else:
        at = at + (ends.cumsum(0) - ends)[:, None]
        k, v = state["k"][at], state["v"][at]
    positions = torch.where(row < new[:, None], (ends - new)[:, None] + row, -1)
    out, sums = _attend(state["query"][state["pad"]], k, v, _sees(positions, keys, case), state["scale"])
    out = out.flatten(0, 1)[state["unpad"]].to(state["query"].dtype)
    if case["kind"] == "window_prompt":
        return out
    _add_weights(state["weights"], state["tables"], ends, ends - new, sums)
    return out, state["weights"]


def _evict(state: dict):
    case, lens, tables, weights = state["case"], state["lens"], state["tables"], state["weights"]
    budget, kv_heads, page = case["budget"], case["kv_heads"], case["page"]
    j = torch.arange(case["context"], device=DEVICE).expand(case["batch"], -1)
    at = j.minimum(lens[:, None] - 1)
    w = weights[tables.long().gather(1, at // page), :, at % page].transpose(1, 2).clone()
    n = lens[:, None]
    w.masked_fill_(((j < case["sinks"]) | (j >= n - case["recent"]))[:, None], math.inf)
    w.masked_fill_((j >= n)[:, None], -math.inf)
    kept = w.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    got = lens.clamp_max(budget)
    slot = torch.arange(kept.shape[2], device=DEVICE)
    kept = torch.where(slot < got[:, None, None], kept, case["context"]).sort(-1).values
    # (a slot past a sequence's new length gets the last kept row again)
    i = slot.minimum(got[:, None] - 1)
    src = kept.gather(2, i[:, None].expand(-1, kv_heads, -1))
    head = torch.arange(kv_heads, device=DEVICE)[None, :, None]
    pages = tables.long()[:, None].expand(-1, kv_heads, -1).gather(2, src // page)
    to = state.get("out_tables", tables).long().gather(1, i // page)[:, None].expand(-1, kv_heads, -1)
    off = (i % page)[:, None].expand(-1, kv_heads, -1)
    for x in ("k", "v"):
        state[x][to, off, head] = state[x][pages, src % page, head]
    weights[to, head, off] = weights[pages, head, src % page]
    full = torch.full((*kept.shape[:2], budget), -1, dtype=torch.int32, device=DEVICE)
    full[..., :kept.shape[2]] = torch.where(slot < got[:, None, None], kept, -1).to(torch.int32)
    return state["k"], state["v"], weights, got, full


def run(state: dict):
    case = state["case"]
    if not own:
        return {"window": _few_rows, "weights": _few_rows, "window_prompt": _prompt, "weights_prompt": _prompt,
                "evict": _evict}[case["kind"]](state)
    from naivllm_amd.layers import attention as ops

    kind, s = case["kind"], state
    if kind in ("window", "weights"):
        shape = (s["scale"], case["heads"], case["kv_heads"], case["dim"], case["page"], 16)
        meta = (s["tables"], s["lens"], s["cu"], s["positions"], *shape)
        if kind == "window":
            return ops.paged_attention_window(s["query"], s["k"], s["v"], *meta, window=case["window"],
                                              sinks=case["sinks"], max_q_len=case["rows"])
        out = ops.paged_attention_weights(s["query"], s["k"], s["v"], s["weights"], *meta, max_q_len=case["rows"])
        return out, s["weights"]
    if kind == "window_prompt":
        return ops.prefill_attention(s["query"], s["k"], s["v"], s["plan"], s["scale"], case["dim"], s.get("tables"))
    if kind == "weights_prompt":
        out = ops.prefill_attention(s["query"], s["k"], s["v"], s["plan"], s["scale"], case["dim"], s["tables"],
                                    stats=s["stats"])
        ops.prefill_key_weights(s["query"], s["k"], s["weights"], s["weights_plan"], s["stats"], s["scale"], case["dim"],
                                s["tables"])
        return out, s["weights"]
    lens, kept = ops.evict_kvcache(s["k"], s["v"], s["weights"], s["tables"], s["lens"], case["budget"],
                                   sinks=case["sinks"], recent=case["recent"], out_block_tables=s.get("out_tables"))
    return s["k"], s["v"], s["weights"], lens, kept


# ---------------------------------------------------------------------------
# 64 bits, one sequence and kv head at a time
# ---------------------------------------------------------------------------


def _exact_head(q, k, v, positions, window, sinks, scale):
    """Attention of rows q [R, G, D] at positions [R] over the keys 0 .. n - 1
    (k, v [n, D]); returns (out [R, G, D], weights [n])."""
    n, out, sums = k.shape[0], torch.zeros_like(q), torch.zeros(k.shape[0], dtype=torch.float64, device=k.device)
    j = torch.arange(n, device=k.device)
    for r0 in range(0, q.shape[0], 2048):
        p = positions[r0:r0 + 2048, None]
        hidden = j[None] > p
        if window:
            hidden |= (j[None] <= p - window) & (j[None] >= sinks)
        hidden = hidden[:, None].expand(-1, q.shape[1], -1)
        logits = (q[r0:r0 + 2048].reshape(-1, q.shape[2]) @ k.T * scale).reshape(hidden.shape)
        logits = torch.where(hidden, -math.inf, logits)
        prob = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
        prob = torch.where(hidden, 0.0, prob)  # (a row that sees nothing: NaN before)
        out[r0:r0 + 2048] = (prob.reshape(-1, n) @ v).view(-1, *q.shape[1:])
        sums += prob.sum((0, 1))
    return out, sums


def _exact_attention(state: dict):
    case = state["case"]
    few = case["kind"] in ("window", "weights")
    group = case["heads"] // case["kv_heads"]
    ends = state["lens"].tolist() if few else state["ends"]
    counts = [case["rows"]] * case["batch"] if few else state["new"]
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device=DEVICE)
    weights = state["weights"].double() if "weights" in state else None
    row = key = 0
    for b, (n, count) in enumerate(zip(ends, counts)):
        if few:
            positions = state["positions"][row:row + count]
        else:
            positions = torch.arange(n - count, n, device=DEVICE)
        if case["page"]:
            pages = state["tables"][b, :-(-n // case["page"])].long()
            k, v = (state[x][pages].flatten(0, 1)[:n] for x in "kv")
        else:
            k, v = (state[x][key:key + n] for x in "kv")
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            o, sums = _exact_head(state["query"][row:row + count, heads].double(), k[:, h].double(), v[:, h].double(),
                                  positions, case.get("window"), case.get("sinks"), state["scale"])
            out[row:row + count, heads] = o
            if weights is not None:
                mine = weights[pages, h].flatten()
                mine[int(positions[0]):n] = 0.0
                mine[:n] += sums
                weights[pages, h] = mine.view(len(pages), -1)
        row, key = row + count, key + n
    return out if weights is None else (out, weights)


def _exact_evict(state: dict):
    case, page = state["case"], state["case"]["page"]
    tables, lens = state["tables"].cpu().numpy(), state["lens"].tolist()
    to_tables = state["out_tables"].cpu().numpy() if case["apart"] else tables
    old = state["weights"].double().cpu().numpy()
    k, v, weights = (state[x].clone() for x in ("k", "v", "weights"))
    all_kept = np.full((case["batch"], case["kv_heads"], case["budget"]), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        for h in range(case["kv_heads"]):
            w = old[tables[b, :-(-n // page)], h].reshape(-1)[:n]
            index = np.arange(n)
            always = (index < case["sinks"]) | (index >= n - case["recent"])
            kept = np.sort(np.lexsort((index, -w, ~always))[:case["budget"]])
            all_kept[b, h, :kept.size] = kept
            i = np.arange(kept.size)
            src, to = tables[b][kept // page], to_tables[b][i // page]
            src, to, off, at = (torch.from_numpy(x).long().to(DEVICE) for x in (src, to, kept % page, i % page))
            k[to, at, h], v[to, at, h] = state["k"][src, off, h], state["v"][src, off, h]
            weights[to, h, at] = state["weights"][src, h, off]
    return (k, v, weights, torch.tensor([min(n, case["budget"]) for n in lens], device=DEVICE),
            torch.from_numpy(all_kept).to(DEVICE))


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return _exact_evict(state) if case["kind"] == "evict" else _exact_attention(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def _visible(first: int, count: int, window: int | None, sinks: int) -> int:
    """Pairs (row, key) of rows at positions first .. first + count - 1."""
    p = np.arange(first, first + count, dtype=np.int64)
    if window is None:
        return int((p + 1).sum())
    return int((np.minimum(p + 1, window) + np.clip(p + 1 - window, 0, sinks)).sum())


def work(case: dict) -> dict:
    elt, kv_heads, dim = (2 if case["dtype"] == "bf16" else 4), case["kv_heads"], case["dim"]
    row = kv_heads * dim * elt * 2  # K and V of one key
    if case["kind"] == "evict":
        lens = _lengths(case, case["context"])
        moved = sum(min(n, case["budget"]) for n in lens if n > case["budget"] or case["apart"])
        read = sum(n for n in lens if n > case["budget"])
        return dict(bytes=read * kv_heads * 4 + 2 * moved * (row + 4 * kv_heads), flops=0)
    few = case["kind"] in ("window", "weights")
    ends = _lengths(case, case["context"] if few else case["new"])
    counts = _row_counts(case, ends) if few else ends
    if not few:
        ends = [n + case["prefix"] for n in ends]
    window, sinks = case.get("window"), case.get("sinks", 0)
    pairs = keys = 0
    for n, count in zip(ends, counts):
        pairs += _visible(n - count, count, window, sinks)
        seen = n if window is None else min(n, window + count - 1)
        keys += seen + min(sinks, n - seen)
    total = keys * row + 2 * sum(counts) * case["heads"] * dim * elt
    if "weights" in case["kind"]:
        total += 8 * kv_heads * keys
    return dict(bytes=total, flops=4 * dim * case["heads"] * pairs)
