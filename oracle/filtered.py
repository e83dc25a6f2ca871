"""CPU oracle of sampling and acceptance under a temperature, top-k, top-p and
min-p — TEST INFRASTRUCTURE ONLY, as oracle/accept.py.

float64 numpy, one row at a time, from the definitions in include/naivspec.h
(nsv_sample_filtered, nsv_accept_filtered).  No reference counterpart.
"""

from __future__ import annotations

import numpy as np

GREEDY = 1e-6


def _argmax(x) -> int:
    nan = np.isnan(x)
    return int(np.argmax(nan)) if nan.any() else int(np.argmax(x))


class Row:
    """What the filters leave of one row: ``order`` (all tokens, by falling
    logit, equal ones by rising index), ``w`` their weights, ``n`` how many
    stay, ``goal`` the sum that top-p had to reach (None: not applied) and
    ``alone``: the argmax stays whatever the filters are."""

    def __init__(self, x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        x = np.asarray(x, dtype=np.float64)
        V = len(x)
        self.vocab, self.goal = V, None
        self.alone = not temperature > GREEDY or np.isnan(x).any() or x.max() == -np.inf
        if self.alone:
            first = _argmax(x)
            self.order = np.array([first] + [i for i in range(V) if i != first])
            self.w = np.zeros(V)
            self.w[0] = 1.0
            self.n = 1
            return
        self.order = np.argsort(-x, kind="stable")
        s = x[self.order]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.exp(np.where(s == -np.inf, -np.inf, (s - s[0]) / temperature))
        w[s == s[0]] = 1.0
        w[s == -np.inf] = 0.0
        self.w = w
        self.n_k = n = int(top_k) if 0 < top_k < V else V
        if top_p < 1:
            sums = np.cumsum(w[:n])
            self.goal = top_p * sums[-1]
            n = min(n, int(np.searchsorted(sums, self.goal, side="left")) + 1)
        self.n_m = V
        if min_p > 0:
            self.n_m = max(1, int(np.count_nonzero((w >= min_p) | (s == s[0]))))
            n = min(n, self.n_m)
        self.n = n

    def kept(self):
        return self.order[:self.n], self.w[:self.n]

    def sample(self, u: float) -> int:
        tokens, w = self.kept()
        sums = np.cumsum(w)
        at = int(np.searchsorted(sums, min(max(float(u), 0.0), 1.0) * sums[-1], side="right"))
        return int(tokens[min(at, int(np.flatnonzero(w)[-1]))])

    def probabilities(self) -> np.ndarray:
        p = np.zeros(self.vocab)
        tokens, w = self.kept()
        p[tokens] = w / w.sum()
        return p

    def admits(self, kept: int, token: int, u: float, eps: float) -> str | None:
        """None if a sampler whose running sums are off by eps at most may
        leave ``kept`` tokens and draw ``token``; else what is wrong."""
        sums = np.concatenate([[0.0], np.cumsum(self.w)])
        if kept != self.n:
            borders = self.goal is not None and kept <= min(self.n_k, self.n_m) and (
                sums[kept] >= self.goal - eps and sums[kept - 1] < self.goal + eps)
            if not borders:
                return f"{kept} tokens kept, {self.n} wanted"
        at = int(np.flatnonzero(self.order == token)[0]) if 0 <= token < self.vocab else -1
        if not 0 <= at < kept:
            return f"token {token} is not among the {kept} kept"
        goal = float(u) * sums[kept]
        if not (sums[at] <= goal + eps and sums[at + 1] > goal - eps):
            return f"token {token}: running sums {sums[at]}..{sums[at + 1]}, goal {goal}, wanted {self.sample(u)}"
        return None


def accept(target, draft, drafts, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> list[int]:
    """One sequence's tokens.  target [n + 1, V], draft [n, V] or None, drafts
    n tokens, uniforms [n + 1] with the last number the draw behind kept
    drafts or from a residual (rows are sampled where draft is None)."""
    f = (temperature, top_k, top_p, min_p)
    n = len(drafts)
    if draft is None or not temperature > GREEDY:
        out = []
        for r in range(n + 1):
            out.append(Row(target[r], *f).sample(uniforms[r]))
            if r == n or out[-1] != drafts[r]:
                return out
    out = []
    for i, d in enumerate(drafts):
        p, q = Row(target[i], *f).probabilities(), Row(draft[i], *f).probabilities()
        inside = 0 <= d < len(p)
        if float(uniforms[i]) * (q[d] if inside else 0.0) < (p[d] if inside else 0.0):
            out.append(int(d))
            continue
        left = np.maximum(p - q, 0.0)
        if not left.sum() > 0:
            left = p
        sums = np.cumsum(left)
        at = int(np.searchsorted(sums, float(uniforms[-1]) * sums[-1], side="right"))
        return out + [min(at, int(np.flatnonzero(left)[-1]))]
    return out + [Row(target[n], *f).sample(uniforms[-1])]
