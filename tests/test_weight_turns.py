"""The calls that an fp32 prefill step with key weights is cut into, on the
CPU."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers import attention


class OnTheHost(attention._WeightTurns):
    def _send(self, work, device, ahead):
        self.work = work


@pytest.fixture(autouse=True)
def _no_device(monkeypatch):
    monkeypatch.setattr(attention, "_send_ahead", lambda: False)


@pytest.mark.parametrize("q_block", [1, 5, 32])
def test_every_row_once_and_sets_before_adds(q_block):
    new, ends = [70, 1, 33, 64], [70, 200, 97, 192]
    tables = torch.arange(4 * 13, dtype=torch.int32).view(4, 13)
    plan = OnTheHost(new, ends, tables, q_block, "cpu")
    assert plan.rows == sum(new)
    first, seen = np.cumsum([0] + new), {}
    for turn, (rows, bt, lens, cu, positions) in enumerate(plan.turns):
        rows = np.arange(*rows) if isinstance(rows, tuple) else rows.numpy()
        assert bt.dtype == cu.dtype == torch.int32 and lens.dtype == positions.dtype == torch.int64
        assert cu[0] == 0 and cu[-1] == len(rows) == len(positions) and bt.shape == (len(lens), 13)
        owners = []
        for i, (a, z) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
            b = int(np.searchsorted(first, rows[a], side="right")) - 1
            owners.append(b)
            assert 0 < z - a <= q_block and torch.equal(bt[i], tables[b]) and lens[i] == positions[z - 1] + 1
            for r, p in zip(rows[a:z], positions[a:z].tolist()):
                assert p == ends[b] - new[b] + r - first[b] and (b, p) not in seen
                seen[b, p] = turn
            # what another sequence sets among the keys before this block's first has its turn by now
            start = int(positions[a])
            seen.setdefault("adds", []).append((turn, start))
        assert len(set(owners)) == len(owners)  # one block of a sequence per turn
    adds = seen.pop("adds")
    assert len(seen) == sum(new)
    for (b, p), turn in seen.items():
        assert all(turn <= t for t, start in adds if p < start)


def test_refused():
    tables = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="2 sequences"):
        OnTheHost([3, 4], [3, 4], tables, 32, "cpu")
    with pytest.raises(ValueError, match="query rows over"):
        OnTheHost([3], [2], tables, 32, "cpu")
