"""Inputs and the bound shared by the tests of filtered sampling."""

import numpy as np
import torch

DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def sum_error(V: int) -> float:
    """How far a running sum of V weights (the largest 1) may be off: each is
    held as an integer multiple of 2^-s with 2^s V <= 2^62, s <= 50, so it is
    half of 2^-s off at most; its exponential and the argument's two roundings
    are within 8 of 2^-53 of it (arguments up to 746 of 2^-53 relative, of
    which weights below 2^-50 need nothing: 35 of 2^-53)."""
    s = min(50, 62 - (V - 1).bit_length())
    return V * (2.0 ** -(s + 1) + 43 * 2.0 ** -53)


def logits(seed: int, rows: int, V: int, dtype: str, shape: str = "flat") -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    x = 2.2 * torch.randn((rows, V), generator=gen)
    if shape == "peaked":
        at = torch.randint(0, V, (rows, 20), generator=gen)
        x.scatter_(1, at, 8.0 + torch.empty((rows, 20)).exponential_(0.35, generator=gen))
    elif shape == "levels":  # a handful of values: ties everywhere
        x = x.round()
    elif shape == "equal":
        x = torch.zeros((rows, V))
    return x.to(DTYPE[dtype])


def settings(seed: int, rows: int) -> dict:
    """Temperatures, top-k, top-p and min-p that differ from row to row."""
    rng = np.random.default_rng(seed)
    which = np.arange(rows) % 7  # top-p; top-k; all; min-p; greedy; none; top-k and min-p
    return dict(
        temperature=np.where(which == 4, 0.0, rng.uniform(0.4, 1.6, rows)).astype(np.float32),
        top_k=np.where(np.isin(which, (1, 2, 6)), rng.integers(1, 300, rows), 0).astype(np.int32),
        top_p=np.where(np.isin(which, (0, 2)), rng.uniform(0.3, 0.999, rows), 1.0).astype(np.float32),
        min_p=np.where(np.isin(which, (2, 3, 6)), rng.uniform(0.0005, 0.2, rows), 0.0).astype(np.float32))


def on_gpu(f: dict) -> dict:
    return {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in f.items()}
