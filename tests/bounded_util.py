"""Bounds and inputs shared by the tests of the bounded cache's operators."""

import numpy as np
import torch

EPS32 = 2.0 ** -24  # half a step of fp32
HALF = {"bf16": 2.0 ** -8, "f32": EPS32}


def weight_error(mag, keys: int, dim: int) -> np.ndarray:
    """How far a softmax weight computed in fp32 may be from its value,
    relative to it, for rows whose scores have the magnitudes ``mag``:
    a score is a sum of dim products, of which each addition is half a step
    off at most, so |error| <= (dim + 2) mag EPS32 (the scale's and log2(e)'s
    roundings included), twice for a weight (its own score's and the
    maximum's), twice again for the sum that divides it; the exponential (one
    step, 2 EPS32) and its argument's subtraction likewise; the sum of
    ``keys`` terms, no longer chain of additions than keys."""
    return 4 * (dim + 2) * mag * EPS32 + (keys + 32) * EPS32


def check_attention(got, want, want_abs, mag, dtype, keys: int, what: str = "") -> float:
    """got against the oracle's values: the weights' own error and, in bf16,
    their rounding before the second product and the output's."""
    got = got.float().cpu().numpy().astype(np.float64)
    rel = weight_error(mag, keys, want.shape[-1])[..., None]
    rounded = HALF["bf16"] if dtype == "bf16" else keys * EPS32
    bound = (rel + rounded) * want_abs * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + 1e-30
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside their bound, worst by {np.nanmax(err / bound):.2f}"
    return float(err.max())


def as_device(x, dtype="f32"):
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to("cuda", t)
