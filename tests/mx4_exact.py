"""Products whose FP32 results are exact, so that one element in 4 bits that is off by its smallest step shows.

Every element is a multiple of 0.5 of at most 6 in magnitude, scales are 1, 2 or 4 for the weights and 1 for the activations. A product is then a multiple of 1/4 and at most
144, and as long as the sum of all magnitudes stays below 2^22 every partial sum, in any order and any grouping, is a multiple of 1/4 below 2^22: 24 bits hold it."""
import torch

import mx4_reference as ref


def weights(rows, K, seed, count=1):
    """Blocks of a file (on the CPU) of count * rows rows."""
    return ref.random_blocks(count * rows * (K // 32), seed, lo=127, hi=130)


def activations(shape, dtype, seed, device="cpu"):
    """Rows that MXFP4 keeps as they are: the largest magnitude of a block is 4 or 6, which gives the scale 1."""
    g = torch.Generator().manual_seed(seed)
    lut = torch.tensor(ref.VALUES)
    x = lut[torch.randint(0, 8, shape, generator=g)].unflatten(-1, (-1, 32))
    at = torch.randint(0, 32, x.shape[:-1] + (1,), generator=g)
    x.scatter_(-1, at, lut[6 + torch.randint(0, 2, at.shape, generator=g)])
    sign = 1.0 - 2.0 * torch.randint(0, 2, x.shape, generator=g)
    return (x * sign).flatten(-2).to(device=device, dtype=dtype)


def sums_are_exact(q, w):
    """Whether every partial sum of q w^T (or of its magnitudes) fits 24 bits."""
    return bool((q.abs() @ w.abs().T).max() < 2 ** 22)


def same(got, want):
    """Raises with the places where the results differ."""
    got = got.double()
    if torch.equal(got, want):
        return
    off = (got != want).nonzero()
    rows, cols = off[:, -2].unique(), off[:, -1].unique()
    first = tuple(off[0].tolist())
    raise AssertionError(f"{len(off)} of {want.numel()} results differ, in rows {rows[:8].tolist()} and columns {cols[:8].tolist()}; at {first} "
                         f"{got[first].item()!r} for {want[first].item()!r}")
