"""CPU: which outputs overlap themselves or an input, against the sets of addresses that the tensors touch."""
import random

import pytest
import torch

from segquant_b200 import ops


def _set(t):
    offs = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        offs = (offs[:, None] + torch.arange(n) * s).flatten()
    return (offs + t.storage_offset()).tolist()


@pytest.mark.parametrize("seed", range(300))
def test_layouts_against_their_addresses(seed):
    """Random small layouts in one buffer: nested ones, gaps, shifts by columns, heads and tokens, strides that meet."""
    rng = random.Random(seed)
    buf = torch.zeros(4000, dtype=torch.bfloat16)

    def draw(strides=None, width=None):
        d = width or rng.choice([2, 8])
        n = [rng.randint(1, 4) for _ in range(3)]
        if strides is None:
            if rng.random() < 0.5:
                strides, at = [], d * rng.choice([1, 1, 2])
                for m in n[::-1]:
                    strides.insert(0, at)
                    at *= m + rng.choice([0, 0, 1, 3])
            else:
                strides = [rng.randint(0 if rng.random() < 0.1 else 1, 80) for _ in n]
            if rng.random() < 0.3:
                rng.shuffle(strides)
        return buf.as_strided((*n, d), (*strides, 1), rng.randint(0, 200)), strides, d

    a, strides, d = draw()
    elements = _set(a)
    assert ops._overlaps_itself(a) == (len(set(elements)) < len(elements))
    b, _, _ = draw(strides, d)                                   # the same strides: exact
    assert ops._overlap(a, b) == bool(set(elements) & set(_set(b)))
    c, _, _ = draw(None, d)                                      # others: never a false alarm
    assert not ops._overlap(a, c) or set(elements) & set(_set(c))


def test_nothing_overlaps_nothing():
    x = torch.zeros(2, 0, 4, 8)
    assert not ops._overlaps_itself(x) and not ops._overlap(x, x)
