"""GPU: columns behind the axes leave ops.rotary with the bits they came with (behind the normalisation: with their own value alone),
in the form with 16-byte vectors as in the one for any layout."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# width, axes, pairing; the last three have layouts that the vectors cannot read
CASES = [(64, (40,), "adjacent"), (64, (42,), "adjacent"), (128, (64,), "adjacent"), (128, (16, 24, 24), "adjacent"), (64, (32,), "halves"), (128, (64,), "halves"),
         (128, (16, 32), "halves"), (256, (32, 64), "halves"), (64, (20,), "halves"), (51, (40,), "adjacent"), (51, (40,), "halves")]


def _bits(t):
    return t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_bits_stay(native_lib, case, dtype):
    """Infinities, NaN and zeros of either sign beside one another and beside negative values."""
    d, axes, pairing = case
    g = torch.Generator(device=DEV).manual_seed(d + sum(axes))
    x = torch.randn(2, 9, 5, d, generator=g, device=DEV).to(dtype)
    first = sum(axes)
    specials = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.0], device=DEV).to(dtype)
    pick = torch.randint(0, 15, x.shape[:-1] + (d - first,), generator=g, device=DEV)
    x[..., first:] = torch.where(pick < 5, specials[pick % 5], x[..., first:])
    pos = torch.randint(0, 999, (9, len(axes)), generator=g, device=DEV, dtype=torch.int32)
    clean = x.clone()
    clean[..., first:] = 1.0
    for q, k in (ops.rotary(x, x[:, :, :2], pos, axes, pairing=pairing), ops.rotary(x, None, pos, axes, pairing=pairing, out_q=x.clone())):
        assert torch.equal(_bits(q[..., first:]), _bits(x[..., first:]))
        assert torch.equal(q[..., :first], ops.rotary(clean, None, pos, axes, pairing=pairing)[0][..., :first])
        assert k is None or torch.equal(_bits(k), _bits(q[:, :, :2]))


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_weights_stay_in_their_column(native_lib, case, dtype):
    """Behind the normalisation an infinite weight of a column that is not turned reaches that column alone, and a weight of -0 keeps its sign."""
    d, axes, pairing = case
    g = torch.Generator(device=DEV).manual_seed(d + sum(axes))
    x = torch.randn(1, 7, 3, d, generator=g, device=DEV).abs().to(dtype) + 0.25
    pos = torch.randint(0, 999, (7, len(axes)), generator=g, device=DEV, dtype=torch.int32)
    w = torch.ones(d, device=DEV, dtype=dtype)
    at = range(sum(axes), d, 2)
    clean = ops.rotary(x, None, pos, axes, pairing=pairing, norm_q=w)[0]
    for value in (math.inf, -0.0):
        w[list(at)] = value
        got = ops.rotary(x, None, pos, axes, pairing=pairing, norm_q=w)[0]
        mask = torch.zeros(d, dtype=torch.bool, device=DEV)
        mask[list(at)] = True
        assert torch.equal(got[..., ~mask], clean[..., ~mask])
        assert torch.equal(_bits(got[..., mask]), _bits(torch.full_like(got[..., mask], value)))
