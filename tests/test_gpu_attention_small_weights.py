"""GPU: many keys of small weight beside one key of large weight.  A weight is rounded to the 16-bit type for the product with v,
counted from at least the row's largest weight so far: fp16 has steps of 2^-24 below 2^-14, so the kernels carry fp16 weights
scaled up by 2^7 (whole sequences; a weight may be 2^8 times the largest one there) or 2^14 (few rows).  Half a step is then 2^-32
or 2^-39 of the largest weight, and an output is off by that times sum |v| beside the terms of a relative rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"


def _check(q, k, v, scale, got, lse):
    """Tolerance: with u half a step of the type, n keys and A = sum p |v|, A (u + 2 eta + n 2^-23) + u |o| + 2^-32 sum |v| where a
    score is off by eta = (D + 1.5) 2^-23 sum |q k| scale + 4e-6 (bf16: no last term)."""
    tq, hq, d = q.shape
    n, hkv, _ = k.shape
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    k, v = k.repeat_interleave(hq // hkv, 0), v.repeat_interleave(hq // hkv, 0)
    s = q @ k.transpose(1, 2) * scale
    eta = (d + 1.5) * 2.0 ** -23 * (q.abs() @ k.abs().transpose(1, 2)).amax(dim=-1) * scale + 4e-6
    total = torch.logsumexp(s, dim=-1)
    p = torch.exp(s - total[..., None])
    o, a = p @ v, p @ v.abs()
    tol = a * (u + 2 * eta[..., None] + n * 2.0 ** -23) + u * o.abs() + (2.0 ** -32 * v.abs().sum(dim=1, keepdim=True) if got.dtype == torch.float16 else 0.0)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25                       # the result's own subnormals
    err = (got.double().transpose(0, 1) - o).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert ((lse.double().transpose(0, 1) - total).abs() <= eta + n * 2.0 ** -24 + 2.0 ** -22 * total.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,hq,hkv", [(1, 4, 1), (1, 1, 1), (300, 2, 2), (40, 4, 1)], ids=str)   # few rows, whole sequences, keys in parts
@pytest.mark.parametrize("below,n", [(25.2, 65536), (20.0, 65536), (23.5, 30000), (14.5, 5000)], ids=str)
@pytest.mark.parametrize("where", ["first", "last", "middle"])
def test_one_strong_key_among_many_weak_ones(native_lib, where, below, n, tq, hq, hkv, d, dtype):
    if tq * n > 300 * 30000:
        n = 30000
    at = {"first": 0, "last": n - 1, "middle": n // 2 + 5}[where]
    q = torch.zeros(1, tq, hq, d, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    k = torch.zeros(1, n, hkv, d, dtype=dtype, device=DEV)
    k[:, at, :, 0] = below * math.log(2.0)
    v = torch.ones(1, n, hkv, d, dtype=dtype, device=DEV)
    v[:, at] = 0.0
    out, lse = ops.attention(q, k, v, scale=1.0, return_lse=True)
    _check(q[0], k[0], v[0], 1.0, out[0], lse[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("tq", [1, 200])
@pytest.mark.parametrize("step", [0.5, 3.9, 7.9, 8.1, 11.0, 15.9])
def test_maximum_that_grows_tile_by_tile(native_lib, step, tq, dtype):
    """Scores that rise by `step` powers of two from one 128 keys to the next: the largest weights that the scaled type has to hold."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n = 128 * 6
    q = torch.zeros(1, tq, 2, 64, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    k = torch.zeros(1, n, 2, 64, dtype=dtype, device=DEV)
    k[..., 0] = (torch.arange(n, device=DEV) // 128 * step * math.log(2.0)).to(dtype)[None, :, None]
    v = torch.randn(1, n, 2, 64, generator=g, device=DEV).to(dtype)
    for order in (slice(None), torch.arange(n - 1, -1, -1, device=DEV)):
        kk, vv = k[:, order].contiguous(), v[:, order].contiguous()
        out, lse = ops.attention(q, kk, vv, scale=1.0, return_lse=True)
        assert torch.isfinite(out).all()
        _check(q[0], kk[0], vv[0], 1.0, out[0], lse[0])


@pytest.mark.parametrize("tq", [1, 200])
def test_largest_values(native_lib, tq):
    """Values at fp16's end times the scaled weights stay finite in the 32-bit sums."""
    k = torch.zeros(1, 4000, 2, 64, dtype=torch.float16, device=DEV)
    v = torch.full_like(k, torch.finfo(torch.float16).max)
    q = torch.ones(1, tq, 2, 64, dtype=torch.float16, device=DEV)
    assert torch.equal(ops.attention(q, k, v), torch.full_like(q, torch.finfo(torch.float16).max))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_many_sequences_of_few_rows(native_lib, dtype):
    """So many sequences that the keys of each stay in one part: one strong key beside a quarter of the weak ones in one warp."""
    n = 8000
    q = torch.zeros(75, 1, 32, 64, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    k = torch.zeros(75, n, 32, 64, dtype=dtype, device=DEV)
    k[:, 5, :, 0] = 25.2 * math.log(2.0)
    v = torch.ones_like(k)
    v[:, 5] = 0.0
    out, lse = ops.attention(q, k, v, scale=1.0, return_lse=True)
    for i in (0, 74):
        _check(q[i], k[i], v[i], 1.0, out[i], lse[i])
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(lse, lse[:1].expand_as(lse))
